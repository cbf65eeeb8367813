"""Attention with a window and first keys that stay visible, on the GPU, against the
float64 restatement in oracle/token_ref.py. Tolerances are those of the attention
without a window: the restatement's bound (p, ds and the results each rounded to the
type once, every rounding at its worst), 2^-14 of the magnitudes summed for
float32's part, and float16's spacing below 2^-14."""

from __future__ import annotations

import zlib

import numpy as np
import pytest
import torch

from oracle import token_ref

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
UNIT = {name: torch.finfo(t).eps / 2 for name, t in TYPES.items()}


def host(t):
    return t.detach().cpu().double().numpy()


def gen(*key):
    return torch.Generator().manual_seed(zlib.crc32(repr(key).encode()))


def offsets(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(int).tolist()


def inputs(key, nq, nk, heads, kv, dim, ty):
    g = gen(*key)
    return [torch.randn(n, h, dim, generator=g).to(TYPES[ty])
            for n, h in ((nq, heads), (nk, kv), (nk, kv), (nq, heads))]


def check(dev, q, k, v, do, q_lens, k_lens, ty, window, sinks, grad=True, scale=None):
    from metal_gauss_amd import attention

    qo, ko = offsets(q_lens), offsets(k_lens)
    put = [torch.tensor(o, dtype=torch.int32, device=dev) for o in (qo, ko)]
    leaves = [t.to(dev).requires_grad_(grad) for t in (q, k, v)]
    kw = dict(causal=True, window=window, sinks=sinks, scale=scale)
    o = attention(*leaves, *put, **kw)
    want, off = token_ref.attention(host(q), host(k), host(v), qo, ko, True,
                                    scale if scale is not None else q.shape[2] ** -0.5,
                                    host(do) if grad else None, UNIT[ty], window, sinks)
    tiny = 2.0 ** -24 if ty == "f16" else 1e-30
    names, got = ("o", "dq", "dk", "dv"), [o]
    if grad:
        got += torch.autograd.grad(o, leaves, do.to(dev))
        with torch.no_grad():
            assert torch.equal(attention(*leaves, *put, **kw), o)
    for name, a, w, b in zip(names, got, want, off):
        a, bound = host(a), b * (1.0 + 2.0 ** -14 / UNIT[ty]) * 1.05 + tiny
        bad = np.abs(a - w) - bound
        assert np.isfinite(a).all() and (bad <= 0).all(), \
            f"{name}: {np.abs(a - w).max():.3e} off, {bad.max():.3e} over the bound"
    return got


PACKS = [
    ([1], [1]), ([65], [65]), ([200, 31, 300, 0, 5], [200, 31, 300, 0, 5]),
    ([1, 1, 1, 1], [1, 700, 64, 129]),              # single tokens over memories
    ([17, 100, 3], [300, 100, 900]),                # chunks over memories
    ([100, 5, 200], [30, 5, 1]),                    # more queries than keys
    ([10, 0, 20], [0, 12, 20]),                     # no keys, no queries
]


@pytest.mark.parametrize("q_lens,k_lens", PACKS)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 3), (40, 0), (64, 4), (100, 33), (130, 70),
                                          (7, 200), (10 ** 9, 5)])
@pytest.mark.parametrize("ty,heads,kv,dim", [("bf16", 4, 2, 64), ("f16", 6, 2, 128),
                                             ("bf16", 3, 3, 32), ("f16", 5, 1, 80)])
def test_window(dev, q_lens, k_lens, window, sinks, ty, heads, kv, dim):
    key = (sum(q_lens), sum(k_lens), window, sinks, ty, dim)
    q, k, v, do = inputs(key, sum(q_lens), sum(k_lens), heads, kv, dim, ty)
    check(dev, q, k, v, do, q_lens, k_lens, ty, window, sinks)


@pytest.mark.parametrize("dim", [8, 24, 40, 72, 96, 104, 120])
def test_window_head_dimensions(dev, dim):
    q, k, v, do = inputs(("dim", dim), 400, 400, 4, 2, dim, "bf16")
    check(dev, q, k, v, do, [277, 123], [277, 123], "bf16", 50, 6)


@pytest.mark.parametrize("sinks", [0, 1, 31, 32, 33, 63, 64, 65, 127, 128, 129, 300])
@pytest.mark.parametrize("ty", ["bf16", "f16"])
def test_window_sinks_about_the_tiles(dev, sinks, ty):
    """Sinks that fill tiles of 32, 64 and 128 keys, or pass them, with queries past
    their windows and, 300 of them, sequences that have not so many keys."""
    q_lens, k_lens = [700, 200, 40, 350], [700, 230, 40, 350]
    q, k, v, do = inputs(("sinks", sinks), sum(q_lens), sum(k_lens), 4, 1, 64, ty)
    check(dev, q, k, v, do, q_lens, k_lens, ty, 97, sinks)


@pytest.mark.parametrize("window", [1, 2, 31, 32, 63, 64, 65, 127, 128, 129, 191, 600, 1999, 2000])
def test_window_lengths_about_the_tiles(dev, window):
    q, k, v, do = inputs(("window", window), 601, 2001, 2, 1, 32, "bf16")
    check(dev, q, k, v, do, [300, 301], [300, 1701], "bf16", window, 5)


@pytest.mark.parametrize("sinks", [0, 5, 64])
def test_window_single_tokens_over_long_memories(dev, sinks):
    """Keys in chunks joined from partial results, over sequences that have fewer keys
    than the window and many more."""
    rng = np.random.default_rng(5)
    k_lens = [int(x) for x in rng.integers(0, 4500, 20)] + [9000, 1, 0]
    q, k, v, do = inputs(("long", sinks), 23, sum(k_lens), 8, 2, 64, "bf16")
    check(dev, q, k, v, do, [1] * 23, k_lens, "bf16", 1500, sinks)
    q_lens, k_lens = [260, 1, 90], [5000, 2000, 3]
    q, k, v, do = inputs(("chunk", sinks), 351, 7003, 4, 2, 128, "f16")
    check(dev, q, k, v, do, q_lens, k_lens, "f16", 1234, sinks)
    q, k, v, do = inputs(("wide", sinks), 200, 9000, 2, 2, 32, "bf16")
    check(dev, q, k, v, do, [200], [9000], "bf16", 5000, sinks)


@pytest.mark.parametrize("n", [62, 63, 127, 385])
def test_window_of_many_sequences(dev, n):
    rng = np.random.default_rng(n)
    q_lens, k_lens = (rng.integers(0, 6, n).tolist() for _ in range(2))
    q_lens[n // 2], k_lens[n // 2] = 350, 340
    q, k, v, do = inputs(("sequences", n), sum(q_lens), sum(k_lens), 2, 1, 32, "f16")
    check(dev, q, k, v, do, q_lens, k_lens, "f16", 30, n % 3)


@pytest.mark.parametrize("seed", range(8))
def test_window_random_packs(dev, seed):
    rng = np.random.default_rng(200 + seed)
    n = int((2, 9, 30, 61, 62, 63, 5, 80)[seed])
    most = 900 if n < 10 else 150
    q_lens = [int(x) for x in rng.integers(0, most, n)]
    k_lens = [int(x) for x in rng.integers(0, most, n)]
    if seed % 2:
        k_lens = list(q_lens)
    heads, kv, dim = ((4, 2, 64), (2, 2, 128), (3, 1, 32), (2, 1, 64))[seed % 4]
    ty = ("bf16", "f16")[seed // 4]
    window, sinks = int(rng.integers(1, most)), int(rng.integers(0, 150)) * (seed % 3 != 1)
    q, k, v, do = inputs(("packs", seed), sum(q_lens), sum(k_lens), heads, kv, dim, ty)
    check(dev, q, k, v, do, q_lens, k_lens, ty, window, sinks)


@pytest.mark.parametrize("heads,kv", [(5, 1), (7, 1), (12, 2), (2, 1), (9, 3)])
@pytest.mark.parametrize("sinks", [0, 3, 140])
def test_window_gradients_of_shared_heads_in_runs(dev, heads, kv, sinks):
    """Runs of whole heads and of parts of heads, with and without sums for sinks."""
    q_lens, k_lens = [1500, 40, 300], [1450, 300, 1]
    q, k, v, do = inputs(("runs", heads, sinks), 1840, 1751, heads, kv, 16, "bf16")
    for window in (90, 900):
        check(dev, q, k, v, do, q_lens, k_lens, "bf16", window, sinks)


@pytest.mark.parametrize("ty,heads,kv,dim", [("bf16", 4, 2, 64), ("f16", 4, 1, 128)])
@pytest.mark.parametrize("window,sinks", [(700, 3), (650, 0), (1, 130)])
def test_window_gradients_of_unequal_sequences(dev, ty, heads, kv, dim, window, sinks):
    """A long sequence's key tiles are cut into runs, short ones' are not."""
    lens = [5, 900, 1, 0, 40, 130, 7]
    n = sum(lens)
    check(dev, *inputs(("unequal", ty, window), n, n, heads, kv, dim, ty), lens, lens, ty, window,
          sinks)


def test_window_of_all_keys_is_none(dev):
    from metal_gauss_amd import attention

    q, k, v, do = (t.to(dev) for t in inputs(("all",), 300, 300, 4, 2, 64, "bf16"))
    off = torch.tensor([0, 120, 300], dtype=torch.int32, device=dev)
    want = attention(q, k, v, off, causal=True)
    for window in (300, 301, 2 ** 40):
        assert torch.equal(attention(q, k, v, off, causal=True, window=window, sinks=7), want)
    # A window of each sequence's keys, one short of all tokens: equal to rounding.
    got = attention(q, k, v, off, causal=True, window=299)
    assert float((got.float() - want.float()).abs().max()) <= 2.0 ** -6


def test_window_tokens_of_no_sequence_and_unseen_keys_may_hold_anything(dev):
    """NaN and infinities before the window, past the query, in other sequences and in
    none; the sinks' neighbours in their tile too."""
    from metal_gauss_amd import attention

    for nq, window, sinks in ((300, 50, 4), (3, 70, 0), (1, 64, 33), (120, 1, 1)):
        q, k, v, _ = (t.to(dev) for t in inputs(("unseen", nq), nq, 700, 2, 1, 64, "bf16"))
        ko = torch.tensor([10, 650], dtype=torch.int32, device=dev)
        qo = torch.tensor([0, nq], dtype=torch.int32, device=dev)
        kw = dict(causal=True, window=window, sinks=sinks)
        clean = attention(q, k, v, qo, ko, **kw)
        first = 640 - nq                        # the key at which query 0 stands
        lost = [*range(10), *range(650, 700),
                *range(10 + sinks, 10 + max(sinks, first - window + 1))]
        for fill in (float("nan"), float("inf"), 3e38):
            k[lost], v[lost] = fill, fill
            assert torch.equal(attention(q, k, v, qo, ko, **kw), clean), (nq, fill)


@pytest.mark.parametrize("ty,heads,kv,dim", [("bf16", 2, 2, 64), ("f16", 4, 1, 128)])
@pytest.mark.parametrize("nq,nk", [(400, 400), (3, 900), (90, 500)])
def test_window_values_that_are_not_finite_reach_those_who_see_them(dev, ty, heads, kv, dim, nq, nk):
    from metal_gauss_amd import attention

    q, k, v, _ = (t.to(dev) for t in inputs(("poison", nq, nk), nq, nk, heads, kv, dim, ty))
    kw = dict(causal=True, window=60, sinks=5)
    clean = attention(q, k, v, **kw).float()
    seen = torch.from_numpy(token_ref.sees(nq, nk, True, 60, 5)).to(dev)
    at = {3: (nk - nq // 2 - 1, float("inf")), 5: (4, float("-inf")), 7: (nk - 2, float("nan")),
          9: (nk - 61, float("inf")), 11: (6, float("nan"))}
    for column, (key, value) in at.items():
        v[key, :, column] = value
    got = attention(q, k, v, **kw).float()
    for column in range(dim):
        want = clean[:, :, column].clone()
        if column in at:
            key, value = at[column]
            want[seen[:, key]] = value
        assert torch.equal(got[:, :, column].isnan(), want.isnan()), column
        ok = ~want.isnan()
        assert torch.equal(got[:, :, column][ok], want[ok]), column


def test_window_falling_offsets_are_made_to_rise(dev):
    from metal_gauss_amd import attention

    q, k, v, do = (t.to(dev) for t in inputs(("fall",), 400, 500, 4, 2, 64, "f16"))
    got = []
    for rising in (False, True):
        offs = []
        for off, n in (([3, 60, 20, 300, 250, 10 ** 9], 400), ([-4, 90, 80, 450, 9, 480], 500)):
            off = np.asarray(off)
            if rising:
                off = np.maximum.accumulate(off.clip(0, n))
            offs.append(torch.tensor(off, dtype=torch.int32, device=dev))
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        o = attention(*leaves, *offs, causal=True, window=70, sinks=9)
        got.append((o, *torch.autograd.grad(o, leaves, do)))
    for a, b in zip(*got):
        assert bool(a.isfinite().all()) and torch.equal(a, b)


def test_window_strided_views(dev):
    from metal_gauss_amd import attention

    g = gen("views")
    qkv = torch.randn(320, 8, 64, generator=g).to(dev, torch.bfloat16)
    q, k, v = qkv[:, :4], qkv[:, 4:6], qkv[:, 6:]
    kw = dict(causal=True, window=40, sinks=4)
    want = attention(q.contiguous(), k.contiguous(), v.contiguous(), **kw)
    assert torch.equal(attention(q, k, v, **kw), want)
    odd = torch.empty(320 * 8 * 64 + 1, device=dev, dtype=torch.bfloat16)[1:].view(320, 8, 64)
    odd.copy_(qkv)                                               # not 16-byte aligned
    assert torch.equal(attention(odd[:, :4], odd[:, 4:6], odd[:, 6:], **kw), want)


def test_window_over_rows_whose_offsets_pass_32_bits(dev):
    """Keys and values 2^23 elements apart, in a memory of 600 of them."""
    from metal_gauss_amd import attention

    g = gen("far rows")
    far = torch.empty(600, 1 << 23, device=dev, dtype=torch.bfloat16)[:, :256].view(600, 4, 64)
    far.copy_(torch.randn(600, 4, 64, generator=g))
    q = torch.randn(600, 4, 64, generator=g).to(dev, torch.bfloat16)
    dy = torch.randn(600, 4, 64, generator=g).to(dev, torch.bfloat16)
    results = []
    for k, v in ((far[:, :2], far[:, 2:]), (far[:, :2].contiguous(), far[:, 2:].contiguous())):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        y = attention(*leaves, causal=True, window=130, sinks=5)
        results.append((y, *torch.autograd.grad(y, leaves, dy)))
        with torch.no_grad():
            results[-1] += (attention(q[-1:], k, v, causal=True, window=130, sinks=5),)
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("grad", [False, True])
def test_window_in_a_graph_and_on_another_stream(dev, grad):
    from metal_gauss_amd import attention

    nq, nk = (200, 200) if grad else (4, 6000)
    q, k, v, do = (t.to(dev) for t in inputs(("graph", grad), nq, nk, 4, 2, 64, "bf16"))
    off = [torch.tensor(o, dtype=torch.int32, device=dev) for o in
           (([0, 90, 200], [0, 90, 200]) if grad else ([0, 1, 2, 4], [0, 50, 3000, 6000]))]
    leaves = [t.requires_grad_(grad) for t in (q, k, v)]

    def step():
        o = attention(*leaves, *off, causal=True, window=60 if grad else 2000, sinks=4)
        return (o.detach(), *(torch.autograd.grad(o, leaves, do) if grad else ()))

    want = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        with torch.no_grad():
            for t in leaves:
                t.copy_(torch.randn(t.shape, generator=gen("again", i)))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_window_gradient_against_differences(dev):
    """A directional derivative of the restatement in float64, along the kernel's
    own inputs, off by what the bounds allow the products with the directions."""
    ty, n = "f16", 80
    q, k, v, do = inputs(("diff",), n, n, 2, 1, 16, ty)
    got = check(dev, q, k, v, do, [n], [n], ty, 20, 3)
    g = np.random.default_rng(3)
    X = [host(t) for t in (q, k, v)]
    at = lambda x: token_ref.attention(*x, [0, n], [0, n], True, 0.25, window=20,  # noqa: E731
                                       sinks=3)[0][0]
    _, off = token_ref.attention(*X, [0, n], [0, n], True, 0.25, host(do), UNIT[ty], 20, 3)
    for i in range(3):
        d = g.standard_normal(X[i].shape)
        up, down = list(X), list(X)
        up[i], down[i] = X[i] + 1e-5 * d, X[i] - 1e-5 * d
        num = ((at(up) - at(down)) * host(do)).sum() / 2e-5
        assert abs(num - (host(got[i + 1]) * d).sum()) <= (off[i + 1] * np.abs(d)).sum() * 1.2


def test_window_refusals(dev):
    from metal_gauss_amd import attention

    b = torch.zeros(4, 2, 64, device=dev, dtype=torch.bfloat16)
    for text, kw in (("needs causal", dict(window=3)), ("at least 1", dict(window=0, causal=True)),
                     ("at least 1", dict(window=3, sinks=-1, causal=True)),
                     ("sinks needs window", dict(sinks=2, causal=True))):
        with pytest.raises(ValueError, match=text):
            attention(b, b, b, **kw)
