"""The token operators on the GPU (layer norm, rotary positions, attention over
packed sequences) against the float64 restatements in oracle/token_ref.py.

Tolerances. With u the unit roundoff of the stored type (2^-24, 2^-8, 2^-11 for
float32, bfloat16, float16):

* norm, rotary: float32 arithmetic rounded once. A rotation's two products and
  its cosine and sine are good to a few 2^-24 of the pair's length; a row's mean
  and variance to 2^-24 of the row's largest value times the depth of the sums
  (under 32 rounded additions a lane and across lanes). 64 * 2^-24 of the row's
  largest result covers either; the rounding adds u of the value.
* the weights' gradients: sums over rows in float32, off by at most (additions a
  value passes through, under 64 + rows / 32) * 2^-24 of the sum of magnitudes.
* attention: the bound of token_ref.attention (p, ds and the results each rounded
  to the type once, every rounding at its worst), plus 2^-14 of the magnitudes
  summed for float32's part: scores of up to 40 powers of two held to 2^-24 each
  leave p exact to 40 * 2^-24 = 2^-18.7, and sums of float32 add less.
"""

from __future__ import annotations

import zlib

import numpy as np
import pytest
import torch

from oracle import token_ref

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
UNIT = {name: torch.finfo(t).eps / 2 for name, t in TYPES.items()}
EPS24 = 2.0 ** -24


def host(t):
    return t.detach().cpu().double().numpy()


def gen(*key):
    return torch.Generator().manual_seed(zlib.crc32(repr(key).encode()))


def close(got, want, bound, what=""):
    got = host(got)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = np.abs(got - want) - bound
    assert np.isfinite(got).all() and (bad <= 0).all(), \
        f"{what}: {np.abs(got - want).max():.3e} off, {bad.max():.3e} over the bound"


# -------------------------------------------------------------------- norm

NORM_SHAPES = [(1, 1), (3, 2), (5, 7), (1, 64), (64, 256), (130, 511), (130, 512), (67, 513),
               (2531, 771), (9, 1024), (33, 1025), (7, 2048), (6, 2049), (5, 4096), (3, 4097),
               (4, 8192), (2, 8193), (3, 16384), (2, 16385), (2, 20001), (70, 16386)]


def norm_inputs(rows, n, ty, wt, offset=0.0):
    g = gen(rows, n, ty, wt)
    x = (torch.randn(rows, n, generator=g) * 1.5 + offset + torch.randn(n, generator=g))
    w = 1.0 + 0.3 * torch.randn(n, generator=g)
    b = 0.3 * torch.randn(n, generator=g)
    dy = torch.randn(rows, n, generator=g)
    return x.to(TYPES[ty]), w.to(TYPES[wt]), b.to(TYPES[wt]), dy.to(TYPES[ty])


def check_norm(dev, x, w, b, dy, ty, wt, eps=1e-5, deep=64):
    from metal_gauss_amd import layer_norm

    xd, wd, bd = (t.to(dev).requires_grad_(True) for t in (x, w, b))
    y = layer_norm(xd, wd, bd, eps)
    dx, dw, db = torch.autograd.grad(y, (xd, wd, bd), dy.to(dev))
    X, W, B, DY = (host(t) for t in (x, w, b, dy))
    want = token_ref.layer_norm(X, W, B, eps)
    gx, gw, gb = token_ref.layer_norm_grad(X, W, DY, eps)
    u, uw, top = UNIT[ty], UNIT[wt], lambda t: np.abs(t).max(1, keepdims=True)
    # The mean's rounding is of the row's largest value, which the division
    # by its deviation carries over.
    m = X.mean(1, keepdims=True)
    sd = np.sqrt(((X - m) ** 2).mean(1, keepdims=True) + eps)
    lift = 1.0 + top(X) / sd
    close(y, want, u * np.abs(want) + deep * EPS24 * lift * (np.abs(W).max() + top(want)), "y")
    unit_dx = (np.abs(DY * W).max(1, keepdims=True) * (1 + np.abs((X - m) / sd).max(1, keepdims=True))) / sd
    close(dx, gx, u * np.abs(gx) + deep * EPS24 * lift * unit_dx, "dx")
    deep_w = (64 + x.shape[0] / 32) * EPS24
    U = np.abs((X - m) / sd) + lift * deep * EPS24 / deep_w
    close(dw, gw, uw * np.abs(gw) + deep_w * (np.abs(DY) * U).sum(0), "dweight")
    close(db, gb, uw * np.abs(gb) + deep_w * np.abs(DY).sum(0), "dbias")
    with torch.no_grad():
        assert torch.equal(layer_norm(xd, wd, bd, eps), y)


@pytest.mark.parametrize("rows,n", NORM_SHAPES)
@pytest.mark.parametrize("ty,wt", [("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16"),
                                   ("f16", "f16")])
def test_norm(dev, rows, n, ty, wt):
    check_norm(dev, *norm_inputs(rows, n, ty, wt), ty, wt)


def test_norm_keeps_the_variance_of_rows_far_from_zero(dev):
    check_norm(dev, *norm_inputs(20, 600, "f32", "f32", offset=300.0), "f32", "f32")


def test_norm_many_rows(dev):
    check_norm(dev, *norm_inputs(9001, 96, "f32", "f32"), "f32", "f32")


def test_norm_constant_rows_and_no_weights(dev):
    from metal_gauss_amd import layer_norm

    x = torch.full((3, 100), 7.0, device=dev, requires_grad=True)
    y = layer_norm(x)
    assert torch.equal(y, torch.zeros_like(y))
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    assert float(dx.abs().max()) < 1e-3        # 1 / sqrt(eps) times a mean's rounding
    g = gen("none")
    x = torch.randn(6, 50, generator=g).to(dev).requires_grad_(True)
    b = torch.randn(50, generator=g).to(dev).requires_grad_(True)
    y = layer_norm(x, None, b)
    dx, db = torch.autograd.grad(y, (x, b), torch.ones_like(y))
    close(y, token_ref.layer_norm(host(x), None, host(b)), 1e-5, "y")
    close(db, np.full(50, 6.0), 1e-5, "db")


def test_norm_strided_rows_and_leading_dimensions(dev):
    from metal_gauss_amd import layer_norm

    g = gen("strided")
    base = torch.randn(4, 5, 200, generator=g).to(dev)
    x = base[..., 3:103].detach().requires_grad_(True)
    dy = torch.randn(4, 5, 200, generator=g).to(dev)[..., 100:]
    y = layer_norm(x)
    dx, = torch.autograd.grad(y, x, dy)
    want = token_ref.layer_norm(host(x).reshape(20, 100)).reshape(4, 5, 100)
    close(y, want, 1e-5, "y")
    gx = token_ref.layer_norm_grad(host(x).reshape(20, 100), None, host(dy).reshape(20, 100))[0]
    close(dx, gx.reshape(4, 5, 100), 2e-5, "dx")
    rows = base.reshape(20, 200)[:, 7:]         # rows 200 apart, unaligned
    close(layer_norm(rows), token_ref.layer_norm(host(rows)), 1e-5, "rows")
    columns = base.reshape(20, 200).t()         # a copy is made
    close(layer_norm(columns), token_ref.layer_norm(host(columns)), 1e-5, "columns")
    # A broadcast gradient and a broadcast input.
    one = base[0, :1].expand(5, 200)
    close(layer_norm(one), token_ref.layer_norm(host(one)), 1e-5, "expanded")
    x2 = base[0].detach().requires_grad_(True)
    d2, = torch.autograd.grad(layer_norm(x2).sum(), x2)
    assert float(d2.abs().max()) < 1e-4


def test_norm_of_no_rows(dev):
    from metal_gauss_amd import layer_norm

    x = torch.zeros(0, 32, device=dev, requires_grad=True)
    w = torch.ones(32, device=dev, requires_grad=True)
    y = layer_norm(x, w)
    dx, dw = torch.autograd.grad(y.sum(), (x, w))
    assert y.shape == (0, 32) and dx.shape == (0, 32)
    assert torch.equal(dw, torch.zeros_like(dw))


def test_norm_nan_stays_in_its_row(dev):
    from metal_gauss_amd import layer_norm

    x = torch.randn(8, 300, generator=gen("nan")).to(dev)
    clean = layer_norm(x)
    x[3, 299] = float("nan")
    x[5, 0] = float("inf")
    y = layer_norm(x)
    for r in range(8):
        assert torch.equal(y[r], clean[r]) if r not in (3, 5) else bool(y[r].isnan().all())


def test_norm_gradient_against_differences(dev):
    """Central differences of the restatement, with a step of 1e-5 in float64: off
    by its square and by float32 in the gradient."""
    g = gen("differences")
    x, dy = torch.randn(2, 37, generator=g), torch.randn(2, 37, generator=g)
    from metal_gauss_amd import layer_norm

    xd = x.to(dev).requires_grad_(True)
    dx, = torch.autograd.grad(layer_norm(xd), xd, dy.to(dev))
    X, DY, num = host(x), host(dy), np.zeros((2, 37))
    for i in range(37):
        for r in range(2):
            e = np.zeros((2, 37))
            e[r, i] = 1e-5
            num[r, i] = ((token_ref.layer_norm(X + e) - token_ref.layer_norm(X - e)) * DY).sum() / 2e-5
    close(dx, num, 1e-5, "dx")


# ------------------------------------------------------------------ rotary

@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("ty", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("tokens,heads,kv,dim,part,axes", [
    (1, 1, 1, 2, 2, 1), (1, 4, 1, 64, 64, 1), (16, 16, 4, 64, 64, 1), (7, 3, 2, 128, 64, 2),
    (33, 5, 5, 96, 96, 3), (9, 2, 1, 80, 40, 2), (5, 3, 1, 30, 10, 1), (11, 1, 0, 66, 66, 1),
    (2100, 4, 2, 32, 32, 1), (3, 2, 2, 1024, 1024, 1), (4, 2, 1, 48, 16, 1)])
def test_rotary(dev, layout, ty, tokens, heads, kv, dim, part, axes):
    from metal_gauss_amd import rotary, rotary_frequencies

    g = gen(layout, ty, tokens, dim, part)
    q = torch.randn(tokens, heads, dim, generator=g).to(TYPES[ty])
    k = torch.randn(tokens, kv, dim, generator=g).to(TYPES[ty]) if kv else None
    dq = torch.randn(tokens, heads, dim, generator=g).to(TYPES[ty])
    pos = torch.randint(-5, 3000, (tokens, axes), generator=g, dtype=torch.int32)
    freq = rotary_frequencies(part, axes=axes, device=dev)
    qd = q.to(dev).requires_grad_(True)
    kd = k.to(dev).requires_grad_(True) if kv else None
    p = (pos if axes > 1 else pos[:, 0]).to(dev)
    out = rotary(qd, kd, p, freq, layout=layout)
    qo, ko = out if kv else (out, None)
    F, P, u = host(freq), pos.numpy(), UNIT[ty]

    def bound(x, want):
        return u * np.abs(want) + 64 * EPS24 * np.abs(x).max()

    want = token_ref.rotary(host(q), P, F, layout)
    close(qo, want, bound(host(q), want), "q")
    if kv:
        want = token_ref.rotary(host(k), P, F, layout)
        close(ko, want, bound(host(k), want), "k")
    want = token_ref.rotary(host(dq), P, F, layout, inverse=True)
    grads = torch.autograd.grad(qo, qd, dq.to(dev), retain_graph=True)
    close(grads[0], want, bound(host(dq), want), "dq")
    if kv:
        both = torch.autograd.grad((qo, ko), (qd, kd), (dq.to(dev), torch.ones_like(ko)))
        assert torch.equal(both[0], grads[0])
        want = token_ref.rotary(np.ones(ko.shape), P, F, layout, inverse=True)
        close(both[1], want, bound(np.ones(1), want), "dk")


@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_rotary_far_positions(dev, kind):
    """Angles of 10^9 radians are as exact as those of 10: the product's whole
    turns leave in float64 (2^-53 of 2^30 is 2^-23 of a turn at most)."""
    from metal_gauss_amd import rotary, rotary_frequencies

    q = torch.randn(6, 2, 64, generator=gen("far")).to(dev)
    pos = torch.tensor([0, 1, 131071, 10 ** 6, 2 ** 30, -(2 ** 30)], dtype=kind)
    freq = rotary_frequencies(64, device=dev)
    got = rotary(q, None, pos.to(dev), freq)
    want = token_ref.rotary(host(q), pos.numpy()[:, None], host(freq), "half")
    close(got, want, 64 * EPS24 * np.abs(host(q)).max() + 2.0 ** -20, "q")


def test_rotary_slices_of_a_projection(dev):
    from metal_gauss_amd import rotary, rotary_frequencies

    qkv = torch.randn(50, 10, 66, generator=gen("slices")).to(dev)
    q, k = qkv[:, :6, :64], qkv[:, 6:8, :64]
    pos = torch.arange(50, dtype=torch.int32, device=dev)
    freq = rotary_frequencies(64, device=dev)
    qo, ko = rotary(q, k, pos, freq)
    q2, k2 = rotary(q.contiguous(), k.contiguous(), pos, freq)
    assert torch.equal(qo, q2) and torch.equal(ko, k2)
    t = torch.randn(64, 6, 50, generator=gen("t")).to(dev).permute(2, 1, 0)
    assert torch.equal(rotary(t, None, pos, freq), rotary(t.contiguous(), None, pos, freq))
    empty = rotary(q[:0], k[:0], pos[:0], freq)
    assert empty[0].shape == (0, 6, 64) and empty[1].shape == (0, 2, 64)


def test_rotary_gradient_of_one_output(dev):
    from metal_gauss_amd import rotary, rotary_frequencies

    q = torch.randn(8, 2, 32, generator=gen(1)).to(dev).requires_grad_(True)
    k = torch.randn(8, 1, 32, generator=gen(2)).to(dev).requires_grad_(True)
    pos = torch.arange(8, dtype=torch.int32, device=dev)
    freq = rotary_frequencies(32, device=dev)
    qo, ko = rotary(q, k, pos, freq)
    dk, = torch.autograd.grad(ko.sum(), k)
    want = token_ref.rotary(np.ones((8, 1, 32)), np.arange(8)[:, None], host(freq), "half", True)
    close(dk, want, 64 * EPS24, "dk")


# --------------------------------------------------------------- attention

def offsets(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(int).tolist()


def attn_inputs(key, nq, nk, heads, kv, dim, ty, gain=1.0):
    g = gen(*key)
    t = [torch.randn(n, h, dim, generator=g) for n, h in ((nq, heads), (nk, kv), (nk, kv),
                                                          (nq, heads))]
    t[0] = t[0] * gain
    return [x.to(TYPES[ty]) for x in t]


def check_attention(dev, q, k, v, do, q_lens, k_lens, ty, causal, grad=True, scale=None):
    from metal_gauss_amd import attention

    qo, ko = offsets(q_lens), offsets(k_lens)
    put = [torch.tensor(o, dtype=torch.int32, device=dev) for o in (qo, ko)]
    leaves = [t.to(dev).requires_grad_(grad) for t in (q, k, v)]
    o = attention(*leaves, *put, causal=causal, scale=scale)
    real = scale if scale is not None else q.shape[2] ** -0.5
    want, off = token_ref.attention(host(q), host(k), host(v), qo, ko, causal, real,
                                    host(do) if grad else None, UNIT[ty])
    # float32's share, and the spacing of float16 below 2^-14.
    tiny = 2.0 ** -24 if ty == "f16" else 1e-30
    names, got = ("o", "dq", "dk", "dv"), [o]
    if grad:
        got += torch.autograd.grad(o, leaves, do.to(dev))
        with torch.no_grad():
            assert torch.equal(attention(*leaves, *put, causal=causal, scale=scale), o)
    for name, g, w, b in zip(names, got, want, off):
        close(g, w, b * (1.0 + 2.0 ** -14 / UNIT[ty]) * 1.05 + tiny, name)
    return got


PACKS = [
    ([1], [1]), ([2], [3]), ([64], [64]), ([65], [65]), ([128, 1, 63], [128, 1, 63]),
    ([200, 31, 300, 0, 5], [200, 31, 300, 0, 5]),
    ([1, 1, 1, 1], [1, 700, 64, 129]),              # single tokens over memories
    ([17, 100, 3], [300, 100, 500]),                # chunks over memories
    ([100, 5, 70], [30, 5, 1]),                     # more queries than keys
    ([10, 0, 20], [0, 12, 20]),                     # no keys, no queries
]


@pytest.mark.parametrize("q_lens,k_lens", PACKS)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("ty,heads,kv,dim", [("bf16", 4, 2, 64), ("f16", 6, 2, 128),
                                             ("bf16", 3, 3, 32), ("f16", 5, 1, 80)])
def test_attention(dev, q_lens, k_lens, causal, ty, heads, kv, dim):
    key = (sum(q_lens), sum(k_lens), causal, ty, dim)
    q, k, v, do = attn_inputs(key, sum(q_lens), sum(k_lens), heads, kv, dim, ty)
    check_attention(dev, q, k, v, do, q_lens, k_lens, ty, causal)


@pytest.mark.parametrize("dim", [8, 16, 24, 40, 48, 72, 88, 96, 104, 112, 120])
def test_attention_head_dimensions(dev, dim):
    q, k, v, do = attn_inputs(("dim", dim), 140, 140, 4, 2, dim, "bf16")
    check_attention(dev, q, k, v, do, [77, 63], [77, 63], "bf16", True)


@pytest.mark.parametrize("ty", ["bf16", "f16"])
@pytest.mark.parametrize("gain", [0.0, 8.0, 300.0])
def test_attention_flat_and_sharp_rows(dev, ty, gain):
    """Equal scores, and scores whose running maximum keeps rising by more than
    the lag that leaves the accumulators as they are."""
    from metal_gauss_amd import attention

    q, k, v, do = attn_inputs(("gain", gain), 150, 400, 2, 1, 64, ty, gain)
    ramp = torch.linspace(0.0, 1.0, 400)[:, None, None]
    k = (k.float() * ramp).to(k.dtype)
    if gain <= 8.0:
        check_attention(dev, q, k, v, do, [150], [400], ty, True)
    else:
        # Scores of thousands have float32 errors of their own: each row is
        # still a mean of values.
        o = attention(*(t.to(dev) for t in (q, k, v))).cpu().float()
        lo, hi = v.float().amin(0), v.float().amax(0)
        assert bool(((o >= lo * (1 + 2.0 ** -7) - 0.1) & (o <= hi * (1 + 2.0 ** -7) + 0.1)).all())


@pytest.mark.parametrize("scale", [0.0, 0.02, 1.0])
def test_attention_scales(dev, scale):
    q, k, v, do = attn_inputs(("scale", scale), 90, 90, 2, 2, 32, "bf16")
    check_attention(dev, q, k, v, do, [90], [90], "bf16", False, scale=scale)


def test_attention_long_memory_of_few_rows(dev):
    """Keys in chunks joined from partial results, ragged and over 64 sequences."""
    rng = np.random.default_rng(5)
    k_lens = [int(x) for x in rng.integers(0, 2500, 20)] + [4000, 1, 0]
    q_lens = [1] * 23
    q, k, v, do = attn_inputs(("long",), 23, sum(k_lens), 8, 2, 64, "bf16")
    check_attention(dev, q, k, v, do, q_lens, k_lens, "bf16", True)
    q_lens, k_lens = [1] * 150, [int(x) for x in rng.integers(0, 300, 150)]
    q, k, v, do = attn_inputs(("many",), 150, sum(k_lens), 4, 4, 32, "f16")
    check_attention(dev, q, k, v, do, q_lens, k_lens, "f16", False)
    q_lens, k_lens = [260, 1, 90], [3000, 2000, 5]
    q, k, v, do = attn_inputs(("chunk",), 351, 5005, 4, 2, 128, "f16")
    check_attention(dev, q, k, v, do, q_lens, k_lens, "f16", True)


@pytest.mark.parametrize("n", [62, 63, 64, 127, 385, 4094, 4095, 4300])
def test_attention_of_many_sequences(dev, n):
    """Sequences found in one step of 64, in several, and in many."""
    rng = np.random.default_rng(n)
    q_lens, k_lens = (rng.integers(0, 4, n).tolist() for _ in range(2))
    q_lens[n // 2], k_lens[n // 2] = 150, 140
    q, k, v, do = attn_inputs(("sequences", n), sum(q_lens), sum(k_lens), 2, 1, 32, "f16")
    check_attention(dev, q, k, v, do, q_lens, k_lens, "f16", n % 2 == 1)


@pytest.mark.parametrize("causal", [False, True])
def test_attention_chunks_of_very_unequal_sequences(dev, causal):
    """One of many sequences holds nearly all queries and keys: its chunks of the
    length that suits the average find no room, and grow."""
    q_lens, k_lens = [1] * 39 + [250], [3 + i for i in range(39)] + [36001]   # narrow items
    q, k, v, do = attn_inputs(("unequal", 1), sum(q_lens), sum(k_lens), 8, 1, 64, "bf16")
    check_attention(dev, q, k, v, do, q_lens, k_lens, "bf16", causal, grad=False)
    q_lens = [700] + [1] * 69                     # narrow, over 64 sequences
    k_lens = [60001] + [5] * 69
    q, k, v, do = attn_inputs(("unequal", 2), sum(q_lens), sum(k_lens), 1, 1, 40, "f16")
    check_attention(dev, q, k, v, do, q_lens, k_lens, "f16", causal, grad=False)
    q_lens, k_lens = [5] * 6 + [2900] + [3] * 5, [7] * 6 + [11900] + [0] * 5   # wide items
    q, k, v, do = attn_inputs(("unequal", 3), sum(q_lens), sum(k_lens), 2, 2, 128, "f16")
    check_attention(dev, q, k, v, do, q_lens, k_lens, "f16", causal, grad=False)


@pytest.mark.parametrize("q_lens,k_lens,heads,kv", [
    ([1] * 40, [64] * 39 + [16320], 4, 1),            # one long memory: narrow, whole
    ([1] * 100, [9000, 1, 0] + [30] * 97, 8, 8),      # items enough by their number alone
    ([2000] + [1] * 63, [2000] + [40] * 63, 1, 1),    # a prompt in narrow items
    ([1] * 10 + [900], [3] * 10 + [5000], 2, 1)],     # wide, whole
    ids=["streams", "heads", "prompt", "chunk"])
@pytest.mark.parametrize("ty", ["bf16", "f16"])
def test_attention_unequal_sequences_that_are_not_cut(dev, q_lens, k_lens, heads, kv, ty):
    """Packs whose average sequence is too short to cut any over its keys."""
    q, k, v, do = attn_inputs(("uncut", heads, kv), sum(q_lens), sum(k_lens), heads, kv, 64, ty)
    check_attention(dev, q, k, v, do, q_lens, k_lens, ty, True)


@pytest.mark.parametrize("seed", range(8))
def test_attention_random_packs(dev, seed):
    """Every tile of every sequence is given out once, in whatever order: up to 80
    sequences (62 are ordered by length, more are not) of any two lengths."""
    rng = np.random.default_rng(100 + seed)
    n = int((3, 9, 30, 61, 62, 63, 64, 80)[seed])
    most = 900 if n < 10 else 150
    q_lens = [int(x) for x in rng.integers(0, most, n)]
    k_lens = [int(x) for x in rng.integers(0, most, n)]
    if seed % 2:
        k_lens = list(q_lens)
    heads, kv, dim = ((4, 2, 64), (2, 2, 128), (3, 1, 32), (2, 1, 64))[seed % 4]
    ty = ("bf16", "f16")[seed // 4]
    q, k, v, do = attn_inputs(("packs", seed), sum(q_lens), sum(k_lens), heads, kv, dim, ty)
    check_attention(dev, q, k, v, do, q_lens, k_lens, ty, bool(seed % 3))


@pytest.mark.parametrize("heads,kv", [(5, 1), (6, 1), (7, 1), (11, 1), (12, 2), (2, 1), (9, 3)])
def test_attention_gradients_of_shared_heads_in_runs(dev, heads, kv):
    """The keys' gradients in runs of whole heads, of parts of heads, and of heads
    that no number of runs divides."""
    q_lens, k_lens = [700, 40, 300], [650, 300, 1]
    q, k, v, do = attn_inputs(("runs", heads), 1040, 951, heads, kv, 16, "bf16")
    for causal in (False, True):
        check_attention(dev, q, k, v, do, q_lens, k_lens, "bf16", causal)


def test_attention_one_sequence_without_offsets(dev):
    from metal_gauss_amd import attention

    q, k, v, _ = (t.to(dev) for t in attn_inputs(("none",), 70, 300, 4, 2, 64, "bf16"))
    off = [torch.tensor([0, n], dtype=torch.int32, device=dev) for n in (70, 300)]
    for causal in (False, True):
        assert torch.equal(attention(q, k, v, causal=causal),
                           attention(q, k, v, *off, causal=causal))
    q, k, v, _ = (t.to(dev) for t in attn_inputs(("self",), 90, 90, 4, 2, 64, "bf16"))
    off = torch.tensor([0, 40, 90], dtype=torch.int32, device=dev)
    assert torch.equal(attention(q, k, v, off), attention(q, k, v, off, off))


def test_attention_tokens_of_no_sequence_get_zeros(dev):
    from metal_gauss_amd import attention

    q, k, v, do = (t.to(dev) for t in attn_inputs(("gap",), 300, 280, 4, 2, 64, "bf16"))
    inner = attention(q[20:220], k[10:200], v[10:200])
    for t in (q, k, v, do):                      # nothing of them is looked at
        n = t.shape[0]
        t[:10], t[n - 60:] = float("nan"), float("nan")
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    qo = torch.tensor([20, 220], dtype=torch.int32, device=dev)
    ko = torch.tensor([10, 200], dtype=torch.int32, device=dev)
    o = attention(*leaves, qo, ko)
    assert torch.equal(o[20:220], inner)
    grads = torch.autograd.grad(o, leaves, do)
    for t, a, b in ((o, 20, 220), (grads[0], 20, 220), (grads[1], 10, 200), (grads[2], 10, 200)):
        assert bool((t[:a] == 0).all()) and bool((t[b:] == 0).all())
        assert bool(t[a:b].isfinite().all())


def test_attention_offsets_are_held_to_the_tensors(dev):
    """Offsets out of range or falling give some result and read nothing else:
    the clamped offsets' result where they are a range."""
    from metal_gauss_amd import attention

    q, k, v, _ = (t.to(dev) for t in attn_inputs(("held",), 100, 100, 2, 2, 32, "bf16"))
    wild = torch.tensor([-5, 40, 10 ** 9], dtype=torch.int32, device=dev)
    held = torch.tensor([0, 40, 100], dtype=torch.int32, device=dev)
    assert torch.equal(attention(q, k, v, wild), attention(q, k, v, held))
    fall = torch.tensor([0, 100, 0, 100, 0, 100], dtype=torch.int32, device=dev)
    assert attention(q, k, v, fall).shape == q.shape


FALLING = [   # queries' tokens and offsets, keys'
    (100, [0, 60, 20, 100], 100, [0, 60, 20, 100]),
    (300, [300, 0, 300, 0, 300], 280, [0, 280, 0, 280, 0]),          # all in one, or none
    (50, [7, 3, -9, 40, 39, 10 ** 9, 5], 9000, [20, 8000, 7000, 8500, 0, 8600, 1]),   # few, many keys
    (400, [0, 10, 390, 2, 395], 9000, [9, 1, 8000, 0, 7000]),
]


@pytest.mark.parametrize("tokens_q,q_off,tokens_k,k_off", FALLING)
@pytest.mark.parametrize("ty", ["bf16", "f16"])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_offsets_that_fall_are_made_to_rise(dev, tokens_q, q_off, tokens_k, k_off, ty,
                                                      causal):
    check_falling_offsets(dev, tokens_q, q_off, tokens_k, k_off, ty, causal)


@pytest.mark.parametrize("n", [61, 62, 63, 64, 126, 127, 200])
def test_attention_offsets_of_many_sequences_that_fall(dev, n):
    """The rise goes on from one step of 64 sequences to the next."""
    rng = np.random.default_rng(n)
    offs = [np.sort(rng.integers(0, 3000, n + 1)) + rng.integers(-200, 200, n + 1)
            for _ in range(2)]
    offs[0][n // 3], offs[1][n // 2] = 2950, 2900      # most that follow lie below
    check_falling_offsets(dev, 3000, offs[0], 3000, offs[1], "f16", n % 2 == 0)


def check_falling_offsets(dev, tokens_q, q_off, tokens_k, k_off, ty, causal):
    """Result and gradients are, bit for bit, those of the offsets' running maximum,
    held to the tensors."""
    from metal_gauss_amd import attention

    q, k, v, do = (t.to(dev) for t in attn_inputs(("fall", tokens_q, tokens_k), tokens_q, tokens_k,
                                                  4, 2, 64, ty))
    got = []
    for rising in (False, True):
        offs = []
        for off, tokens in ((q_off, tokens_q), (k_off, tokens_k)):
            off = np.asarray(off)
            if rising:
                off = np.maximum.accumulate(off.clip(0, tokens))
            offs.append(torch.tensor(off, dtype=torch.int32, device=dev))
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        o = attention(*leaves, *offs, causal=causal)
        got.append((o, *torch.autograd.grad(o, leaves, do)))
        with torch.no_grad():
            assert torch.equal(attention(*leaves, *offs, causal=causal), o)
    for a, b in zip(*got):
        assert bool(a.isfinite().all()) and torch.equal(a, b)


def test_attention_unseen_keys_may_hold_anything(dev):
    """NaN and infinities in keys and values that the mask leaves out, in their own
    sequence and in its neighbours'."""
    from metal_gauss_amd import attention

    q, k, v, _ = (t.to(dev) for t in attn_inputs(("unseen",), 100, 100, 2, 2, 64, "bf16"))
    off = torch.tensor([0, 50, 100], dtype=torch.int32, device=dev)
    clean = attention(q, k, v, off, causal=True)
    k[49], k[99] = float("nan"), float("inf")
    v[99] = 3e38
    got = attention(q, k, v, off, causal=True)
    rows = [*range(49), *range(50, 99)]
    assert torch.equal(got[rows], clean[rows])
    v[:50] = float("nan")
    got = attention(q, k, v, off, causal=True)
    assert torch.equal(got[50:99], clean[50:99])


@pytest.mark.parametrize("ty,heads,kv,dim", [("bf16", 2, 2, 64), ("f16", 4, 1, 128),
                                             ("bf16", 1, 1, 32)])
@pytest.mark.parametrize("nq,nk", [(200, 200), (3, 700), (90, 300)])
def test_attention_values_that_are_not_finite_reach_those_who_see_them(dev, ty, heads, kv, dim,
                                                                       nq, nk):
    from metal_gauss_amd import attention

    q, k, v, _ = (t.to(dev) for t in attn_inputs(("poison", nq, nk), nq, nk, heads, kv, dim, ty))
    clean = attention(q, k, v, causal=True).float()
    first = nk - nq                  # the key at which query 0 stands
    plus, minus, nan = first + nq // 3, first + nq // 2, first + nq - 1
    v[plus, :, 3], v[minus, :, 3], v[minus, :, 5], v[nan, :, 7] = (
        float("inf"), float("-inf"), float("-inf"), float("nan"))
    got = attention(q, k, v, causal=True).float()
    stands = torch.arange(nq, device=dev) + first
    for column in range(dim):
        want = clean[:, :, column].clone()
        if column == 3:              # of three queries both stand at one key
            want[stands >= plus] = float("inf")
            want[stands >= minus] = float("nan" if plus != minus else "-inf")
        elif column == 5:
            want[stands >= minus] = float("-inf")
        elif column == 7:
            want[stands >= nan] = float("nan")
        assert torch.equal(got[:, :, column].isnan(), want.isnan()), column
        fine = want.isfinite()
        assert torch.equal(got[:, :, column][~fine & ~want.isnan()], want[~fine & ~want.isnan()])
        # The finite part is the same products in the same order.
        assert torch.equal(got[:, :, column][fine], want[fine]), column


def test_attention_in_a_graph(dev):
    """A token step captured once and replayed on new inputs, with eager work
    between: chunks of keys and their joining allocate nothing and clear nothing."""
    from metal_gauss_amd import attention, layer_norm, rotary, rotary_frequencies

    g = gen("graph")
    q = torch.randn(4, 8, 64, generator=g).to(dev, torch.bfloat16)
    kv = torch.randn(9000, 2, 2, 64, generator=g).to(dev, torch.bfloat16)
    pos = torch.arange(4, dtype=torch.int32, device=dev)
    freq = rotary_frequencies(64, device=dev)
    qo = torch.arange(5, dtype=torch.int32, device=dev)
    ko = torch.tensor([0, 3000, 3100, 8990, 9000], dtype=torch.int32, device=dev)

    def step():
        x = rotary(layer_norm(q), None, pos, freq)
        return attention(x, kv[:, 0], kv[:, 1], qo, ko, causal=True)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        q.copy_(torch.randn(4, 8, 64, generator=g))
        kv.copy_(torch.randn(9000, 2, 2, 64, generator=g))
        graph.replay()
        got = out.clone()
        torch.cuda.synchronize()
        assert torch.equal(got, step())


def test_attention_strided_views_and_broadcast_heads(dev):
    from metal_gauss_amd import attention

    g = gen("views")
    qkv = torch.randn(120, 8, 64, generator=g).to(dev, torch.bfloat16)
    q, k, v = qkv[:, :4], qkv[:, 4:6], qkv[:, 6:]
    want = attention(q.contiguous(), k.contiguous(), v.contiguous(), causal=True)
    assert torch.equal(attention(q, k, v, causal=True), want)
    flip = qkv.transpose(0, 1).contiguous().transpose(0, 1)      # heads outermost
    assert torch.equal(attention(flip[:, :4], flip[:, 4:6], flip[:, 6:], causal=True), want)
    odd = torch.randn(120 * 8 * 64 + 1, generator=g).to(dev, torch.bfloat16)[1:]
    odd = odd.view(120, 8, 64)                                   # not 16-byte aligned
    odd.copy_(qkv)
    assert torch.equal(attention(odd[:, :4], odd[:, 4:6], odd[:, 6:], causal=True), want)
    one_k = k[:, :1].detach().requires_grad_(True)
    one_v = v[:, :1].detach().requires_grad_(True)
    shared = attention(q, one_k, one_v)
    spread = attention(q, one_k.expand(-1, 4, -1), one_v.expand(-1, 4, -1))
    # One key head for all, and the same head four times: equal to rounding.
    a = torch.autograd.grad(shared, (one_k, one_v), torch.ones_like(shared))
    b = torch.autograd.grad(spread, (one_k, one_v), torch.ones_like(spread))
    assert float((shared.float() - spread.float()).abs().max()) <= 2.0 ** -7
    for x, y in zip(a, b):
        assert float((x.float() - y.float()).norm() / x.float().norm()) < 0.03


def test_attention_on_another_stream(dev):
    from metal_gauss_amd import attention

    q, k, v, do = (t.to(dev) for t in attn_inputs(("stream",), 500, 500, 4, 2, 64, "bf16"))
    want = attention(q, k, v, causal=True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = attention(q, k, v, causal=True)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)


def test_attention_gradient_against_differences(dev):
    """A directional derivative of the restatement in float64, along the kernel's
    own inputs: the products of the gradients with the directions, off by what
    the bounds allow them."""
    ty, n = "f16", 48
    q, k, v, do = attn_inputs(("diff",), n, n, 2, 1, 16, ty)
    got = check_attention(dev, q, k, v, do, [n], [n], ty, True)
    g = np.random.default_rng(3)
    X = [host(t) for t in (q, k, v)]

    def value(at):
        return (token_ref.attention(*at, [0, n], [0, n], True, 0.25)[0][0] * host(do)).sum()

    _, off = token_ref.attention(*X, [0, n], [0, n], True, 0.25, host(do), UNIT[ty])
    for i in range(3):
        d = g.standard_normal(X[i].shape)
        up, down = list(X), list(X)
        up[i], down[i] = X[i] + 1e-5 * d, X[i] - 1e-5 * d
        num = (value(up) - value(down)) / 2e-5
        assert abs(num - (host(got[i + 1]) * d).sum()) <= (off[i + 1] * np.abs(d)).sum() * 1.2


def test_attention_float16_small_gradients(dev):
    """Gradients of 1e-3 over 3000 keys: p and ds have almost no digits in
    float16 as they are, and their results have."""
    q, k, v, do = attn_inputs(("small",), 64, 3000, 2, 1, 64, "f16")
    check_attention(dev, q, k, v, (do.float() * 1e-3).half(), [64], [3000], "f16", False)


@pytest.mark.parametrize("fill", [6e4, float("inf"), float("nan")])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_float16_gradients_without_tokens_of_no_sequence(dev, fill, causal):
    """The unused ends of the tensors hold anything: the powers of two that float16's
    ds is taken by come of the sequences' own tokens."""
    from metal_gauss_amd import attention

    q, k, v, do = (t.to(dev) for t in attn_inputs(("ends",), 300, 3100, 4, 2, 64, "f16"))
    do *= 1e-3
    off = [torch.tensor(o, dtype=torch.int32, device=dev) for o in ([20, 90, 220], [10, 80, 3010])]
    got = []
    for value in (0.0, fill):
        for t, a, b in ((q, 20, 220), (k, 10, 3010), (v, 10, 3010), (do, 20, 220)):
            t[:a], t[b:] = value, value
        leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v)]
        o = attention(*leaves, *off, causal=causal)
        got.append((o, *torch.autograd.grad(o, leaves, do)))
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_attention_float16_gradients_of_sequences_and_rows_of_unlike_size(dev):
    """Gradients of 1e-3 packed with others of 1e3, in another sequence and (their own
    gradients, the queries') in other rows of theirs."""
    q_lens, k_lens = [64, 70, 33], [3000, 300, 500]
    q, k, v, do = attn_inputs(("unlike",), 167, 3800, 2, 1, 64, "f16")
    size = torch.full((167, 1, 1), 1e-3)
    size[64:134], size[140:150] = 1e3, 1e3
    check_attention(dev, q, k, v, (do.float() * size).half(), q_lens, k_lens, "f16", False)


@pytest.mark.parametrize("q_lens,k_lens", [([16], [16000]), ([100], [16000]),
                                           ([16] + [1] * 39, [16000] + [1] * 39),
                                           ([900] + [1] * 21, [16000] + [1] * 21)],
                         ids=["narrow-split", "wide-split", "narrow-whole", "wide-whole"])
@pytest.mark.parametrize("ty", ["f16", "bf16"])
@pytest.mark.parametrize("bits", [18, 22, 24])
@pytest.mark.parametrize("where", [0, 40, 15999])
def test_attention_many_keys_far_below_one(dev, ty, q_lens, k_lens, bits, where):
    """One key whose value is zero, and 15999 others of 1.37 * 2^-bits of its
    weight, which make the result: their weights keep the digits of the type
    (float16's own end at 2^-14, and the kernels take them 2^11 times as large)."""
    nq, nk = sum(q_lens), sum(k_lens)
    q, k, v, do = attn_inputs(("far", bits, where), nq, nk, 2, 1, 64, "f32")
    q, k, v = 2.0 + 0.05 * q, 0.02 * k, 1.0 + 0.1 * v
    k[where] = (bits * np.log(2.0) - np.log(1.37)) / 16.0      # a score of 16 times that
    v[where] = 0.0
    q, k, v, do = (t.to(TYPES[ty]) for t in (q, k, v, do))
    check_attention(dev, q, k, v, do, q_lens, k_lens, ty, False, grad=nq < 200)


def test_attention_of_nothing(dev):
    from metal_gauss_amd import attention

    e = torch.empty(0, 2, 64, device=dev, dtype=torch.bfloat16)
    q = torch.ones(3, 2, 64, device=dev, dtype=torch.bfloat16, requires_grad=True)
    assert attention(e, e, e).shape == (0, 2, 64)
    o = attention(q, e, e)
    assert bool((o == 0).all())
    dq, = torch.autograd.grad(o.sum(), q)
    assert bool((dq == 0).all())
    k = torch.ones(3, 2, 64, device=dev, dtype=torch.bfloat16, requires_grad=True)
    o = attention(e, k, k)
    dk, = torch.autograd.grad(o.sum(), k)
    assert bool((dk == 0).all())


def test_saved_tensors_may_come_back_in_another_layout(dev):
    """Hooks on saved tensors (they offload, or pack) keep values, not strides."""
    from metal_gauss_amd import attention, layer_norm, rotary, rotary_frequencies

    def spread(t):
        """t's values with gaps between all elements."""
        wide = torch.full((*t.shape, 3), 7, dtype=t.dtype, device=t.device)
        wide[..., 1] = t
        return wide[..., 1]

    g = gen("hooks")
    q, k, v = (torch.randn(90, h, 32, generator=g).to(dev, torch.bfloat16).requires_grad_(True)
               for h in (4, 2, 2))
    x = torch.randn(9, 40, generator=g).to(dev).requires_grad_(True)
    w, b = (torch.randn(40, generator=g).to(dev).requires_grad_(True) for _ in range(2))
    off = torch.tensor([0, 33, 90], dtype=torch.int32, device=dev)
    pos = torch.arange(90, dtype=torch.int32, device=dev)
    freq = rotary_frequencies(32, device=dev)
    calls = [(lambda: attention(q, k, v, off, causal=True), (q, k, v)),
             (lambda: layer_norm(x, w, b), (x, w, b)),
             (lambda: torch.cat(rotary(q, k, pos, freq), 1), (q, k))]
    for call, leaves in calls:
        y = call()
        dy = torch.randn(y.shape, generator=g).to(y)
        want = torch.autograd.grad(y, leaves, dy)
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, spread):
            y = call()
        got = torch.autograd.grad(y, leaves, dy)
        assert all(torch.equal(a, c) for a, c in zip(got, want))


# ---------------------------------------------------------------- refusals

def test_refusals(dev):
    from metal_gauss_amd import attention, layer_norm, rotary, rotary_frequencies

    f = rotary_frequencies(64, device=dev)
    x = torch.zeros(4, 2, 64, device=dev)
    b = x.bfloat16()
    pos = torch.zeros(4, dtype=torch.int32, device=dev)
    off = torch.tensor([0, 4], dtype=torch.int32, device=dev)
    bad = [
        (RuntimeError, "must be a HIP", lambda: layer_norm(torch.zeros(3, 4))),
        (RuntimeError, "float32, bfloat16 or float16", lambda: layer_norm(x.double())),
        (ValueError, "weight must have shape", lambda: layer_norm(x, torch.ones(63, device=dev))),
        (ValueError, "one type", lambda: layer_norm(x, f.float().repeat(2), b[0, 0])),
        (RuntimeError, "weights must be float32", lambda: layer_norm(b, b[0, 0].half())),
        (ValueError, "at least one element", lambda: layer_norm(x[..., :0])),
        (ValueError, "tokens, heads, dim", lambda: rotary(x[0], None, pos, f)),
        (ValueError, "unknown layout", lambda: rotary(x, None, pos, f, layout="other")),
        (RuntimeError, "int32 or int64", lambda: rotary(x, None, pos.float(), f)),
        (ValueError, "positions must be", lambda: rotary(x, None, pos[:3], f)),
        (RuntimeError, "float64", lambda: rotary(x, None, pos, f.float())),
        (RuntimeError, "frequencies turn", lambda: rotary(x[..., :32], None, pos, f)),
        (RuntimeError, "do not divide", lambda: rotary(x, None, pos[:, None].expand(4, 3), f)),
        (ValueError, "must match q's", lambda: rotary(x, b, pos, f)),
        (RuntimeError, "bfloat16 or float16", lambda: attention(x, x, x)),
        (RuntimeError, "must be a HIP", lambda: attention(b.cpu(), b, b)),
        (ValueError, "tokens, heads, dim", lambda: attention(b[0], b, b)),
        (ValueError, "must match q's", lambda: attention(b, b[..., :32], b)),
        (ValueError, "one shape", lambda: attention(b, b, b[:, :1])),
        (RuntimeError, "multiple of 2 key heads", lambda: attention(b[:, :1], b, b)),
        (RuntimeError, "multiples of 8", lambda: attention(b[..., :20], b[..., :20], b[..., :20])),
        (RuntimeError, "up to 128", lambda: attention(*[b.repeat(1, 1, 3)] * 3)),
        (RuntimeError, "scale", lambda: attention(b, b, b, scale=-1.0)),
        (RuntimeError, "scale", lambda: attention(b, b, b, scale=float("nan"))),
        (RuntimeError, "int32", lambda: attention(b, b, b, off.long())),
        (ValueError, "sequences \\+ 1", lambda: attention(b, b, b, off[:1])),
        (ValueError, "k_offsets is needed", lambda: attention(b, b[:3], b[:3], off)),
        (ValueError, "needs q_offsets", lambda: attention(b, b, b, None, off)),
        (ValueError, "one number of sequences",
         lambda: attention(b, b, b, off, torch.cat([off, off[1:]]))),
    ]
    for kind, text, call in bad:
        with pytest.raises(kind, match=text):
            call()


def test_heads_of_no_elements_are_refused(dev):
    from metal_gauss_amd import attention

    b = torch.zeros(4, 2, 0, dtype=torch.bfloat16, device=dev)
    with pytest.raises(RuntimeError, match="multiples of 8"):
        attention(b, b, b)


def test_second_derivatives_are_refused(dev):
    """A graph of the backward pass can be made; going through it is refused, not
    answered with zeros."""
    from metal_gauss_amd import layer_norm

    x = torch.randn(3, 8, generator=gen("twice")).to(dev).requires_grad_(True)
    dx, = torch.autograd.grad(layer_norm(x).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dx.sum().backward()


def test_forward_mode_derivatives_are_refused(dev):
    """A tangent of an input, or of a result's gradient, is refused, not dropped;
    tensors without one are served while others' are taken."""
    import torch.autograd.forward_ad as fw
    from metal_gauss_amd import attention, layer_norm, rotary, rotary_frequencies

    g = gen("tangents")
    q, k, v = (torch.randn(9, 2, 32, generator=g).to(dev, torch.bfloat16) for _ in range(3))
    x, w, b = (torch.randn(*s, generator=g).to(dev) for s in ((5, 24), (24,), (24,)))
    pos, freq = torch.arange(9, device=dev), rotary_frequencies(32, device=dev)
    calls = [(lambda q, k, v: attention(q, k, v), (q, k, v), 3),
             (lambda x, w, b: layer_norm(x, w, b), (x, w, b), 3),
             (lambda q, k, f: rotary(q, k, pos, f)[0], (q, k, freq), 2),
             (lambda q, f: rotary(q, None, pos, f), (q, freq), 1)]
    for call, inputs, leaves in calls:
        plain = call(*inputs)
        with fw.dual_level():
            assert torch.equal(call(*inputs), plain) and not call(*inputs).requires_grad
            for i in range(len(inputs)):
                dual = list(inputs)
                dual[i] = fw.make_dual(inputs[i], torch.ones_like(inputs[i]))
                with pytest.raises(NotImplementedError):
                    call(*dual)
                with torch.no_grad(), pytest.raises(NotImplementedError):
                    call(*dual)
            at = [t.detach().requires_grad_(i < leaves) for i, t in enumerate(inputs)]
            y = call(*at)
            dy = torch.ones_like(y)
            torch.autograd.grad(y, at[:leaves], dy, retain_graph=True, allow_unused=True)
            with pytest.raises(NotImplementedError):
                torch.autograd.grad(y, at[:leaves], fw.make_dual(dy, dy), allow_unused=True)


def test_rotary_refuses_frequencies_that_require_a_gradient(dev):
    """Learned frequencies would stay as they are in silence."""
    from metal_gauss_amd import rotary, rotary_frequencies

    x = torch.randn(4, 2, 32, generator=gen("learned")).to(dev)
    pos = torch.arange(4, device=dev)
    freq = rotary_frequencies(32, device=dev).requires_grad_(True)
    for q in (x, x.detach().requires_grad_(True)):
        with pytest.raises(RuntimeError, match="frequencies must not require"):
            rotary(q, None, pos, freq)
    want = rotary(x, None, pos, freq.detach())
    with torch.no_grad():
        assert torch.equal(rotary(x, None, pos, freq), want)
