"""Attention over memories that several sequences share, on the GPU, against the
float64 restatement in oracle/token_ref.py. Tolerances are those of attention: the
restatement's bound (p and the result each rounded to the type once, every rounding
at its worst), 2^-14 of the magnitudes summed for float32's part, and float16's
spacing below 2^-14."""

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


def inputs(key, nq, nk, ns, heads, kv, dim, ty):
    g = gen(*key)
    return [torch.randn(n, h, dim, generator=g).to(TYPES[ty])
            for n, h in ((nq, heads), (nk, kv), (nk, kv), (ns, kv), (ns, kv))]


def put(dev, *offs):
    return [torch.tensor(o, dtype=torch.int32, device=dev) for o in offs]


def check(dev, tensors, qo, ko, go, so, ty, causal, scale=None):
    from metal_gauss_amd import shared_attention

    at = [t.to(dev) for t in tensors]
    got = shared_attention(*at, *put(dev, qo, ko, go, so), causal=causal, scale=scale)
    assert torch.equal(got, shared_attention(*at, *put(dev, qo, ko, go, so), causal=causal,
                                             scale=scale))
    want, off = token_ref.shared_attention(
        *(host(t) for t in tensors), qo, ko, go, so, causal,
        scale if scale is not None else tensors[0].shape[2] ** -0.5, UNIT[ty])
    tiny = 2.0 ** -24 if ty == "f16" else 1e-30
    bound = off * (1.0 + 2.0 ** -14 / UNIT[ty]) * 1.05 + tiny
    bad = np.abs(host(got) - want) - bound
    assert np.isfinite(host(got)).all() and (bad <= 0).all(), \
        f"{np.abs(host(got) - want).max():.3e} off, {bad.max():.3e} over the bound"
    return got


# Sequences' query and key tokens, their number in each group, the shared tokens.
PACKS = [
    ([1], [1], [1], [1]), ([1], [0], [1], [65]), ([3], [5], [1], [0]),
    ([1] * 8, [1, 2, 3, 5, 8, 13, 21, 34], [8], [700]),          # streams over one memory
    ([1] * 9, [0, 40, 1, 0, 7, 300, 2, 2, 900], [2, 0, 7], [100, 50, 1300]),
    ([70, 1, 0, 130], [70, 90, 12, 130], [1, 3], [333, 64]),     # frames
    ([200, 60], [30, 5], [2], [129]),                            # more queries than keys
    ([1] * 70, [5] * 70, [69, 1], [31, 2000]),                   # over 64 sequences
    ([20, 0, 3], [0, 9, 1], [1, 1, 1], [0, 40, 0]),
]


@pytest.mark.parametrize("q_lens,k_lens,members,shared", PACKS)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("ty,heads,kv,dim", [("bf16", 4, 2, 64), ("f16", 6, 2, 128),
                                             ("bf16", 3, 3, 32), ("f16", 5, 1, 80)])
def test_shared(dev, q_lens, k_lens, members, shared, causal, ty, heads, kv, dim):
    key = (sum(q_lens), sum(k_lens), sum(shared), causal, ty, dim)
    t = inputs(key, sum(q_lens), sum(k_lens), sum(shared), heads, kv, dim, ty)
    qo = offsets(q_lens)
    check(dev, t, qo, offsets(k_lens), [qo[m] for m in offsets(members)], offsets(shared), ty,
          causal)


@pytest.mark.parametrize("dim", [8, 24, 48, 72, 96, 112])
def test_shared_head_dimensions(dev, dim):
    t = inputs(("dim", dim), 9, 30, 150, 4, 2, dim, "bf16")
    check(dev, t, [0, 4, 9], [0, 20, 30], [0, 9], [0, 150], "bf16", True)


@pytest.mark.parametrize("ty", ["bf16", "f16"])
@pytest.mark.parametrize("streams,heads,kv,shared,own", [
    (6, 4, 1, 9000, 2), (40, 8, 2, 5000, 30), (3, 2, 2, 70, 4000), (60, 4, 1, 1500, 900)])
def test_shared_chunks(dev, ty, streams, heads, kv, shared, own):
    """Memories, and own keys, in chunks of which the sequences have unlike numbers."""
    rng = np.random.default_rng(streams)
    k_lens = [int(x) for x in rng.integers(0, 2 * own, streams)]
    k_lens[0] = 0
    t = inputs(("chunks", streams), streams, sum(k_lens), shared + 40, heads, kv, 64, ty)
    qo = list(range(streams + 1))
    check(dev, t, qo, offsets(k_lens), [0, streams - 1, streams], [0, shared, shared + 40], ty,
          True)


def test_shared_equals_attention_with_the_memory_before_each_sequence(dev):
    """Within the rounding of p and of the result, twice."""
    from metal_gauss_amd import attention, shared_attention

    q, k, v, sk, sv = (t.to(dev) for t in inputs(("both",), 90, 140, 400, 4, 2, 64, "bf16"))
    qo, ko = [0, 40, 41, 90], [0, 60, 91, 140]
    got = shared_attention(q, k, v, sk, sv, *put(dev, qo, ko), causal=True)
    kk, vv = (torch.cat([torch.cat([a, b[s:e]]) for s, e in zip(ko[:-1], ko[1:])])
              for a, b in ((sk, k), (sv, v)))
    whole = attention(q, kk, vv, *put(dev, qo, offsets([460, 431, 449])), causal=True)
    assert float((got.float() - whole.float()).abs().max()) < 4 * 2.0 ** -8


def test_shared_without_one_of_them(dev):
    """No memory: attention's result to rounding; no own keys: the memory's."""
    from metal_gauss_amd import attention, shared_attention

    q, k, v, sk, sv = (t.to(dev) for t in inputs(("one",), 50, 50, 300, 4, 4, 64, "f16"))
    off, = put(dev, [0, 20, 50])
    none = sk[:0]
    a = shared_attention(q, k, v, none, none, off, causal=True)
    assert float((a.float() - attention(q, k, v, off, causal=True).float()).abs().max()) < 2e-3
    off2, = put(dev, [0, 0, 0])
    a = shared_attention(q, k[:0], v[:0], sk, sv, off, off2)
    assert float((a.float() - attention(q, sk, sv).float()).abs().max()) < 2e-3
    assert torch.equal(shared_attention(q, k[:0], v[:0], none, none, off, off2),
                       torch.zeros_like(q))
    assert shared_attention(q[:0], k, v, sk, sv).shape == (0, 4, 64)


def test_shared_tokens_of_no_group_and_of_no_sequence(dev):
    """And what no query sees may hold anything."""
    from metal_gauss_amd import attention, shared_attention

    q, k, v, sk, sv = (t.to(dev) for t in inputs(("gaps",), 60, 80, 200, 4, 2, 64, "bf16"))
    qo, ko, go, so = put(dev, [5, 20, 40], [10, 30, 70], [10, 30, 50], [20, 90, 180])
    clean = shared_attention(q, k, v, sk, sv, qo, ko, go, so, causal=True)
    for t, lost in ((k, [*range(10), *range(70, 80)]), (sk, [*range(20), *range(180, 200)])):
        t[lost] = float("nan")
    for t, lost in ((v, [*range(10), *range(70, 80)]), (sv, [*range(20), *range(180, 200)])):
        t[lost] = float("inf")
    q[:5], q[50:] = float("nan"), float("nan")
    got = shared_attention(q, k, v, sk, sv, qo, ko, go, so, causal=True)
    assert torch.equal(got, clean)
    assert bool((got[:5] == 0).all()) and bool((got[50:] == 0).all())
    want = attention(q[5:20], k[10:30], v[10:30], causal=True)[:5]          # of no group
    assert float((got[5:10].float() - want.float()).abs().max()) < 2.0 ** -6
    want = attention(q[40:50], sk[90:180], sv[90:180])                      # of no sequence
    assert float((got[40:50].float() - want.float()).abs().max()) < 2.0 ** -6


def test_shared_values_that_are_not_finite_reach_those_who_see_them(dev):
    from metal_gauss_amd import shared_attention

    q, k, v, sk, sv = (t.to(dev) for t in inputs(("poison",), 12, 12, 900, 2, 1, 64, "bf16"))
    qo, go, so = put(dev, [0, 5, 12], [0, 5, 12], [0, 400, 900])
    clean = shared_attention(q, k, v, sk, sv, qo, qo, go, so, causal=True).float()
    sv[399, :, 3], v[7, :, 5], sv[400, :, 9] = float("inf"), float("nan"), float("-inf")
    got = shared_attention(q, k, v, sk, sv, qo, qo, go, so, causal=True).float()
    clean[:5, :, 3], clean[7:, :, 5], clean[5:, :, 9] = float("inf"), float("nan"), float("-inf")
    assert torch.equal(got.isnan(), clean.isnan())
    assert torch.equal(got.nan_to_num(7.0), clean.nan_to_num(7.0))


def test_shared_offsets_are_held_and_made_to_rise(dev):
    from metal_gauss_amd import shared_attention

    t = [x.to(dev) for x in inputs(("fall",), 100, 120, 300, 4, 2, 64, "f16")]
    got = []
    for rising in (False, True):
        offs = []
        for off, n in (([3, 60, 20, 90], 100), ([-4, 90, 80, 450], 120), ([50, 20, 10 ** 9], 100),
                       ([10, 250, 100], 300)):
            off = np.asarray(off)
            offs.append(np.maximum.accumulate(off.clip(0, n)) if rising else off)
        got.append(shared_attention(*t, *put(dev, *offs), causal=True))
    assert torch.equal(*got) and bool(got[0].isfinite().all())


def test_shared_strided_views(dev):
    from metal_gauss_amd import shared_attention

    g = gen("views")
    qkv = torch.randn(60, 8, 64, generator=g).to(dev, torch.bfloat16)
    rows = torch.randn(300, 2, 2, 64, generator=g).to(dev, torch.bfloat16)
    q, k, v, sk, sv = qkv[:, :4], qkv[:, 4:6], qkv[:, 6:], rows[:, 0], rows[:, 1]
    want = shared_attention(*(t.contiguous() for t in (q, k, v, sk, sv)), causal=True)
    assert torch.equal(shared_attention(q, k, v, sk, sv, causal=True), want)
    odd = torch.empty(300 * 4 * 64 + 1, device=dev, dtype=torch.bfloat16)[1:].view(300, 2, 2, 64)
    odd.copy_(rows)                                              # not 16-byte aligned
    assert torch.equal(shared_attention(q, k, v, odd[:, 0], odd[:, 1], causal=True), want)


def test_shared_rows_whose_offsets_pass_32_bits(dev):
    """A memory of 600 keys and values 2^23 elements apart."""
    from metal_gauss_amd import shared_attention

    g = gen("far rows")
    far = torch.empty(600, 1 << 23, device=dev, dtype=torch.bfloat16)[:, :256].view(600, 4, 64)
    far.copy_(torch.randn(600, 4, 64, generator=g))
    q, k, v = (torch.randn(9, h, 64, generator=g).to(dev, torch.bfloat16) for h in (4, 2, 2))
    want = shared_attention(q, k, v, far[:, :2].contiguous(), far[:, 2:].contiguous(), causal=True)
    assert torch.equal(shared_attention(q, k, v, far[:, :2], far[:, 2:], causal=True), want)


def test_shared_in_a_graph_and_on_another_stream(dev):
    """Two graphs, replayed in turn with eager work between."""
    from metal_gauss_amd import shared_attention

    graphs = []
    for n, shared in ((6, 5000), (200, 700)):
        t = [x.to(dev) for x in inputs(("graph", n), n, 900, shared, 4, 2, 64, "bf16")]
        off = put(dev, list(range(n + 1)), [900 * i // n for i in range(n + 1)])
        step = lambda t=t, off=off: shared_attention(*t, *off, causal=True)  # noqa: E731
        want = step()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got = step()
        torch.cuda.current_stream().wait_stream(s)
        assert torch.equal(got, want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out, t, step))
    for i in range(3):
        for graph, out, t, step in graphs:
            for x in t:
                x.copy_(torch.randn(x.shape, generator=gen("again", i)))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, step())


def test_shared_refusals(dev):
    import torch.autograd.forward_ad as fw
    from metal_gauss_amd import shared_attention

    b = torch.zeros(4, 2, 64, device=dev, dtype=torch.bfloat16)
    off, two = put(dev, [0, 4], [0, 2, 4])
    bad = [
        (RuntimeError, "shared_k must be bfloat16 or float16",
         lambda: shared_attention(b, b, b, b.float(), b)),
        (RuntimeError, "must be a HIP", lambda: shared_attention(b, b, b, b, b.cpu())),
        (ValueError, "must match q's", lambda: shared_attention(b, b, b, b.half(), b)),
        (ValueError, "must match q's", lambda: shared_attention(b, b, b, b, b[..., :32])),
        (ValueError, "one shape", lambda: shared_attention(b, b, b, b[:3], b)),
        (ValueError, "of k's 2 heads", lambda: shared_attention(b, b, b, b[:, :1], b[:, :1])),
        (ValueError, "go together", lambda: shared_attention(b, b, b, b, b, group_offsets=off)),
        (ValueError, "one number of groups",
         lambda: shared_attention(b, b, b, b, b, None, None, off, two)),
        (RuntimeError, "int32", lambda: shared_attention(b, b, b, b, b, None, None, off.long(),
                                                         off)),
        (RuntimeError, "scale", lambda: shared_attention(b, b, b, b, b, scale=-1.0)),
        (RuntimeError, "multiple of 2 key heads",
         lambda: shared_attention(b[:, :1], b, b, b, b)),
        (RuntimeError, "has no gradient",
         lambda: shared_attention(b, b, b, b.clone().requires_grad_(True), b)),
    ]
    for kind, text, call in bad:
        with pytest.raises(kind, match=text):
            call()
    leaf = b.clone().requires_grad_(True)
    with torch.no_grad():
        assert shared_attention(leaf, b, b, b, b).shape == b.shape
    with fw.dual_level():
        assert shared_attention(b, b, b, b, b).shape == b.shape
        with pytest.raises(NotImplementedError):
            shared_attention(b, b, b, fw.make_dual(b, b), b)
