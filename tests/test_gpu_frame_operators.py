"""The operators of networks over frames on the GPU (heads normed and turned,
dropout, rotary sections) against the float64 restatements in oracle/token_ref.py.

Tolerances. With u the unit roundoff of the stored type (2^-24, 2^-8, 2^-11 for
float32, bfloat16, float16):

* heads normed and turned: float32 arithmetic rounded once. A head's mean of squares
  is a sum of at most 512 positive terms (off by under 32 * 2^-24 of itself, in a
  tree over the lanes), and each result is a few products: 64 * 2^-24 of the
  largest result of the pair, head or gradient covers them; the rounding adds u of
  the value. Gradients of the weights: sums over tokens and heads in float32, off by
  at most (additions a value passes through, under 64 + heads / 32) * 2^-24 of the
  sum of magnitudes.
* dropout: a product and a sum in float32 (2 * 2^-24 of the magnitudes), rounded
  once; which elements are kept is exact.
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
# Below 2^-14 float16's values lie 2^-24 apart, so that a rounding there is off by
# up to 2^-25 and not by u of the value. (bfloat16's and float32's begin at 2^-126.)
LEAST = {"f32": 0.0, "bf16": 0.0, "f16": 2.0 ** -25}


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


# ------------------------------------------------------- heads normed and turned

def check_norm_rotary(dev, ty, wt, tokens, heads, kv, dim, part, sections, order, layout,
                      positions=None, eps=1e-6, gain=1.0, weights=True):
    from metal_gauss_amd import norm_rotary, rotary_frequencies

    g = gen(ty, wt, tokens, heads, kv, dim, part, sections, order, layout)
    leaves = [gain * torch.randn(tokens, h, dim, generator=g) for h in (heads, kv)]
    leaves = [t.to(TYPES[ty]) for t in leaves]
    ws = [(1.0 + 0.3 * torch.randn(dim, generator=g)).to(TYPES[wt]) for _ in range(2)]
    dys = [torch.randn(tokens, h, dim, generator=g).to(TYPES[ty]) for h in (heads, kv)]
    if positions is None:
        positions = torch.randint(-5, 3000, (tokens, len(sections)), generator=g,
                                  dtype=torch.int32)
    freq = rotary_frequencies(part, device=dev)
    put = [t.to(dev).requires_grad_(True) for t in leaves]
    wput = [t.to(dev).requires_grad_(True) if weights else None for t in ws]
    if kv == 0:
        put[1] = wput[1] = None
    call = lambda: norm_rotary(put[0], put[1], wput[0], wput[1], positions.to(dev), freq,  # noqa: E731
                               eps=eps, layout=layout, sections=sections, order=order)
    out = call()
    out = out if kv else (out,)
    inputs = [t for t in (*put, *wput) if t is not None]
    grads = torch.autograd.grad(out, inputs, [d.to(dev) for d in dys[:len(out)]])
    with torch.no_grad():
        again = call()
        assert all(torch.equal(a, b) for a, b in zip(again if kv else (again,), out))
    axes = token_ref.axes_of(sections, order)
    P, F, u, uw = positions.numpy(), host(freq), UNIT[ty], UNIT[wt]
    turn = lambda x: token_ref.rotary_axes(x, P, F, layout, axes)  # noqa: E731
    back = lambda x: token_ref.rotary_axes(x, P, F, layout, axes, True)  # noqa: E731
    n = 1 + (kv > 0)
    for i in range(n):
        x, dy = host(leaves[i]), host(dys[i])
        w = host(ws[i]) if weights else None
        want = token_ref.norm_rotary(x, w, eps, turn)
        top = np.abs(want).max(-1, keepdims=True)
        # A pair's rotation may leave little of two large elements.
        close(out[i], want, u * np.abs(want) + 64 * EPS24 * 2 * top, f"y {i}")
        dx, dw = token_ref.norm_rotary_grad(x, w, eps, back, dy)
        s = 1.0 / np.sqrt((x ** 2).mean(-1, keepdims=True) + eps)
        size = s * np.abs(dy).max(-1, keepdims=True) * 2 * (1 if w is None else np.abs(w).max())
        size = size * (1 + (x * s) ** 2).max(-1, keepdims=True)
        close(grads[i], dx, u * np.abs(dx) + 64 * EPS24 * size, f"dx {i}")
        if weights:
            deep = (64 + tokens * (heads, kv)[i] / 32) * EPS24
            mag = (np.abs(back(dy)) * np.abs(x * s)).sum((0, 1))
            # A turned element is off by 2^-22 of its pair's length.
            pair = np.abs(dy).max(-1, keepdims=True) * np.abs(x * s) * 8 * EPS24
            close(grads[n + i], dw, uw * np.abs(dw) + deep * mag + pair.sum((0, 1)), f"dw {i}")


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("ty,wt", [("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16"),
                                   ("f16", "f16")])
@pytest.mark.parametrize("tokens,heads,kv,dim,part,sections,order", [
    (1, 1, 1, 2, 2, (1,), "runs"), (1, 4, 1, 64, 64, (32,), "runs"),
    (16, 16, 4, 64, 64, (8, 12, 12), "runs"), (7, 3, 2, 128, 64, (1, 0, 31), "turns"),
    (33, 5, 5, 96, 96, (16, 24, 8), "turns"), (9, 2, 1, 80, 40, (10, 10), "runs"),
    (5, 3, 1, 30, 10, (5,), "runs"), (11, 1, 0, 66, 66, (1, 2, 30), "turns"),
    (2100, 4, 2, 32, 32, (16,), "runs"), (3, 2, 2, 512, 512, (100, 156), "runs"),
    (4, 2, 1, 48, 16, (3, 5), "turns"), (6, 70, 3, 256, 256, (128,), "runs"),
    (5, 300, 130, 64, 64, (20, 12), "runs"), (3, 2, 1, 46, 22, (11,), "runs"),
    (3, 2, 1, 510, 254, (127,), "runs")])
def test_norm_rotary(dev, layout, ty, wt, tokens, heads, kv, dim, part, sections, order):
    check_norm_rotary(dev, ty, wt, tokens, heads, kv, dim, part, sections, order, layout)


@pytest.mark.parametrize("dim,part", [(31, 10), (65, 64), (257, 128), (511, 254)])
def test_norm_rotary_odd_heads(dev, dim, part):
    check_norm_rotary(dev, "bf16", "f32", 5, 3, 2, dim, part, (part // 2,), "runs", "half")


def test_norm_rotary_many_tokens(dev):
    """More batches than workgroups, whose sums over the tokens are joined."""
    check_norm_rotary(dev, "bf16", "f32", 5003, 6, 2, 128, 128, (16, 24, 24), "runs", "half")


@pytest.mark.parametrize("gain", [1e-4, 1e4])
def test_norm_rotary_small_and_large_heads(dev, gain):
    check_norm_rotary(dev, "f32", "f32", 6, 2, 2, 64, 64, (32,), "runs", "half", gain=gain)


@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("gain,eps", [(1e14, 1e-6), (1e-14, 0.0)])
def test_norm_rotary_heads_whose_cubes_pass_the_range(dev, ty, gain, eps):
    """1 / rms cubed is not in float32's range; the gradients are."""
    check_norm_rotary(dev, ty, "f32", 6, 2, 2, 64, 64, (32,), "runs", "half", gain=gain, eps=eps)


def test_norm_rotary_without_weights(dev):
    check_norm_rotary(dev, "bf16", "f32", 6, 2, 2, 64, 32, (16,), "runs", "interleaved",
                      weights=False)


@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_norm_rotary_far_positions(dev, kind):
    """As rotary: angles of 10^9 radians are as exact as those of 10 (2^-23 of a turn),
    which 2^-20 of the largest element covers."""
    from metal_gauss_amd import norm_rotary, rotary_frequencies

    q = torch.randn(6, 2, 64, generator=gen("far")).to(dev)
    pos = torch.tensor([0, 1, 131071, 10 ** 6, 2 ** 30, -(2 ** 30)], dtype=kind)
    freq = rotary_frequencies(64, device=dev)
    got = norm_rotary(q, None, None, None, pos.to(dev), freq)
    want = token_ref.norm_rotary(host(q), None, 1e-6, lambda x: token_ref.rotary(
        x, pos.numpy()[:, None], host(freq), "half"))
    close(got, want, (64 * EPS24 + 2.0 ** -20) * np.abs(want).max(-1, keepdims=True), "q")


def test_norm_rotary_equals_its_two_steps(dev):
    """The norm in float64 and rotary(), within the two roundings of the latter."""
    from metal_gauss_amd import norm_rotary, rotary, rotary_frequencies

    x = torch.randn(40, 4, 64, generator=gen("steps")).to(dev)
    pos = torch.randint(0, 99, (40, 3), generator=gen("at"), dtype=torch.int32).to(dev)
    freq = rotary_frequencies(64, device=dev)
    u = (x.double() / (x.double().square().mean(-1, keepdim=True) + 1e-6).sqrt()).float()
    for order in ("runs", "turns"):
        kw = dict(sections=(8, 12, 12), order=order)
        a = norm_rotary(x, None, None, None, pos, freq, **kw)
        b = rotary(u, None, pos, freq, **kw)
        assert float((a - b).abs().max()) < 64 * EPS24 * float(u.abs().max())


def test_norm_rotary_slices_and_strides(dev):
    from metal_gauss_amd import norm_rotary, rotary_frequencies

    g = gen("slices")
    qkv = torch.randn(50, 10, 66, generator=g).to(dev)
    w = torch.randn(130, generator=g).to(dev)[1::2][:64]          # strided weights
    pos = torch.arange(100, dtype=torch.int32, device=dev)[::2]
    freq = rotary_frequencies(64, device=dev)
    q, k = qkv[:, :6, :64], qkv[:, 6:8, :64]
    turned = qkv.permute(2, 1, 0).contiguous().permute(2, 1, 0)   # dim outermost
    dy = [torch.randn(64, h, 50, generator=g).to(dev).permute(2, 1, 0) for h in (6, 2)]
    results = []
    for a, b in ((q, k), (q.contiguous(), k.contiguous()),
                 (turned[:, :6, :64], turned[:, 6:8, :64])):
        a, b = a.detach().requires_grad_(True), b.detach().requires_grad_(True)
        wl = w.detach().requires_grad_(True)
        out = norm_rotary(a, b, wl, wl, pos, freq)
        results.append((*out, *torch.autograd.grad(out, (a, b, wl), dy)))
    for other in results[1:]:
        assert all(torch.equal(x, y) for x, y in zip(results[0], other))
    one = qkv[:1, :6, :64].detach().expand(50, 6, 64)             # a broadcast input
    assert torch.equal(norm_rotary(one, None, w, None, pos, freq),
                       norm_rotary(one.contiguous(), None, w, None, pos, freq))


def test_norm_rotary_rows_whose_offsets_pass_32_bits(dev):
    from metal_gauss_amd import norm_rotary, rotary_frequencies

    g = gen("far rows")
    far = torch.empty(600, 1 << 23, device=dev, dtype=torch.bfloat16)[:, :256].view(600, 4, 64)
    far.copy_(torch.randn(600, 4, 64, generator=g))
    far_dy = torch.empty(600, 1 << 23, device=dev, dtype=torch.bfloat16)[:, :128].view(600, 2, 64)
    far_dy.copy_(torch.randn(600, 2, 64, generator=g))
    w = torch.rand(64, generator=g).to(dev)
    pos, freq = torch.arange(600, device=dev), rotary_frequencies(64, device=dev)
    results = []
    for x, dy in ((far, far_dy), (far.contiguous(), far_dy.contiguous())):
        leaves = [t.detach().requires_grad_(True) for t in (x[:, :2], x[:, 2:], w)]
        y = norm_rotary(leaves[0], leaves[1], leaves[2], leaves[2], pos, freq)
        results.append((*y, *torch.autograd.grad(y, leaves, (dy, dy))))
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_norm_rotary_gradients_of_some(dev):
    """Of one result, of the weights alone, of the inputs alone."""
    from metal_gauss_amd import norm_rotary, rotary_frequencies

    g = gen("some")
    q, k = (torch.randn(8, h, 32, generator=g).to(dev, torch.bfloat16) for h in (4, 2))
    qw, kw = (1.0 + torch.rand(32, generator=g)).to(dev), torch.ones(32, device=dev)
    pos = torch.arange(8, dtype=torch.int32, device=dev)
    freq = rotary_frequencies(32, device=dev)
    leaves = [t.requires_grad_(True) for t in (q, k, qw, kw)]
    out = norm_rotary(*leaves, pos, freq)
    dys = [torch.randn(o.shape, generator=g).to(o) for o in out]
    full = torch.autograd.grad(out, leaves, dys, retain_graph=True)
    for i in range(2):
        x, w = torch.autograd.grad(out[i], (leaves[i], leaves[2 + i]), dys[i], retain_graph=True)
        assert torch.equal(x, full[i]) and torch.equal(w, full[2 + i])
    for pick in ((0, 1), (2, 3), (0, 3), (2,)):
        some = [t if i in pick else t.detach() for i, t in enumerate(leaves)]
        got = torch.autograd.grad(norm_rotary(*some, pos, freq), [leaves[i] for i in pick], dys)
        assert all(torch.equal(a, full[i]) for a, i in zip(got, pick))
    plain = norm_rotary(q, k, None, kw, pos, freq)
    assert torch.equal(plain[1], out[1])


def test_norm_rotary_of_no_tokens_and_of_zeros(dev):
    from metal_gauss_amd import norm_rotary, rotary_frequencies

    freq = rotary_frequencies(32, device=dev)
    q = torch.zeros(0, 2, 32, device=dev, requires_grad=True)
    w = torch.ones(32, device=dev, requires_grad=True)
    y = norm_rotary(q, None, w, None, torch.zeros(0, dtype=torch.int32, device=dev), freq)
    dq, dw = torch.autograd.grad(y.sum(), (q, w))
    assert y.shape == dq.shape == (0, 2, 32) and torch.equal(dw, torch.zeros_like(dw))
    q = torch.zeros(3, 2, 32, device=dev, requires_grad=True)
    pos = torch.arange(3, dtype=torch.int32, device=dev)
    y = norm_rotary(q, None, w, None, pos, freq)
    dq, = torch.autograd.grad(y, q, torch.ones_like(y))
    assert torch.equal(y, torch.zeros_like(y)) and bool(dq.isfinite().all())


def test_norm_rotary_nan_stays_in_its_head(dev):
    from metal_gauss_amd import norm_rotary, rotary_frequencies

    x = torch.randn(9, 3, 64, generator=gen("nan")).to(dev)
    pos = torch.arange(9, dtype=torch.int32, device=dev)
    freq = rotary_frequencies(32, device=dev)
    clean = norm_rotary(x, None, None, None, pos, freq)
    x[4, 1, 63], x[0, 0, 0] = float("nan"), float("nan")
    y = norm_rotary(x, None, None, None, pos, freq)
    bad = torch.zeros(9, 3, dtype=torch.bool, device=dev)
    bad[4, 1] = bad[0, 0] = True
    assert bool(y[bad].isnan().all()) and torch.equal(y[~bad], clean[~bad])


def test_norm_rotary_gradient_against_differences(dev):
    """Central differences of the restatement, with a step of 1e-5 in float64: off
    by its square and by float32 in the gradient."""
    from metal_gauss_amd import norm_rotary, rotary_frequencies

    g = gen("differences")
    x, dy = torch.randn(2, 1, 24, generator=g), torch.randn(2, 1, 24, generator=g)
    w = 1.0 + 0.3 * torch.randn(24, generator=g)
    pos = torch.tensor([[3, 1], [50, 7]], dtype=torch.int32)
    freq = rotary_frequencies(16, device=dev)
    xd, wd = x.to(dev).requires_grad_(True), w.to(dev).requires_grad_(True)
    y = norm_rotary(xd, None, wd, None, pos.to(dev), freq, sections=(3, 5))
    dx, dw = torch.autograd.grad(y, (xd, wd), dy.to(dev))
    turn = lambda t: token_ref.rotary_axes(t, pos.numpy(), host(freq), "half",  # noqa: E731
                                           token_ref.axes_of((3, 5), "runs"))
    X, W, DY = host(x), host(w), host(dy)
    value = lambda a, b: (token_ref.norm_rotary(a, b, 1e-6, turn) * DY).sum()  # noqa: E731
    for i in range(24):
        e = np.zeros(24)
        e[i] = 1e-5
        num = (value(X, W + e) - value(X, W - e)) / 2e-5
        assert abs(num - float(dw[i])) < 1e-5
        for t in range(2):
            d = np.zeros((2, 1, 24))
            d[t, 0, i] = 1e-5
            num = (value(X + d, W) - value(X - d, W)) / 2e-5
            assert abs(num - float(dx[t, 0, i])) < 1e-5


# --------------------------------------------------------------- rotary sections

@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("ty,tokens,heads,kv,dim,sections", [
    ("f32", 7, 3, 2, 64, (8, 12, 12)), ("bf16", 300, 4, 0, 80, (20,)),
    ("f16", 5, 2, 2, 32, (0, 1, 15)), ("bf16", 9, 1, 1, 512, (100, 100, 50, 6))])
@pytest.mark.parametrize("order", ["runs", "turns"])
def test_rotary_sections(dev, layout, ty, tokens, heads, kv, dim, sections, order):
    from metal_gauss_amd import rotary, rotary_frequencies

    g = gen(layout, ty, dim, sections, order)
    q, k = (torch.randn(tokens, h, dim, generator=g).to(dev, TYPES[ty]).requires_grad_(True)
            for h in (heads, kv))
    pos = torch.randint(0, 5000, (tokens, len(sections)), generator=g).to(dev)
    freq = rotary_frequencies(2 * sum(sections), device=dev)
    out = rotary(q, k if kv else None, pos, freq, layout=layout, sections=sections, order=order)
    axes, P, F = token_ref.axes_of(sections, order), pos.cpu().numpy(), host(freq)
    for x, y in zip((q, k), out if kv else (out,)):
        bound = lambda want, top: UNIT[ty] * np.abs(want) + 64 * EPS24 * top  # noqa: E731
        want = token_ref.rotary_axes(host(x), P, F, layout, axes)
        close(y, want, bound(want, np.abs(host(x)).max()), "y")
        dy = torch.randn(y.shape, generator=g).to(y)
        dx, = torch.autograd.grad(y, x, dy, retain_graph=True)
        want = token_ref.rotary_axes(host(dy), P, F, layout, axes, True)
        close(dx, want, bound(want, np.abs(host(dy)).max()), "dx")


def test_rotary_equal_sections_are_equal_runs(dev):
    from metal_gauss_amd import rotary, rotary_frequencies

    q = torch.randn(30, 2, 64, generator=gen("equal")).to(dev)
    pos = torch.randint(0, 99, (30, 2), generator=gen("p")).to(dev)
    freq = rotary_frequencies(64, axes=2, device=dev)
    assert torch.equal(rotary(q, None, pos, freq),
                       rotary(q, None, pos, freq, sections=(16, 16)))


# ----------------------------------------------------------------- dropout

@pytest.mark.parametrize("x_ty,r_ty", [("f32", None), ("f32", "f32"), ("bf16", None),
                                       ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f32"),
                                       ("f16", "f16"), ("f16", None)])
@pytest.mark.parametrize("shape,p", [((1,), 0.5), ((7,), 0.3), ((8, 1), 0.1), ((3, 5, 67), 0.25),
                                     ((4096,), 0.9), ((2, 2049), 0.1), ((70, 129), 0.5)])
def test_dropout(dev, x_ty, r_ty, shape, p):
    from metal_gauss_amd import dropout

    g = gen("dropout", x_ty, r_ty, shape)
    x = torch.randn(*shape, generator=g).to(TYPES[x_ty])
    r = None if r_ty is None else torch.randn(*shape, generator=g).to(TYPES[r_ty])
    seed = 2 ** 63 + 12345678901
    leaves = [t.to(dev).requires_grad_(True) for t in (x, r) if t is not None]
    y = dropout(leaves[0], p, seed, residual=leaves[1] if r is not None else None, site=3)
    out = r_ty or x_ty
    dy = torch.randn(*shape, generator=g).to(TYPES[out])
    grads = torch.autograd.grad(y, leaves, dy.to(dev))
    drop = round(p * 65536)
    keep = token_ref.kept(x.numel(), drop, seed, 3).reshape(shape)
    gain = 65536 / (65536 - drop)
    part = np.where(keep, host(x) * gain, 0.0)
    want = part + (0.0 if r is None else host(r))
    size = np.abs(part) + (0.0 if r is None else np.abs(host(r)))
    assert y.dtype == TYPES[out]
    close(y, want, UNIT[out] * np.abs(want) + 2 * EPS24 * size + LEAST[out], "y")
    back = np.where(keep, host(dy) * gain, 0.0)
    close(grads[0], back, (UNIT[x_ty] + 2 * EPS24) * np.abs(back) + LEAST[x_ty], "dx")
    assert grads[0].dtype == TYPES[x_ty]
    if r is not None:
        assert torch.equal(grads[1].cpu(), dy)


def test_dropout_draws_do_not_depend_on_type_shape_or_layout(dev):
    from metal_gauss_amd import dropout

    x = torch.ones(40, 50, device=dev)
    keep = dropout(x, 0.5, 9) != 0
    assert torch.equal(keep, dropout(x.bfloat16(), 0.5, 9) != 0)
    assert torch.equal(keep.flatten(), dropout(x.flatten(), 0.5, 9) != 0)
    assert torch.equal(keep, dropout(torch.ones(50, 40, device=dev).t(), 0.5, 9) != 0)
    assert torch.equal(keep, dropout(x[:1].expand(40, 50), 0.5, 9) != 0)
    odd = torch.ones(2001, device=dev)[1:].view(40, 50)                 # not 16-byte aligned
    assert torch.equal(keep, dropout(odd, 0.5, 9) != 0)
    at = torch.tensor([9], device=dev)
    assert torch.equal(keep, dropout(x, 0.5, at) != 0)
    for other in (dropout(x, 0.5, 10), dropout(x, 0.5, 9, site=1), dropout(x, 0.5, 9 + 2 ** 32)):
        assert 800 < int((keep == (other != 0)).sum()) < 1200           # 2000 fair coins


def test_dropout_share_and_mean(dev):
    """10^6 elements: 5 standard deviations of the number kept, and the gain by it."""
    from metal_gauss_amd import dropout

    for p in (0.01, 0.1, 0.5, 0.87):
        y = dropout(torch.ones(10 ** 6, device=dev), p, 4)
        held = round(p * 65536) / 65536
        n = int((y != 0).sum())
        assert abs(n - 1e6 * (1 - held)) < 5 * (1e6 * held * (1 - held)) ** 0.5
        assert bool((y[y != 0] - 1 / (1 - held)).abs().max() < 1e-5)


def test_dropout_ends_of_the_range(dev):
    from metal_gauss_amd import dropout

    x = torch.randn(1000, generator=gen("ends")).to(dev)
    x[3], x[4] = float("nan"), float("inf")
    r = torch.randn(1000, generator=gen("r")).to(dev)
    assert torch.equal(dropout(x, 1.0, 1), torch.zeros_like(x))
    assert torch.equal(dropout(x, 1.0, 1, residual=r), r)
    y = dropout(x, 0.0, 1)
    assert torch.equal(y[5:], x[5:]) and bool(y[3].isnan()) and y.data_ptr() != x.data_ptr()
    assert dropout(x[:0], 0.5, 1).shape == (0,)
    # p below 1 keeps something of enough elements: 2^-16 of them.
    assert 0 < int((dropout(torch.ones(10 ** 7, device=dev), 1.0 - 1e-9, 5) != 0).sum()) < 400


def test_dropout_many_elements(dev):
    """Counters past 2^24 of the first word."""
    from metal_gauss_amd import dropout

    n = 2 ** 27 + 5
    y = dropout(torch.ones(n, device=dev, dtype=torch.bfloat16), 0.5, 77)
    for first in (0, 2 ** 26 + 3, n - 40):
        want = token_ref.kept(40, 32768, 77, first=first)
        assert np.array_equal((y[first:first + 40] != 0).cpu().numpy(), want)


def test_dropout_past_32_bits(dev):
    """Element numbers of 2^32 and more."""
    from metal_gauss_amd import dropout

    n = 2 ** 32 + 997
    y = dropout(torch.ones(1, device=dev, dtype=torch.bfloat16).expand(n), 0.5, 11, site=2)
    for first in (2 ** 31 - 20, 2 ** 32 - 20, n - 40):
        want = token_ref.kept(40, 32768, 11, site=2, first=first)
        assert np.array_equal((y[first:first + 40] != 0).cpu().numpy(), want)


def test_dropout_seed_counted_on_in_a_graph(dev):
    """Captured once with its gradient, replayed on a seed that a captured step counts
    on and on new inputs, with eager work between."""
    from metal_gauss_amd import dropout

    x = torch.randn(300, 70, generator=gen("graph")).to(dev, torch.bfloat16).requires_grad_(True)
    r = torch.randn(300, 70, generator=gen("residual")).to(dev)
    dy = torch.randn(300, 70, generator=gen("dy")).to(dev)
    seed = torch.tensor([41], device=dev)

    def step():
        y = dropout(x, 0.2, seed, residual=r)
        y2 = dropout(x, 0.2, seed, residual=y, site=1)
        return y2.detach(), torch.autograd.grad(y2, x, dy)[0]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
        seed.add_(1)
    seen = []
    for i in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(300, 70, generator=gen("x", i)))
        want = step()
        assert int(seed) == 41 + i
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        seen.append(got[0].clone())
    assert not torch.equal(seen[0], seen[1])


def test_dropout_seed_changed_before_the_backward_pass_is_refused(dev):
    from metal_gauss_amd import dropout

    x = torch.ones(64, device=dev, requires_grad=True)
    seed = torch.tensor([1], device=dev)
    y = dropout(x, 0.5, seed)
    seed.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


# ---------------------------------------------------------------- shared ways

def calls(dev):
    """(call, its leaves) of each operator."""
    from metal_gauss_amd import dropout, norm_rotary, rotary, rotary_frequencies

    g = gen("calls")
    q, k = (torch.randn(90, h, 32, generator=g).to(dev, torch.bfloat16).requires_grad_(True)
            for h in (4, 2))
    w, v = ((1.0 + torch.rand(32, generator=g)).to(dev).requires_grad_(True) for _ in range(2))
    r = torch.randn(90, 4, 32, generator=g).to(dev).requires_grad_(True)
    pos = torch.randint(0, 500, (90, 3), generator=g).to(dev)
    seed = torch.tensor([3], device=dev)
    freq = rotary_frequencies(32, device=dev)
    kw = dict(sections=(4, 6, 6))
    return [(lambda: torch.cat(norm_rotary(q, k, w, v, pos, freq, **kw), 1), (q, k, w, v)),
            (lambda: dropout(q, 0.3, seed, residual=r), (q, r)),
            (lambda: torch.cat(rotary(q, k, pos, freq, **kw), 1), (q, k))]


def test_saved_tensors_may_come_back_in_another_layout(dev):
    def spread(t):
        wide = torch.full((*t.shape, 3), 7, dtype=t.dtype, device=t.device)
        wide[..., 1] = t
        return wide[..., 1]

    for call, leaves in calls(dev):
        y = call()
        dy = torch.randn(y.shape, generator=gen("hooks")).to(y)
        want = torch.autograd.grad(y, leaves, dy)
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, spread):
            y = call()
        got = torch.autograd.grad(y, leaves, dy)
        assert all(torch.equal(a, c) for a, c in zip(got, want))


def test_on_another_stream_and_in_a_graph(dev):
    for call, leaves in calls(dev):
        dy = torch.ones_like(call())

        def step():
            y = call()
            return (y.detach(), *torch.autograd.grad(y, leaves, dy))

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
        for i in range(3):
            with torch.no_grad():
                leaves[0].copy_(torch.randn(leaves[0].shape, generator=gen("in", i)))
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_derivatives_that_are_refused(dev):
    """Second derivatives, and tangents of inputs and of gradients."""
    import torch.autograd.forward_ad as fw

    for call, leaves in calls(dev):
        y = call()
        dx, = torch.autograd.grad(y.square().sum(), leaves[0], create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            dx.sum().backward()
        with fw.dual_level():
            y = call()
            dy = torch.ones_like(y)
            with pytest.raises(NotImplementedError):
                torch.autograd.grad(y, leaves, fw.make_dual(dy, dy))


def test_tangents_of_inputs_are_refused(dev):
    import torch.autograd.forward_ad as fw
    from metal_gauss_amd import dropout, norm_rotary, rotary_frequencies

    x = torch.randn(9, 2, 32, generator=gen("t")).to(dev)
    w = torch.ones(32, device=dev)
    pos, freq = torch.arange(9, device=dev), rotary_frequencies(32, device=dev)
    with fw.dual_level(), torch.no_grad():
        dual = lambda t: fw.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: norm_rotary(dual(x), None, w, None, pos, freq),
                     lambda: norm_rotary(x, x, w, dual(w), pos, freq),
                     lambda: dropout(dual(x), 0.5, 1), lambda: dropout(x, 0.5, 1, residual=dual(x))):
            with pytest.raises(NotImplementedError):
                call()
        assert torch.equal(dropout(x, 0.5, 1), dropout(x.clone(), 0.5, 1))


def test_refusals(dev):
    from metal_gauss_amd import dropout, norm_rotary, rotary, rotary_frequencies

    f = rotary_frequencies(64, device=dev)
    x = torch.zeros(4, 2, 64, device=dev)
    b = x.bfloat16()
    w = torch.ones(64, device=dev)
    pos = torch.zeros(4, dtype=torch.int32, device=dev)
    pos3 = pos[:, None].expand(4, 3)

    def norm(q=x, k=None, qw=w, kw=None, p=pos, freq=f, **more):
        return lambda: norm_rotary(q, k, qw, kw, p, freq, **more)

    bad = [
        (RuntimeError, "must be a HIP", norm(torch.zeros(4, 2, 64))),
        (RuntimeError, "float32, bfloat16 or float16", norm(x.double())),
        (ValueError, "tokens, heads, dim", norm(x[0])),
        (ValueError, "must match q's", norm(x, b)),
        (ValueError, "k_weight needs k", norm(kw=w)),
        (ValueError, "q_weight must have shape", norm(qw=w[:63])),
        (RuntimeError, "q_weight must be on GPU", norm(qw=torch.ones(64))),
        (RuntimeError, "q_weight must be float32", norm(qw=w.double())),
        (RuntimeError, "q_weight must be float32", norm(b, qw=w.half())),
        (ValueError, "one type", norm(b, b, w, w.bfloat16())),
        (RuntimeError, "2 to 512", norm(torch.zeros(4, 2, 514, device=dev), qw=None)),
        (RuntimeError, "frequencies turn", norm(x[..., :32], qw=None)),
        (RuntimeError, "do not divide", norm(p=pos3)),
        (RuntimeError, "eps", norm(eps=-1.0)),
        (RuntimeError, "eps", norm(eps=float("nan"))),
        (ValueError, "unknown layout", norm(layout="other")),
        (ValueError, "unknown order", norm(sections=(32,), order="other")),
        (ValueError, "needs sections", norm(order="turns")),
        (ValueError, "one for each of the 3 axes", norm(p=pos3, sections=(16, 16))),
        (ValueError, "add up to the 32", norm(p=pos3, sections=(16, 16, 1))),
        (ValueError, "numbers of pairs", norm(p=pos3, sections=(16, 17, -1))),
        (ValueError, "add up to the 32", lambda: rotary(x, None, pos, f, sections=(31,))),
        (ValueError, "up to 256",
         lambda: rotary(torch.zeros(1, 1, 600, device=dev), None, pos[:1],
                        rotary_frequencies(600, device=dev), sections=(300,))),
        (RuntimeError, "frequencies must not require",
         norm(freq=f.clone().requires_grad_(True))),
        (RuntimeError, "must be a HIP", lambda: dropout(torch.zeros(3), 0.5, 1)),
        (RuntimeError, "float32, bfloat16 or float16", lambda: dropout(x.double(), 0.5, 1)),
        (ValueError, "between 0 and 1", lambda: dropout(x, 1.5, 1)),
        (ValueError, "between 0 and 1", lambda: dropout(x, float("nan"), 1)),
        (ValueError, "one shape", lambda: dropout(x, 0.5, 1, residual=x[0])),
        (RuntimeError, "residual must be float32", lambda: dropout(x, 0.5, 1, residual=b)),
        (RuntimeError, "residual must be float32", lambda: dropout(b, 0.5, 1, residual=b.half())),
        (ValueError, "0 to 2\\^64", lambda: dropout(x, 0.5, -1)),
        (ValueError, "0 to 2\\^64", lambda: dropout(x, 0.5, 2 ** 64)),
        (ValueError, "0 to 2\\^64", lambda: dropout(x, 0.5, 1, site=-1)),
        (ValueError, "one int64", lambda: dropout(x, 0.5, torch.zeros(2, dtype=torch.int64))),
        (ValueError, "one int64", lambda: dropout(x, 0.5, torch.zeros(1, device=dev))),
        (RuntimeError, "seed must be on", lambda: dropout(x, 0.5, torch.tensor([1]))),
    ]
    for kind, text, call in bad:
        with pytest.raises(kind, match=text):
            call()
