"""The operators of networks over frames on the CPU: the C entries' refusals, the
room for partial results, the axes of pairs, the compiled loads, and the float64
restatements themselves."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from oracle import token_ref
from test_token_operators import unready_lds_loads


def refused(lib, rc, text):
    assert rc == 1 and text in lib.mg_last_error().decode(), lib.mg_last_error()


# ------------------------------------------------------------ C entry points

def _norm_rotary(lib, tokens=4, dtype=1, heads=2, kv=1, dim=64, wtype=0, eps=1e-6, axes=1,
                 axis_of=None, pairs=32, q=16, out=16):
    return lib.mg_norm_rotary_forward(tokens, dtype, q, 128, 64, heads, 16, 128, 64, kv, dim, wtype,
                                      None, None, eps, 16, 0, axes, axis_of, 16, pairs, 0, out, 16,
                                      None)


def _norm_rotary_grad(lib, tokens=4, heads=2, kv=1, dq=16, dk=16, dqw=16, dkw=16, ws=16,
                      size=1 << 24):
    return lib.mg_norm_rotary_backward(tokens, 1, 16, 128, 64, heads, 16, 128, 64, kv, 64, 0, None,
                                       None, 1e-6, 16, 0, 1, None, 16, 32, 0, 16, 128, 64, 16, 128,
                                       64, dq, dk, dqw, dkw, ws, size, None)


def test_heads_that_are_refused_before_any_launch():
    from metal_gauss_amd import _lib

    lib = _lib.open_library()
    axes = ctypes.create_string_buffer(bytes([0] * 31 + [3]), 32)
    for text, kw in (("type code 7", dict(dtype=7)), ("weights must be float32", dict(wtype=2)),
                     ("tokens", dict(tokens=-1)), ("and 1 heads", dict(heads=-1)),
                     ("0 and 0 heads", dict(heads=0, kv=0)), ("2 to 512", dict(dim=513)),
                     ("2 to 512", dict(dim=1)), ("frequencies turn", dict(pairs=33)),
                     ("frequencies turn", dict(pairs=0)), ("do not divide", dict(axes=3)),
                     ("pair's axis", dict(axes=3, axis_of=axes)), ("eps", dict(eps=-1.0)),
                     ("eps", dict(eps=float("nan"))), ("NULL", dict(q=None)),
                     ("NULL", dict(out=None))):
        refused(lib, _norm_rotary(lib, **kw), text)
    assert _norm_rotary(lib, tokens=0) == 0
    refused(lib, _norm_rotary_grad(lib, tokens=0), "of no tokens are zeros")
    refused(lib, _norm_rotary_grad(lib, kv=0), "gradients of no heads")
    refused(lib, _norm_rotary_grad(lib, size=8), "workspace of 8 bytes")
    refused(lib, _norm_rotary_grad(lib, ws=None), "workspace")
    assert _norm_rotary_grad(lib, dq=None, dk=None, dqw=None, dkw=None) == 0
    refused(lib, lib.mg_rotary_axes(4, 0, 16, 64, 64, 1, None, 0, 0, 0, 64, 16, 0, 3, axes, 16, 32, 0,
                                    0, 16, None, None), "by one of the 3 axes")
    refused(lib, lib.mg_rotary_axes(4, 0, 16, 64, 64, 1, None, 0, 0, 0, 64, 16, 0, 3, None, 16, 32, 0,
                                    0, 16, None, None), "axes are NULL")
    refused(lib, lib.mg_rotary_axes(4, 0, 16, 600, 600, 1, None, 0, 0, 0, 600, 16, 0, 1, axes, 16,
                                    300, 0, 0, 16, None, None), "at most 256")


@pytest.mark.parametrize("q_heads,k_heads,dim", [(1, 0, 2), (16, 4, 128), (65536, 65536, 511),
                                                 (7, 3, 512), (4096, 1, 64)])
def test_room_for_the_weights_sums(q_heads, k_heads, dim):
    """Two rows a workgroup: 1024 of them, or one for each four heads of a token."""
    from metal_gauss_amd import _lib

    need = _lib.open_library().mg_norm_rotary_backward_workspace_bytes(q_heads, k_heads, dim)
    assert need >= 8 * dim * max(1024, (q_heads + k_heads + 3) // 4)


def test_dropout_refused_before_any_launch():
    from metal_gauss_amd import _lib

    lib = _lib.open_library()

    def call(n=8, dtype=1, out=1, drop=9, residual=None, x=16, y=16):
        return lib.mg_dropout(n, dtype, x, out, residual, y, drop, 1, None, 0, None)

    refused(lib, call(dtype=5), "type codes")
    refused(lib, call(dtype=1, out=2), "must be float32")
    refused(lib, call(dtype=0, out=1, residual=16), "residual")
    refused(lib, call(drop=65537), "65537 of 65536")
    refused(lib, call(drop=-1), "-1 of 65536")
    refused(lib, call(n=-1), "-1 elements")
    refused(lib, call(n=1 << 36), "too many for one call")
    refused(lib, call(x=None), "NULL")
    assert call(n=0, x=None) == 0


def _window(lib, window=5, sinks=0, nq=4, nk=4, n=1, off=None, ws=None, size=0):
    return lib.mg_attention_window_forward(1, nq, nk, 2, 2, 64, 16, 128, 64, 16, 128, 64, 16, 128, 64,
                                           off, off, n, window, sinks, 1.0, 16, None, None, ws, size,
                                           None)


def test_windows_refused_before_any_launch():
    from metal_gauss_amd import _lib

    lib = _lib.open_library()
    refused(lib, _window(lib, window=0), "a window of 0 keys")
    refused(lib, _window(lib, window=-3), "a window of -3 keys")
    refused(lib, _window(lib, sinks=-1), "and -1 first ones")
    refused(lib, _window(lib, window=3000, nk=100000), "workspace")
    refused(lib, lib.mg_attention_window_backward(
        1, 100, 100, 2, 2, 64, 16, 128, 64, 16, 128, 64, 16, 128, 64, None, None, 1, 9, 3, 1.0, 16,
        None, 16, 16, 128, 64, 16, 16, 16, 16, 8, None), "workspace of 8 bytes")
    many = 1 << 25
    refused(lib, _window(lib, nq=many, nk=many, n=many, off=16), "too many work items")
    for query in (lib.mg_attention_window_forward_workspace_bytes,
                  lib.mg_attention_window_backward_workspace_bytes):
        assert query(4, 4, 2, 2, 64, 1, 0, 0) == 0 and query(4, 4, 2, 2, 64, 1, 3, -1) == 0


def test_room_of_windows():
    """It goes by the window, not by the memories; sinks take places by the queries."""
    from metal_gauss_amd import _lib

    lib = _lib.open_library()
    short, long = (lib.mg_attention_window_forward_workspace_bytes(16, keys, 16, 4, 64, 16, 2000, 4)
                   for keys in (16 * 4000, 16 * 10 ** 6))
    assert 0 < short == long < 1 << 27
    whole = lib.mg_attention_forward_workspace_bytes(16, 16 * 4000, 16, 4, 64, 16)
    assert lib.mg_attention_window_forward_workspace_bytes(16, 16 * 4000, 16, 4, 64, 16, 10 ** 9,
                                                           4) == whole
    none, some = (lib.mg_attention_window_backward_workspace_bytes(16320, 16320, 16, 4, 128, 1, 1900,
                                                                   sinks) for sinks in (0, 16))
    assert none < some < none + (64 << 20)


def _shared(lib, nq=4, nk=4, ns=4, heads=2, kv=2, dim=64, n=1, groups=1, off=None, goff=None, q=16,
            sk=16, stride=128, scale=1.0, ws=None, size=0):
    return lib.mg_shared_attention(1, nq, nk, ns, heads, kv, dim, q, 128, 64, 16, 128, 64, 16, 128,
                                   64, sk, stride, 64, 16, 128, 64, off, off, n, goff, goff, groups,
                                   1, scale, 16, ws, size, None)


def test_shared_refused_before_any_launch():
    from metal_gauss_amd import _lib

    lib = _lib.open_library()
    refused(lib, _shared(lib, heads=3), "no multiple")
    refused(lib, _shared(lib, dim=60), "multiples of 8")
    refused(lib, _shared(lib, ns=1 << 30), "shared tokens")
    refused(lib, _shared(lib, n=2), "without offsets")
    refused(lib, _shared(lib, groups=2), "without offsets")
    refused(lib, _shared(lib, stride=100), "16-byte aligned")
    refused(lib, _shared(lib, sk=8), "16-byte aligned")
    refused(lib, _shared(lib, scale=-1.0), "scale")
    refused(lib, _shared(lib, q=None), "NULL")
    refused(lib, _shared(lib, sk=None), "NULL")
    refused(lib, _shared(lib), "workspace of 0 bytes")
    refused(lib, _shared(lib, nq=1 << 25, n=1 << 25, off=16, kv=2), "too many work items")
    assert _shared(lib, nq=0) == 0
    query = lib.mg_shared_attention_workspace_bytes
    assert query(4, 4, 4, 2, 2, 64, 0, 1) == 0 and query(4, 4, 4, 2, 2, 64, 1, 0) == 0
    # Two sets of partial results: 128 streams in 33 chunks at most.
    assert 0 < query(128, 32000, 16320, 16, 4, 128, 128, 1) < 128 * 16 * 66 * (128 * 4 + 8) + 4096


# ------------------------------------------------------------------- pairs

@pytest.mark.parametrize("sections,order,want", [
    ((2, 3), "runs", [0, 0, 1, 1, 1]), ((2, 3), "turns", [0, 1, 0, 1, 1]),
    ((1, 0, 3), "turns", [0, 2, 2, 2]), ((4,), "turns", [0] * 4),
    ((2, 2, 2), "turns", [0, 1, 2, 0, 1, 2])])
def test_axes_of_pairs(sections, order, want):
    from metal_gauss_amd.rotary import _table

    assert list(_table(sections, order).raw) == want == token_ref.axes_of(sections, order)


def test_sections_that_are_refused():
    from metal_gauss_amd.rotary import axis_table

    pos, freq = torch.zeros(4, 2, dtype=torch.int32), torch.zeros(8, dtype=torch.float64)
    assert axis_table(None, "runs", pos, freq) is None
    assert len(axis_table([3, 5], "turns", pos, freq)) == 8
    for sections, order, text in (((4, 4), "other", "unknown order"), (None, "turns", "needs"),
                                  ((8,), "runs", "each of the 2 axes"), ((4, 5), "runs", "add up"),
                                  ((-1, 9), "runs", "numbers of pairs"), ((), "runs", "numbers"),
                                  ((0, 0), "runs", "numbers"), ((128, 129), "runs", "up to 256")):
        with pytest.raises(ValueError, match=text):
            axis_table(sections, order, pos, freq)


# --------------------------------------------------------------- the oracle

def test_generator_against_its_publications_answers():
    """The known answers of Philox4x32-10: counters and keys of zeros, of ones, and of
    the digits of pi."""
    for counter, key, want in (
            ((0,) * 4, (0,) * 2, "6627e8d5 e169c58d bc57ac4c 9b00dbd8"),
            ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, "408f276d 41c83b0e a20bc7c6 6d5451fd"),
            ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
             "d16cfe09 94fdcceb 5001e420 24126ea1")):
        assert " ".join(f"{w:08x}" for w in token_ref.philox4x32(counter, key)) == want


def test_oracle_gradients_are_their_values_differences():
    g = np.random.default_rng(0)
    x, dy, d = g.standard_normal((3, 2, 3, 10))
    w, e = g.standard_normal((2, 10))
    pos, freq = g.integers(0, 9, (2, 2)), np.array([1.0, 0.3, 0.1, 0.05])
    turn = lambda t: token_ref.rotary_axes(t, pos, freq, "half", [0, 1, 0, 1])  # noqa: E731
    back = lambda t: token_ref.rotary_axes(t, pos, freq, "half", [0, 1, 0, 1], True)  # noqa: E731
    dx, dw = token_ref.norm_rotary_grad(x, w, 1e-3, back, dy)
    at = lambda a, b: (token_ref.norm_rotary(a, b, 1e-3, turn) * dy).sum()  # noqa: E731
    num = (at(x + 1e-6 * d, w) - at(x - 1e-6 * d, w)) / 2e-6
    assert abs(num - (dx * d).sum()) < 1e-8
    num = (at(x, w + 1e-6 * e) - at(x, w - 1e-6 * e)) / 2e-6
    assert abs(num - (dw * e).sum()) < 1e-8


def test_oracle_windows():
    seen = token_ref.sees(4, 6, True, 2, 1)
    assert seen.astype(int).tolist() == [[1, 1, 1, 0, 0, 0], [1, 0, 1, 1, 0, 0], [1, 0, 0, 1, 1, 0],
                                         [1, 0, 0, 0, 1, 1]]
    g = np.random.default_rng(1)
    t = [g.standard_normal(s) for s in ((7, 2, 8), (9, 1, 8), (9, 1, 8))]
    do = g.standard_normal((7, 2, 8))
    value = lambda x: (token_ref.attention(*x, [0, 4, 7], [0, 6, 9], True, 0.4,  # noqa: E731
                                           window=2, sinks=1)[0][0] * do).sum()
    (_, *grads), _ = token_ref.attention(*t, [0, 4, 7], [0, 6, 9], True, 0.4, do, window=2, sinks=1)
    for i in range(3):
        d = g.standard_normal(t[i].shape)
        up, down = list(t), list(t)
        up[i], down[i] = t[i] + 1e-6 * d, t[i] - 1e-6 * d
        assert abs((value(up) - value(down)) / 2e-6 - (grads[i] * d).sum()) < 1e-7


def test_oracle_shared_is_attention_over_both():
    g = np.random.default_rng(2)
    q, k, v, sk, sv = (g.standard_normal(s) for s in ((3, 2, 8), (4, 1, 8), (4, 1, 8), (5, 1, 8),
                                                      (5, 1, 8)))
    got, _ = token_ref.shared_attention(q, k, v, sk, sv, [0, 3], [0, 4], [0, 3], [0, 5], True, 0.3)
    want, _ = token_ref.attention(q, np.concatenate([sk, k]), np.concatenate([sv, v]), [0, 3], [0, 9],
                                  True, 0.3)
    assert np.allclose(got, want[0], atol=1e-13)


# ------------------------------------------------------------ compiled loads

def test_tile_loads_wait_for_their_scalars(tmp_path):
    """As in the other attention kernels: assembly that the compiler's hazard pass
    does not look into."""
    from test_lds_barrier_audit import _assemble, _build_module

    source = "attention_shared.hip"
    out = _assemble(_build_module().CSRC / source, tmp_path / "out.s", source)
    lines = [s.split(";")[0].strip() for s in out.read_text().splitlines()]
    lines = [s for s in lines if s and not s.startswith(".") and not s.endswith(":")]
    assert sum(s.endswith(" lds") for s in lines) > 50
    assert not unready_lds_loads(lines)
