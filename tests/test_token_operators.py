"""The token operators' host side and index rules, on the CPU: what LDS place,
row and column every lane of the attention kernels' operands has, the frequency
tables, the C entries' refusals and the float64 restatements themselves."""

from __future__ import annotations

import math
import re

import numpy as np
import pytest
import torch

from oracle import token_ref
from test_kernel_indexes import _run


# ------------------------------------------------------------- index rules

@pytest.mark.parametrize("dk", [32, 64, 96, 128])
def test_fills_and_operands_agree_on_every_place(tmp_path, dk):
    rows = _run(tmp_path, "attention_tiles.h", f"""
        const int loads = 64 * tile_chunks<{dk}>() / 64;
        std::printf("%d\\n", tile_chunks<{dk}>());
        for (int i = 0; i < loads; ++i)
            for (int l = 0; l < 64; ++l)
                std::printf("0 %d %d %d\\n", (64 * i + l) * 16, fill_row<{dk}>(i, l),
                            fill_chunk<{dk}>(i, l));
        for (int r = 0; r < 64; r += 32)
            for (int s = 0; s < {dk} / 16; ++s)
                for (int l = 0; l < 64; ++l)
                    std::printf("1 %d %d %d %d\\n", row_operand_byte<{dk}>(row_lane_byte<{dk}>(l), r, s), r, s, l);
        for (int r = 0; r < 64; r += 8)
            for (int b = 0; b < {dk} / 32; ++b)
                for (int l = 0; l < 64; ++l)
                    std::printf("2 %d %d %d %d\\n", column_operand_byte<{dk}>(column_lane_byte<{dk}>(l), r, b), r, b, l);""")
    chunks = rows[0][0]
    place = {}
    for _, byte, r, c in (x for x in rows[1:] if x[0] == 0):
        assert byte not in place and 0 <= r < 64 and 0 <= c < chunks
        place[byte] = (r, c)
    assert sorted(place) == list(range(0, 64 * chunks * 16, 16))
    assert len(set(place.values())) == len(place)
    for _, byte, r, s, l in (x for x in rows[1:] if x[0] == 1):
        assert place[byte] == (r + l % 32, 2 * s + l // 32)
    banks = {}
    for _, byte, r, b, l in (x for x in rows[1:] if x[0] == 2):
        # Lane l of 16 hands over row l / 4 and columns 4 (l % 4) .. of its 16.
        want_row = r + 4 * (l // 32) + l % 16 // 4
        want_col = 32 * b + 16 * (l // 16 % 2) + 4 * (l % 4)
        at, within = byte - byte % 16, byte % 16
        assert place[at] == (want_row, want_col // 8) and within == want_col % 8 * 2
        banks.setdefault((r, b, l // 32), []).append(byte % 256)
    for seen in banks.values():
        assert len(set(seen)) == 32, "32 lanes' reads of 8 bytes spread over 256"


@pytest.mark.parametrize("dk", [32, 64, 96, 128])
def test_rows_read_together_lie_in_different_banks(tmp_path, dk):
    rows = _run(tmp_path, "attention_tiles.h", f"""
        for (int s = 0; s < {dk} / 16; ++s)
            for (int l = 0; l < 64; ++l) std::printf("%d\\n", row_operand_byte<{dk}>(row_lane_byte<{dk}>(l), 0, s));""")
    at = [r[0] % 256 for r in rows]
    for i in range(0, len(at), 16):
        assert len(set(at[i:i + 16])) == (16 if dk > 64 else 8)


def test_a_products_rows_are_the_next_ones_operand(tmp_path):
    """Elements 8 s .. 8 s + 7 of a product are rows 16 s + 4 h + {0..3} and 16 s + 8 +
    4 h + {0..3}: what two transposing reads from rows 16 s and 16 s + 8 give."""
    rows = _run(tmp_path, "attention_tiles.h",
                'for (int h = 0; h < 2; ++h) for (int e = 0; e < 16; ++e) '
                'std::printf("%d %d %d\\n", h, e, c_row(e, h));')
    for h, e, r in rows:
        s, j = divmod(e, 8)
        assert r == 16 * s + 8 * (j // 4) + 4 * h + j % 4
    assert sorted(r for _, _, r in rows) == list(range(32))


def test_runs_are_even_where_they_can_be(tmp_path):
    cases = [(r, g, m) for g in range(1, 20) for m in (1, 4, 8) for r in range(1, m + 1)]
    rows = _run(tmp_path, "attention_tiles.h", "".join(
        f'std::printf("%d\\n", even_runs({r}, {g}, {m}));' for r, g, m in cases))
    for (r, g, m), (got,) in zip(cases, rows):
        assert 1 <= got <= m
        if got % g and g % got:                      # uneven: no even number was left
            assert got == r and all(g % n for n in range(r, m + 1))


# ------------------------------------------------------------- frequencies

def test_frequencies():
    from metal_gauss_amd import rotary_frequencies

    f = rotary_frequencies(8, device="cpu")
    assert f.dtype == torch.float64
    assert np.allclose(f, [10000.0 ** (-i / 4) for i in range(4)], rtol=1e-14)
    assert torch.equal(rotary_frequencies(16, axes=2, device="cpu"), f.repeat(2))
    assert np.allclose(rotary_frequencies(8, scaling="linear", factor=4.0, device="cpu"), f / 4)
    b = rotary_frequencies(8, scaling="base", factor=4.0, device="cpu")
    assert b[0] == 1.0 and math.isclose(float(b[-1]), float(f[-1]) / 4, rel_tol=1e-12)
    f = rotary_frequencies(64, device="cpu")
    c = rotary_frequencies(64, scaling="bands", factor=8.0, original_length=2048, device="cpu")
    turns = 2048 * f / (2 * math.pi)
    assert torch.equal(c[turns >= 32], f[turns >= 32])
    assert np.allclose(c[turns <= 1], f[turns <= 1] / 8)
    assert bool(((c <= f) & (c >= f / 8 * (1 - 1e-12))).all()) and bool((c[1:] < c[:-1]).all())


@pytest.mark.parametrize("args,kw", [((7,), {}), ((0,), {}), ((8,), {"axes": 3}),
                                     ((8,), {"scaling": "other"}), ((8,), {"scaling": "bands"}),
                                     ((8,), {"factor": 0.0})])
def test_frequencies_refusals(args, kw):
    from metal_gauss_amd import rotary_frequencies

    with pytest.raises(ValueError):
        rotary_frequencies(*args, device="cpu", **kw)


# ------------------------------------------------------------ C entry points

def _attn(lib, dtype=1, nq=4, nk=4, heads=2, kv=2, dim=64, q=16, stride=64, off=None, n=1,
          scale=1.0, out=16, ws=None, ws_bytes=0):
    return lib.mg_attention_forward(dtype, nq, nk, heads, kv, dim, q, stride, 64, 16, stride, 64,
                                    16, stride, 64, off, off, n, 0, scale, out, None, None,
                                    ws, ws_bytes, None)


def test_refusals_before_any_launch():
    from metal_gauss_amd import _lib

    lib = _lib.open_library()

    def refused(rc, text):
        assert rc == 1 and text in lib.mg_last_error().decode(), lib.mg_last_error()

    refused(lib.mg_layer_norm_forward(1, 0, 0, 16, 8, 0, None, None, 1e-5, 16, None, None, None),
            "rows of 0 elements")
    refused(lib.mg_layer_norm_forward(1, 8, 7, 16, 8, 7, None, None, 1e-5, 16, None, None, None),
            "type code 7")
    refused(lib.mg_layer_norm_forward(1, 8, 0, 16, 8, 1, None, None, 1e-5, 16, None, None, None),
            "weights must be float32 or of the input's type")
    refused(lib.mg_layer_norm_forward(1, 8, 0, None, 8, 0, None, None, 1e-5, 16, None, None, None),
            "x and y")
    refused(lib.mg_layer_norm_forward(1, 8, 0, 16, 8, 0, None, None, 1e-5, 16, 16, None, None),
            "go together")
    refused(lib.mg_layer_norm_backward(9, 8, 0, 16, 8, 16, 8, 0, None, 16, 16, 16, 16, None, 16,
                                       8, None), "workspace of 8 bytes")
    refused(lib.mg_rotary(4, 0, 16, 64, 64, 1, None, 0, 0, 0, 64, 16, 0, 3, 16, 32, 0, 0, 16,
                          None, None), "do not divide")
    refused(lib.mg_rotary(4, 0, 16, 64, 64, 1, None, 0, 0, 0, 62, 16, 0, 1, 16, 32, 0, 0, 16,
                          None, None), "frequencies turn")
    refused(lib.mg_rotary(4, 0, 16, 64, 64, 1, None, 0, 0, 1, 64, 16, 0, 1, 16, 32, 0, 0, 16,
                          None, None), "NULL")
    refused(_attn(lib, dtype=0), "bfloat16 or float16")
    refused(_attn(lib, dim=60), "multiples of 8")
    refused(_attn(lib, dim=136), "up to 128")
    refused(_attn(lib, heads=3), "no multiple")
    refused(_attn(lib, q=8), "16-byte aligned")
    refused(_attn(lib, stride=68), "16-byte aligned")
    refused(_attn(lib, stride=1 << 24), "token strides")
    refused(_attn(lib, n=2), "without offsets")
    refused(_attn(lib, scale=-1.0), "scale")
    refused(_attn(lib, scale=float("nan")), "scale")
    refused(_attn(lib, out=None), "NULL")
    refused(_attn(lib, nk=100000), "workspace")
    refused(lib.mg_attention_backward(1, 4, 4, 2, 2, 64, 16, 64, 64, 16, 64, 64, 16, 64, 64, None,
                                      None, 1, 0, 1.0, 16, None, 16, 16, 64, 64, 16, 16, None,
                                      16, 1 << 20, None), "go together")
    refused(lib.mg_attention_backward(1, 4, 4, 2, 2, 64, 16, 64, 64, 16, 64, 64, 16, 64, 64, None,
                                      None, 1, 0, 1.0, 16, None, 16, 16, 64, 64, 16, 16, 16,
                                      16, 8, None), "workspace of 8 bytes")


def test_launches_of_more_threads_than_are_counted_are_refused():
    """Before the launch: 2^32 threads are too many."""
    from metal_gauss_amd import _lib

    lib = _lib.open_library()

    def refused(rc, text):
        assert rc == 1 and text in lib.mg_last_error().decode(), lib.mg_last_error()

    off, many = 16, 1 << 24          # one work item a sequence and head at least
    refused(_attn(lib, nq=many, nk=many, heads=4, kv=4, off=off, n=many), "too many work items")
    for n, kv in ((many, 1), (many // 8, 8)):
        refused(lib.mg_attention_backward(2, n, n, kv, kv, 64, 16, 64, 64, 16, 64, 64, 16, 64, 64,
                                          off, off, n, 0, 1.0, 16, None, 16, 16, 64, 64, 16, 16,
                                          16, 16, 1 << 50, None), "too many work items")
    refused(lib.mg_layer_norm_forward(1 << 22, 16385, 0, 16, 16385, 0, None, None, 1e-5, 16, None,
                                      None, None), "too many for one call")
    refused(lib.mg_rotary(1 << 24, 1, 16, 2046, 1023, 2, None, 0, 0, 0, 1023, 16, 0, 1, 16, 32, 0,
                          0, 16, None, None), "too many for one call")


def test_workspace_queries():
    from metal_gauss_amd import _lib

    lib = _lib.open_library()
    # Rows that fill the GPU take none, few rows over many keys do.
    assert lib.mg_attention_forward_workspace_bytes(100000, 100000, 16, 16, 64, 1) == 0
    few = lib.mg_attention_forward_workspace_bytes(16, 75000, 16, 4, 64, 16)
    assert 0 < few < 1 << 28
    assert lib.mg_attention_backward_workspace_bytes(1000, 5, 4, 2, 64, 1) >= 4 * 4000
    assert lib.mg_layer_norm_backward_workspace_bytes(1, 100) >= 800
    assert lib.mg_layer_norm_backward_workspace_bytes(0, 100) == 0


def test_rotary_refuses_tokens_of_more_elements_than_are_counted():
    """Before any launch: 65537 heads of 65536 elements pass 32 bits."""
    from metal_gauss_amd import _lib

    lib = _lib.open_library()
    for heads, k_heads in ((65536, 1), (16384, 1), (65536, 65536)):
        rc = lib.mg_rotary(1, 0, None, 65536, 65536, heads, None, 65536, 65536, k_heads, 65536,
                           None, 0, 1, None, 32, 0, 0, None, None, None)
        assert rc == 1 and "too long" in lib.mg_last_error().decode(), lib.mg_last_error()


@pytest.mark.parametrize("streams,heads,kv,keys", [(384, 32, 1, 1000), (128, 32, 1, 4096),
                                                   (64, 32, 8, 4096), (300, 8, 1, 800)])
def test_workspace_of_single_tokens_over_many_memories(streams, heads, kv, keys):
    """Partial results of at most 1536 items at once and two more chunks a sequence
    and head, of 32 rows of 128 columns: eight times that is the most asked for."""
    from metal_gauss_amd import _lib

    lib = _lib.open_library()
    need = lib.mg_attention_forward_workspace_bytes(streams, streams * keys, heads, kv, 128,
                                                    streams)
    assert 0 < need <= 8 * (1536 + 2 * streams * kv) * 32 * 128 * 4


# ----------------------------------------------------------------- autograd

def test_a_backward_pass_refuses_tangents():
    """The decorator of the operators' backward passes: a gradient with a tangent is
    refused, one without is passed on, and second derivatives are refused."""
    import torch.autograd.forward_ad as fw
    from metal_gauss_amd import _lib

    class Twice(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            return 2.0 * x

        @staticmethod
        @_lib.differentiable_once
        def backward(ctx, dy):
            return torch.from_numpy(2.0 * dy.detach().numpy())

    x = torch.randn(4).requires_grad_(True)
    dy = torch.ones(4)
    assert not _lib.forward_mode()
    assert torch.equal(torch.autograd.grad(Twice.apply(x), x, dy)[0], 2.0 * dy)
    with fw.dual_level():
        assert _lib.forward_mode()
        assert torch.equal(torch.autograd.grad(Twice.apply(x), x, dy)[0], 2.0 * dy)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(Twice.apply(x), x, fw.make_dual(dy, dy))
    dx, = torch.autograd.grad(Twice.apply(x).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dx.sum().backward()


# ---------------------------------------------------- the oracle's own checks

def _difference(f, x, d):
    return (f(x + 1e-6 * d) - f(x - 1e-6 * d)) / 2e-6


def test_oracle_gradients_are_their_values_differences():
    g = np.random.default_rng(0)
    x, w, dy, d = g.standard_normal((4, 3, 9))
    w = w[0]
    dx, dw, db = token_ref.layer_norm_grad(x, w, dy)
    at = lambda a, b, c: (token_ref.layer_norm(a, b, c) * dy).sum()  # noqa: E731
    assert abs(_difference(lambda a: at(a, w, 0 * w), x, d) - (dx * d).sum()) < 1e-8
    assert abs(_difference(lambda b: at(x, b, 0 * w), w, d[0]) - (dw * d[0]).sum()) < 1e-8
    assert abs(_difference(lambda c: at(x, w, c), w, d[0]) - (db * d[0]).sum()) < 1e-8
    for causal in (False, True):
        qo, ko = [0, 4, 4, 7], [0, 3, 5, 8]
        t = [g.standard_normal(s) for s in ((7, 4, 8), (8, 2, 8), (8, 2, 8))]
        do = g.standard_normal((7, 4, 8))
        (_, *grads), _ = token_ref.attention(*t, qo, ko, causal, 0.4, do)
        for i in range(3):
            d = g.standard_normal(t[i].shape)
            f = lambda x: (token_ref.attention(  # noqa: E731
                *[x if j == i else t[j] for j in range(3)], qo, ko, causal, 0.4)[0][0] * do).sum()
            assert abs(_difference(f, t[i], d) - (grads[i] * d).sum()) < 1e-7


def test_oracle_against_torch():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(5, 12, generator=g, dtype=torch.float64)
    w, b = torch.randn(2, 12, generator=g, dtype=torch.float64)
    assert np.allclose(token_ref.layer_norm(x.numpy(), w.numpy(), b.numpy()),
                       torch.nn.functional.layer_norm(x, (12,), w, b), atol=1e-13)
    q = torch.randn(6, 2, 8, generator=g, dtype=torch.float64)
    k, v = torch.randn(2, 6, 2, 8, generator=g, dtype=torch.float64)
    want = torch.nn.functional.scaled_dot_product_attention(
        q.transpose(0, 1), k.transpose(0, 1), v.transpose(0, 1), is_causal=True).transpose(0, 1)
    got, _ = token_ref.attention(q.numpy(), k.numpy(), v.numpy(), [0, 6], [0, 6], True, 8 ** -0.5)
    assert np.allclose(got[0], want, atol=1e-13)


def test_oracle_rotation_keeps_lengths_and_turns_back():
    g = np.random.default_rng(2)
    x, pos = g.standard_normal((5, 2, 12)), g.integers(0, 99, (5, 2))
    for layout in ("half", "interleaved"):
        y = token_ref.rotary(x, pos, np.array([1.0, 0.1, 1.0, 0.1]), layout)
        assert np.allclose((y ** 2).sum(-1), (x ** 2).sum(-1))
        assert np.array_equal(y[..., 8:], x[..., 8:])
        back = token_ref.rotary(y, pos, np.array([1.0, 0.1, 1.0, 0.1]), layout, inverse=True)
        assert np.allclose(back, x)


# ------------------------------------------------------------ compiled loads

def unready_lds_loads(lines):
    """Loads into LDS in straight code less than five wait states after a vector
    instruction wrote a scalar they read, or less than one after m0 was written."""
    bad = []
    for i, line in enumerate(lines):
        if not (line.startswith("buffer_load") and line.endswith(" lds")):
            continue
        first, last = map(int, re.search(r"s\[(\d+):(\d+)\]", line).groups())
        states, m0 = 0, None
        for back in range(i - 1, max(i - 12, -1), -1):
            s = lines[back]
            if m0 is None and re.match(r"s_\w+ m0,", s):
                m0 = states
            to = re.match(r"v_\w+ s(?:(\d+)|\[(\d+):(\d+)\])", s)
            if to and states < 5:
                lo = int(to.group(1) or to.group(2))
                hi = int(to.group(1) or to.group(3))
                if lo <= last and hi >= first:
                    bad.append((s, line))
            nop = re.match(r"s_nop (\d+)", s)
            states += int(nop.group(1)) + 1 if nop else 1
        if m0 is None or m0 < 1:
            bad.append(("m0", line))
    return bad


@pytest.mark.parametrize("source", ["attention.hip", "attention_bwd.hip"])
def test_tile_loads_wait_for_their_scalars(tmp_path, source):
    """The loads into LDS are assembly that the compiler's hazard pass does not
    look into."""
    from test_lds_barrier_audit import _assemble, _build_module

    out = _assemble(_build_module().CSRC / source, tmp_path / "out.s", source)
    lines = [s.split(";")[0].strip() for s in out.read_text().splitlines()]
    lines = [s for s in lines if s and not s.startswith(".") and not s.endswith(":")]
    assert sum(s.endswith(" lds") for s in lines) > 50
    assert not unready_lds_loads(lines)


def test_the_check_flags_a_descriptor_just_written():
    load = "buffer_load_dwordx4 v1, s[8:11], 0 offen lds"
    wait = ["s_mov_b32 m0, s2", "s_nop 0"]
    assert unready_lds_loads(["v_readfirstlane_b32 s9, v3", *wait, load])
    assert unready_lds_loads(["v_cmp_eq_u32_e64 s[10:11], v3, v4", *wait, load])
    assert not unready_lds_loads(["v_readfirstlane_b32 s12, v3", *wait, load])
    assert not unready_lds_loads(["v_readfirstlane_b32 s9, v3", "s_mov_b32 m0, s2", "s_nop 4", load])
    assert unready_lds_loads(["s_nop 4", "s_mov_b32 m0, s2", load])


def undeclared_m0(text):
    """Assembly statements that write m0 and do not say so."""
    bad = []
    for start in re.finditer(r"\basm\b[^(;]*\(", text):
        depth, at = 1, start.end()
        while depth:
            depth += {"(": 1, ")": -1}.get(text[at], 0)
            at += 1
        statement = text[start.end():at - 1]
        if re.search(r"s_\w+ m0,", statement) and '"m0"' not in statement.rpartition(":")[2]:
            bad.append(statement)
    return bad


def test_assembly_that_writes_m0_says_so():
    """The compiler may hold a value of its own there."""
    from test_lds_barrier_audit import _build_module

    sources = [p for p in sorted(_build_module().CSRC.iterdir()) if p.suffix in (".h", ".hip")]
    texts = {p.name: p.read_text() for p in sources}
    assert sum(len(re.findall(r"s_\w+ m0,", t)) for t in texts.values()) >= 3
    assert not {n: u for n, t in texts.items() if (u := undeclared_m0(t))}


def test_the_check_flags_an_undeclared_m0():
    write = 'asm volatile("s_mov_b32 m0, %0\\n\\t" "buffer_load_dword %1, %2, 0 offen lds" : : "s"(f((int)a)), "v"(b)'
    assert undeclared_m0(write + ");")
    assert undeclared_m0(write + ' : "memory");')
    assert not undeclared_m0(write + ' : "m0", "memory");')
    assert not undeclared_m0('asm volatile("s_waitcnt vmcnt(0)" ::: "memory");')


@pytest.mark.parametrize("source", ["attention.hip", "attention_bwd.hip"])
def test_m0_is_for_the_tile_loads_alone(tmp_path, source):
    """Nothing else in the compiled kernels reads or writes it."""
    from test_lds_barrier_audit import _assemble, _build_module

    out = _assemble(_build_module().CSRC / source, tmp_path / "out.s", source)
    lines = [s.split(";")[0].strip() for s in out.read_text().splitlines()]
    lines = [s for s in lines if s and not s.startswith(".") and not s.endswith(":")]
    at = [i for i, s in enumerate(lines) if re.search(r"\bm0\b", s)]
    assert len(at) > 50
    for i in at:
        assert re.fullmatch(r"s_mov_b32 m0, (s\d+|vcc_lo|vcc_hi)", lines[i])
        assert re.fullmatch(r"s_nop \d", lines[i + 1]) and lines[i + 2].endswith(" lds"), lines[i]
