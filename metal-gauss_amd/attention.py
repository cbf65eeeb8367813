"""Attention over packed sequences on the GPU, forward and backward
(mg_attention_*).

The reference has no counterpart: this is one of the operators of a network
that predicts or refines splats, next to ``layer_norm`` and ``rotary``.
"""

from __future__ import annotations

import torch

from . import _lib


def _rows(x: torch.Tensor):
    """x, or a copy of it whose rows lie as the kernels read them (contiguous and
    16-byte aligned; slices of a projection do as they are), with its pointer,
    token stride and head stride."""
    tok, head, one = x.stride()
    tokens, heads, _ = x.shape
    if tokens <= 1:
        tok = 0
    if heads <= 1:
        head = 0
    at = x.data_ptr()
    if one != 1 or at % 16 or tok % 8 or head % 8 or tok >= 1 << 24:
        x = x.clone(memory_format=torch.contiguous_format)
        at, tok, head = x.data_ptr(), x.stride(0), x.stride(1)
    return x, (at if tokens else None, tok, head)


def _forward(q, k, v, q_offsets, k_offsets, causal, scale, keep):
    lib = _lib.load()
    (q, q_at), (k, k_at), (v, v_at) = _rows(q), _rows(k), _rows(v)
    Tq, Hq, D = q.shape
    Tk, Hk, _ = k.shape
    n = 1 if q_offsets is None else q_offsets.numel() - 1
    # With a backward pass ahead, what rounding takes from the result is kept too.
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    rest = torch.empty_like(out) if keep else None
    lse = torch.empty(Hq, Tq, device=q.device) if keep else None
    need = lib.mg_attention_forward_workspace_bytes(Tq, Tk, Hq, Hk, D, n)
    ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    _lib.launch(lib.mg_attention_forward, q.get_device(), _lib.TYPE_CODES[q.dtype], Tq, Tk, Hq,
                Hk, D, *q_at, *k_at, *v_at,
                None if q_offsets is None else q_offsets.data_ptr(),
                None if k_offsets is None else k_offsets.data_ptr(), n, causal, scale,
                out.data_ptr(), rest.data_ptr() if keep else None,
                lse.data_ptr() if keep else None,
                ws.data_ptr() if need else None, need)
    return out, rest, lse, q, k, v


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, q_offsets, k_offsets, causal, scale):
        out, rest, lse, q, k, v = _forward(q, k, v, q_offsets, k_offsets, causal, scale, True)
        ctx.save_for_backward(q, k, v, q_offsets, k_offsets, out, rest, lse)
        ctx.causal, ctx.scale = causal, scale
        return out

    @staticmethod
    @_lib.differentiable_once
    def backward(ctx, dout):
        # Hooks on saved tensors may give them back in another layout.
        q, k, v, *others = ctx.saved_tensors
        q_offsets, k_offsets, out, rest, lse = (
            None if t is None else t.contiguous() for t in others)
        (q, q_at), (k, k_at), (v, v_at) = _rows(q), _rows(k), _rows(v)
        lib = _lib.load()
        Tq, Hq, D = q.shape
        Tk, Hk = k.shape[0], k.shape[1]
        n = 1 if q_offsets is None else q_offsets.numel() - 1
        dout, dout_at = _rows(dout if dout.dtype == q.dtype else dout.to(q.dtype))
        dq = torch.empty_like(out)
        keys = ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        dk = torch.empty(Tk, Hk, D, dtype=q.dtype, device=q.device) if keys else None
        dv = torch.empty(Tk, Hk, D, dtype=q.dtype, device=q.device) if keys else None
        need = lib.mg_attention_backward_workspace_bytes(Tq, Tk, Hq, Hk, D, n)
        ws = torch.empty(need, dtype=torch.uint8, device=q.device)
        _lib.launch(lib.mg_attention_backward, q.get_device(), _lib.TYPE_CODES[q.dtype], Tq, Tk,
                    Hq, Hk, D, *q_at, *k_at, *v_at,
                    None if q_offsets is None else q_offsets.data_ptr(),
                    None if k_offsets is None else k_offsets.data_ptr(), n, ctx.causal,
                    ctx.scale, out.data_ptr(), rest.data_ptr(), lse.data_ptr(), *dout_at, dq.data_ptr(),
                    dk.data_ptr() if keys else None, dv.data_ptr() if keys else None,
                    ws.data_ptr(), need)
        return dq, dk, dv, None, None, None, None


def _check_offsets(off, what, index):
    if off.dim() != 1 or off.shape[0] < 2:
        raise ValueError(f"{what} must be (sequences + 1,), got {tuple(off.shape)}")
    if not off.is_cuda or off.dtype != torch.int32 or not off.is_contiguous():
        _lib.dev_tensor(off, what, torch.int32)
    if off.get_device() != index:
        raise RuntimeError(f"{what} must be on GPU {index}, got device '{off.device}'")


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
              q_offsets: torch.Tensor | None = None, k_offsets: torch.Tensor | None = None, *,
              causal: bool = False, scale: float | None = None) -> torch.Tensor:
    """softmax(scale * q k^T) v within each of the sequences packed one after the
    other along the tokens.

    ``q`` (tokens, heads, dim), ``k`` and ``v`` (their own tokens, key heads, dim) are
    bfloat16 or float16, dim a multiple of 8 up to 128; the query heads are a
    multiple of the key heads, and query head h goes by key head
    ``h // (heads / key heads)``. Tokens and heads may have any stride: slices of
    one projection, or of a memory that holds keys and values side by side, are
    read where they lie.

    ``q_offsets`` and ``k_offsets`` (sequences + 1, int32, on the GPU) bound the
    sequences; k_offsets defaults to q_offsets, and both to one sequence of all
    tokens. A sequence may have more keys than queries (new tokens over a
    memory, down to one token), fewer, or none of either. ``causal``: a query sees
    the keys that stand at or before it, a sequence's last query standing at its
    last key. A query that sees no key, or belongs to no sequence, gets zeros;
    infinities and NaN in keys and values that it does not see leave no trace in
    its result (the backward pass asks for finite inputs within a sequence).
    ``scale`` (default dim ** -0.5) may not be negative.

    Scores, softmax and sums are float32; p is rounded to the inputs' type for
    its product with v. Differentiable in q, k and v, with the same bits from
    call to call; for that, what rounding took from the result is kept, a second
    tensor of its size.
    """
    dtype, dim, index = q.dtype, q.shape[-1] if q.dim() else 0, q.get_device()
    for t, what in ((q, "q"), (k, "k"), (v, "v")):
        if _lib.type_code(t, what) == 0:
            raise RuntimeError(f"{what} must be bfloat16 or float16, got {t.dtype}")
        if t.dim() != 3:
            raise ValueError(f"{what} must be (tokens, heads, dim), got {tuple(t.shape)}")
        if t.dtype != dtype or t.shape[2] != dim or t.get_device() != index:
            raise ValueError(f"{what} must match q's type, device and head dimension; got "
                             f"{t.dtype} {tuple(t.shape)} on {t.device}")
    if k.shape != v.shape:
        raise ValueError(f"k is {tuple(k.shape)} and v {tuple(v.shape)}; one shape is needed")
    if q_offsets is not None:
        _check_offsets(q_offsets, "q_offsets", index)
        if k_offsets is None:
            if k.shape[0] != q.shape[0]:
                raise ValueError(f"k_offsets is needed: {q.shape[0]} query tokens and "
                                 f"{k.shape[0]} key tokens")
            k_offsets = q_offsets
    if k_offsets is not None and k_offsets is not q_offsets:
        if q_offsets is None:
            raise ValueError("k_offsets needs q_offsets")
        _check_offsets(k_offsets, "k_offsets", index)
        if k_offsets.shape[0] != q_offsets.shape[0]:
            raise ValueError(f"q_offsets is {tuple(q_offsets.shape)} and k_offsets "
                             f"{tuple(k_offsets.shape)}; one number of sequences is needed")
    scale = max(dim, 1) ** -0.5 if scale is None else float(scale)
    if (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)) \
            or _lib.forward_mode():
        return _Attention.apply(q, k, v, q_offsets, k_offsets, bool(causal), scale)
    return _forward(q, k, v, q_offsets, k_offsets, bool(causal), scale, False)[0]
