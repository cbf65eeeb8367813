"""Attention over packed sequences on the GPU, forward and backward
(mg_attention_*), and over memories that several sequences share
(mg_shared_attention).

The reference has no counterpart: this is one of the operators of a network
that predicts or refines splats, next to ``layer_norm`` and ``rotary``.
"""

from __future__ import annotations

import operator

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


def _calls(lib, which, causal, window):
    """The C entry and its workspace query, with what each takes of the mask."""
    if window is None:
        return (getattr(lib, f"mg_attention_{which}"), (causal,),
                getattr(lib, f"mg_attention_{which}_workspace_bytes"), ())
    return (getattr(lib, f"mg_attention_window_{which}"), window,
            getattr(lib, f"mg_attention_window_{which}_workspace_bytes"), window)


def _forward(q, k, v, q_offsets, k_offsets, causal, window, scale, keep):
    lib = _lib.load()
    call, mask, workspace, more = _calls(lib, "forward", causal, window)
    (q, q_at), (k, k_at), (v, v_at) = _rows(q), _rows(k), _rows(v)
    Tq, Hq, D = q.shape
    Tk, Hk, _ = k.shape
    n = 1 if q_offsets is None else q_offsets.numel() - 1
    # With a backward pass ahead, what rounding takes from the result is kept too.
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    rest = torch.empty_like(out) if keep else None
    lse = torch.empty(Hq, Tq, dtype=torch.float32, device=q.device) if keep else None
    need = workspace(Tq, Tk, Hq, Hk, D, n, *more)
    ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    _lib.launch(call, q.get_device(), _lib.TYPE_CODES[q.dtype], Tq, Tk, Hq,
                Hk, D, *q_at, *k_at, *v_at,
                None if q_offsets is None else q_offsets.data_ptr(),
                None if k_offsets is None else k_offsets.data_ptr(), n, *mask, scale,
                out.data_ptr(), rest.data_ptr() if keep else None,
                lse.data_ptr() if keep else None,
                ws.data_ptr() if need else None, need)
    return out, rest, lse, q, k, v


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, q_offsets, k_offsets, causal, window, scale):
        out, rest, lse, q, k, v = _forward(q, k, v, q_offsets, k_offsets, causal, window, scale,
                                           True)
        ctx.save_for_backward(q, k, v, q_offsets, k_offsets, out, rest, lse)
        ctx.causal, ctx.window, ctx.scale = causal, window, scale
        return out

    @staticmethod
    @_lib.differentiable_once
    def backward(ctx, dout):
        # Hooks on saved tensors may give them back in another layout.
        q, k, v, *others = ctx.saved_tensors
        q_offsets, k_offsets, out, rest, lse = (
            None if t is None else t.contiguous() for t in others)
        (q, q_at), (k, k_at), (v, v_at) = _rows(q), _rows(k), _rows(v)
        call, mask, workspace, more = _calls(_lib.load(), "backward", ctx.causal, ctx.window)
        Tq, Hq, D = q.shape
        Tk, Hk = k.shape[0], k.shape[1]
        n = 1 if q_offsets is None else q_offsets.numel() - 1
        dout, dout_at = _rows(dout if dout.dtype == q.dtype else dout.to(q.dtype))
        dq = torch.empty_like(out)
        keys = ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        dk = torch.empty(Tk, Hk, D, dtype=q.dtype, device=q.device) if keys else None
        dv = torch.empty(Tk, Hk, D, dtype=q.dtype, device=q.device) if keys else None
        need = workspace(Tq, Tk, Hq, Hk, D, n, *more)
        ws = torch.empty(need, dtype=torch.uint8, device=q.device)
        _lib.launch(call, q.get_device(), _lib.TYPE_CODES[q.dtype], Tq, Tk,
                    Hq, Hk, D, *q_at, *k_at, *v_at,
                    None if q_offsets is None else q_offsets.data_ptr(),
                    None if k_offsets is None else k_offsets.data_ptr(), n, *mask,
                    ctx.scale, out.data_ptr(), rest.data_ptr(), lse.data_ptr(), *dout_at, dq.data_ptr(),
                    dk.data_ptr() if keys else None, dv.data_ptr() if keys else None,
                    ws.data_ptr(), need)
        return dq, dk, dv, None, None, None, None, None


def _check_offsets(off, what, index):
    if off.dim() != 1 or off.shape[0] < 2:
        raise ValueError(f"{what} must be (sequences + 1,), got {tuple(off.shape)}")
    if not off.is_cuda or off.dtype != torch.int32 or not off.is_contiguous():
        _lib.dev_tensor(off, what, torch.int32)
    if off.get_device() != index:
        raise RuntimeError(f"{what} must be on GPU {index}, got device '{off.device}'")


def _check_heads(q, k, v, *more):
    """The head dimension and the GPU of all of them."""
    dtype, dim, index = q.dtype, q.shape[-1] if q.dim() else 0, q.get_device()
    others = (k, v, *more)
    fine = index >= 0 and q.dim() == 3 and (dtype is torch.bfloat16 or dtype is torch.float16)
    for t in others:
        fine = fine and t.dtype is dtype and t.get_device() == index and t.dim() == 3 \
            and t.shape[2] == dim
    if not fine:
        for t, what in zip((q, *others), ("q", "k", "v", "shared_k", "shared_v")):
            if _lib.type_code(t, what) == 0:
                raise RuntimeError(f"{what} must be bfloat16 or float16, got {t.dtype}")
            if t.dim() != 3:
                raise ValueError(f"{what} must be (tokens, heads, dim), got {tuple(t.shape)}")
            if t.dtype != dtype or t.shape[2] != dim or t.get_device() != index:
                raise ValueError(f"{what} must match q's type, device and head dimension; got "
                                 f"{t.dtype} {tuple(t.shape)} on {t.device}")
    if k.shape != v.shape:
        raise ValueError(f"k is {tuple(k.shape)} and v {tuple(v.shape)}; one shape is needed")
    return dim, index


def _check_bounds(q, k, q_offsets, k_offsets, index):
    """k_offsets, or what stands for them."""
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
    return k_offsets


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
              q_offsets: torch.Tensor | None = None, k_offsets: torch.Tensor | None = None, *,
              causal: bool = False, window: int | None = None, sinks: int = 0,
              scale: float | None = None) -> torch.Tensor:
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

    ``window`` (with ``causal``; 1 or more) leaves a query the last ``window`` of these
    keys, its own included, and the sequence's first ``sinks``; time goes by the keys
    that are left, and scratch memory is bounded by the tokens, not by the sequences.

    ``scale`` (default dim ** -0.5) may not be negative.

    Scores, softmax and sums are float32; p is rounded to the inputs' type for
    its product with v. Differentiable in q, k and v, with the same bits from
    call to call; for that, what rounding took from the result is kept, a second
    tensor of its size.
    """
    dim, index = _check_heads(q, k, v)
    k_offsets = _check_bounds(q, k, q_offsets, k_offsets, index)
    scale = max(dim, 1) ** -0.5 if scale is None else float(scale)
    if window is not None:
        if not causal:
            raise ValueError("window needs causal=True")
        window, sinks = operator.index(window), operator.index(sinks)
        if window < 1 or sinks < 0:
            raise ValueError(f"window must be at least 1 and sinks 0, got {window} and {sinks}")
        # More than any tensor has is all of them.
        window = (min(window, 2 ** 31 - 1), min(sinks, 2 ** 31 - 1))
    elif sinks:
        raise ValueError("sinks needs window: without one all first keys are seen")
    if (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)) \
            or _lib.forward_mode():
        return _Attention.apply(q, k, v, q_offsets, k_offsets, bool(causal), window, scale)
    return _forward(q, k, v, q_offsets, k_offsets, bool(causal), window, scale, False)[0]


class _Shared(torch.autograd.Function):
    """Calls while forward-mode derivatives are taken: autograd refuses a tangent."""

    @staticmethod
    def forward(ctx, *args):
        return _shared_forward(*args)

    @staticmethod
    def backward(ctx, dout):
        raise NotImplementedError("shared_attention has no gradient")


def _shared_forward(q, k, v, shared_k, shared_v, q_offsets, k_offsets, group_offsets,
                    shared_offsets, causal, scale):
    lib = _lib.load()
    rows = [_rows(t) for t in (q, k, v, shared_k, shared_v)]     # copies live until the launch
    Tq, Hq, D = q.shape
    Tk, Hk, _ = k.shape
    Ts = shared_k.shape[0]
    n = 1 if q_offsets is None else q_offsets.numel() - 1
    groups = 1 if group_offsets is None else group_offsets.numel() - 1
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    need = lib.mg_shared_attention_workspace_bytes(Tq, Tk, Ts, Hq, Hk, D, n, groups)
    ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    at = [None if t is None else t.data_ptr()
          for t in (q_offsets, k_offsets, group_offsets, shared_offsets)]
    _lib.launch(lib.mg_shared_attention, q.get_device(), _lib.TYPE_CODES[q.dtype], Tq, Tk, Ts, Hq,
                Hk, D, *(a for _, args in rows for a in args), at[0], at[1], n, at[2], at[3],
                groups, causal, scale, out.data_ptr(), ws.data_ptr() if need else None, need)
    return out


def shared_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, shared_k: torch.Tensor,
                     shared_v: torch.Tensor, q_offsets: torch.Tensor | None = None,
                     k_offsets: torch.Tensor | None = None,
                     group_offsets: torch.Tensor | None = None,
                     shared_offsets: torch.Tensor | None = None, *, causal: bool = False,
                     scale: float | None = None) -> torch.Tensor:
    """Attention of packed sequences to their own keys and, in the same softmax, to
    all of a memory that several sequences share (candidate cameras over one scene):
    what ``attention`` gives with the memory's keys and values before each sequence's
    own, while a shared key is read once for all of its group's queries and kept
    once.

    ``q``, ``k``, ``v``, ``q_offsets`` and ``k_offsets`` are those of ``attention``, and
    so is ``causal``, which bounds a sequence's own keys alone. ``shared_k`` and
    ``shared_v`` (their own tokens, k's heads, dim) may lie as k and v.
    ``group_offsets`` and ``shared_offsets`` (groups + 1, int32, on the GPU) bound each
    group's query tokens and its memory's tokens; both default to one group of all
    queries over all of the memory. Queries of no group have no shared keys, those of
    no sequence no own ones; a query without any gets zeros.

    bfloat16 or float16; scores, softmax and sums are float32 and p is rounded for
    its product with v, as in ``attention``. For serving: inputs that require a
    gradient are refused (train with ``attention`` over packed sequences).
    """
    dim, index = _check_heads(q, k, v, shared_k, shared_v)
    if shared_k.shape != shared_v.shape or shared_k.shape[1] != k.shape[1]:
        raise ValueError(f"shared_k is {tuple(shared_k.shape)} and shared_v "
                         f"{tuple(shared_v.shape)}; one shape, of k's {k.shape[1]} heads, is "
                         "needed")
    k_offsets = _check_bounds(q, k, q_offsets, k_offsets, index)
    if (group_offsets is None) != (shared_offsets is None):
        raise ValueError("group_offsets and shared_offsets go together")
    if group_offsets is not None:
        _check_offsets(group_offsets, "group_offsets", index)
        _check_offsets(shared_offsets, "shared_offsets", index)
        if group_offsets.shape[0] != shared_offsets.shape[0]:
            raise ValueError(f"group_offsets is {tuple(group_offsets.shape)} and shared_offsets "
                             f"{tuple(shared_offsets.shape)}; one number of groups is needed")
    if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v, shared_k, shared_v)):
        raise RuntimeError("shared_attention has no gradient, and an input requires one")
    scale = max(dim, 1) ** -0.5 if scale is None else float(scale)
    run = _Shared.apply if _lib.forward_mode() else _shared_forward
    return run(q, k, v, shared_k, shared_v, q_offsets, k_offsets, group_offsets, shared_offsets,
               bool(causal), scale)
