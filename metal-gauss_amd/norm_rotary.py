"""Queries' and keys' heads normed and turned by their positions in one pass, on
the GPU (mg_norm_rotary_*).

The reference has no counterpart: this is one of the operators of a network
that predicts or refines splats, next to ``layer_norm``, ``rotary`` and
``attention``.
"""

from __future__ import annotations

import torch

from . import _lib
from .rotary import _check, _heads, axis_table


def _args(x, weight):
    """What a C call takes of one tensor's heads."""
    if x is None:
        return (None, 0, 0, 0), None
    tok, head, _ = x.stride()
    return ((x.data_ptr(), tok, head, x.shape[1]), None if weight is None else weight.data_ptr())


def _weight_code(q_weight, k_weight, code):
    w = k_weight if q_weight is None else q_weight
    return code if w is None else _lib.TYPE_CODES[w.dtype]


def _position_args(positions, frequencies, table, layout):
    return (positions.data_ptr(), positions.dtype == torch.int64,
            1 if positions.dim() == 1 else positions.shape[1], table, frequencies.data_ptr(),
            frequencies.numel(), layout == "interleaved")


def _forward(q, k, q_weight, k_weight, positions, frequencies, eps, layout, table):
    q, k = _heads(q), None if k is None else _heads(k)
    code = _lib.TYPE_CODES[q.dtype]
    tokens, _, dim = q.shape
    q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    k_out = None if k is None else torch.empty_like(k, memory_format=torch.contiguous_format)
    (q_at, qw), (k_at, kw) = _args(q, q_weight), _args(k, k_weight)
    _lib.launch(_lib.load().mg_norm_rotary_forward, q.get_device(), tokens, code, *q_at, *k_at,
                dim, _weight_code(q_weight, k_weight, code), qw, kw, eps,
                *_position_args(positions, frequencies, table, layout), q_out.data_ptr(),
                None if k is None else k_out.data_ptr())
    return q_out, k_out


class _NormRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, positions, frequencies, eps, layout, table):
        ctx.save_for_backward(q, k, q_weight, k_weight, positions, frequencies)
        ctx.eps, ctx.layout, ctx.table = eps, layout, table
        ctx.set_materialize_grads(False)
        return _forward(q, k, q_weight, k_weight, positions, frequencies, eps, layout, table)

    @staticmethod
    @_lib.differentiable_once
    def backward(ctx, dq_out, dk_out):
        # Hooks on saved tensors may give them back in another layout.
        q, k, q_weight, k_weight, positions, frequencies = ctx.saved_tensors
        positions, frequencies = positions.contiguous(), frequencies.contiguous()
        need_q, need_k, need_qw, need_kw = ctx.needs_input_grad[:4]
        tokens, _, dim = q.shape
        code = _lib.TYPE_CODES[q.dtype]
        first = _gradients_of(q, q_weight, dq_out, need_q, need_qw)
        second = _gradients_of(k, k_weight, dk_out, need_k, need_kw)
        (_, q_at, qw, dy_q, dq, dqw), (_, k_at, kw, dy_k, dk, dkw) = first, second
        if tokens and (first[0] or second[0]):
            lib, ws, size = _lib.load(), None, 0
            if dqw is not None or dkw is not None:
                size = lib.mg_norm_rotary_backward_workspace_bytes(q_at[3], k_at[3], dim)
                ws = torch.empty(size, dtype=torch.uint8, device=q.device)
            _lib.launch(lib.mg_norm_rotary_backward, q.get_device(), tokens, code, *q_at, *k_at,
                        dim, _weight_code(q_weight, k_weight, code), qw, kw, ctx.eps,
                        *_position_args(positions, frequencies, ctx.table, ctx.layout), *dy_q,
                        *dy_k, *(None if t is None else t.data_ptr() for t in (dq, dk, dqw, dkw)),
                        None if ws is None else ws.data_ptr(), size)
        return dq, dk, dqw, dkw, None, None, None, None, None


def _gradients_of(x, w, dy, need_x, need_w):
    """One tensor's part of the backward call: what has to live until the launch, what
    the call takes of its heads, weights and results' gradient, and its gradients."""
    if dy is None or not (need_x or need_w):
        return (), (None, 0, 0, 0), None, (None, 0, 0), None, None
    x, dy = _heads(x), _heads(dy if dy.dtype == x.dtype else dy.to(x.dtype))
    w = None if w is None else w.contiguous()
    at, weight = _args(x, w)
    tok, head, _ = dy.stride()
    dx = torch.empty_like(x, memory_format=torch.contiguous_format) if need_x else None
    dw = None
    if w is not None and need_w:
        dw = torch.empty_like(w) if x.shape[0] else torch.zeros_like(w)
    return (x, w, dy), at, weight, (dy.data_ptr(), tok, head), dx, dw


def _check_weight(w, what, dim, index, dtype):
    if w.dim() != 1 or w.shape[0] != dim:
        raise ValueError(f"{what} must have shape ({dim},), got {tuple(w.shape)}")
    if not w.is_cuda or w.get_device() != index:
        raise RuntimeError(f"{what} must be on GPU {index}, got device '{w.device}'")
    if w.dtype not in (torch.float32, dtype):
        raise RuntimeError(f"{what} must be float32 or {dtype}, got {w.dtype}")
    return w if w.is_contiguous() else w.contiguous()


def norm_rotary(q: torch.Tensor, k: torch.Tensor | None, q_weight: torch.Tensor | None,
                k_weight: torch.Tensor | None, positions: torch.Tensor,
                frequencies: torch.Tensor, *, eps: float = 1e-6, layout: str = "half",
                sections: tuple[int, ...] | None = None, order: str = "runs"):
    """Norm each head by its root mean square, ``x / sqrt(mean(x^2) + eps) * weight``,
    and turn it as ``rotary`` does, in one pass.

    ``q`` (tokens, heads, dim) and ``k`` (tokens, its own heads, dim; or None) are
    float32, bfloat16 or float16, dim 2 to 512, with any strides over tokens and
    heads. ``q_weight`` and ``k_weight`` (dim,) are shared by the heads, float32 or of
    q's type, both alike; either may be None (ones). ``positions``, ``frequencies``,
    ``layout``, ``sections`` and ``order`` are those of ``rotary``.

    Returns new contiguous tensors (q, k), or q alone where k is None. All
    arithmetic is float32, rounded once. Differentiable in q, k and the weights,
    with the same bits from call to call; nothing but the inputs is kept for it.
    """
    index, positions = _check(q, k, positions, frequencies, layout)
    table = axis_table(sections, order, positions, frequencies)
    dim, dtype = q.shape[2], q.dtype
    if k is None and k_weight is not None:
        raise ValueError("k_weight needs k")
    if q_weight is not None:
        q_weight = _check_weight(q_weight, "q_weight", dim, index, dtype)
    if k_weight is not None:
        k_weight = _check_weight(k_weight, "k_weight", dim, index, dtype)
        if q_weight is not None and q_weight.dtype != k_weight.dtype:
            raise ValueError(f"q_weight is {q_weight.dtype} and k_weight {k_weight.dtype}; one "
                             "type is needed")
    run = _forward
    if (torch.is_grad_enabled() and (
            q.requires_grad or (k is not None and k.requires_grad) or
            (q_weight is not None and q_weight.requires_grad) or
            (k_weight is not None and k_weight.requires_grad))) or _lib.forward_mode():
        run = _NormRotary.apply
    out = run(q, k, q_weight, k_weight, positions, frequencies, float(eps), layout, table)
    return out if k is not None else out[0]
