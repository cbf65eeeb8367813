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
        lib = _lib.load()
        dev, dtype, code = q.device, q.dtype, _lib.TYPE_CODES[q.dtype]
        tokens, _, dim = q.shape
        need = ctx.needs_input_grad
        make = torch.zeros if tokens == 0 else torch.empty
        heads, weight_at, dy_at, dx, dw, kept = [], [], [], [], [], []
        for x, w, dy, need_x, need_w in ((q, q_weight, dq_out, need[0], need[2]),
                                         (k, k_weight, dk_out, need[1], need[3])):
            if dy is None or not (need_x or need_w):
                x = w = dy = None
            else:
                x, dy = _heads(x), _heads(dy if dy.dtype == dtype else dy.to(dtype))
                w = None if w is None else w.contiguous()
                kept.append((x, w, dy))            # copies live until the launch
            at, weight = _args(x, w)
            heads += at
            weight_at.append(weight)
            dy_at += (None, 0, 0) if dy is None else (dy.data_ptr(), dy.stride(0), dy.stride(1))
            dx.append(None if x is None or not need_x
                      else torch.empty(x.shape, dtype=dtype, device=dev))
            dw.append(None if w is None or not need_w else make(dim, dtype=w.dtype, device=dev))
        if tokens and kept:
            ws, size = None, 0
            if dw[0] is not None or dw[1] is not None:
                size = lib.mg_norm_rotary_backward_workspace_bytes(heads[3], heads[7], dim)
                ws = torch.empty(size, dtype=torch.uint8, device=dev)
            _lib.launch(lib.mg_norm_rotary_backward, q.get_device(), tokens, code, *heads, dim,
                        _weight_code(q_weight, k_weight, code), *weight_at, ctx.eps,
                        *_position_args(positions, frequencies, ctx.table, ctx.layout), *dy_at,
                        *(None if t is None else t.data_ptr() for t in (*dx, *dw)),
                        None if ws is None else ws.data_ptr(), size)
        return dx[0], dx[1], dw[0], dw[1], None, None, None, None, None


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
