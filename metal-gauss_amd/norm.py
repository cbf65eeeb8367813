"""Layer norm on the GPU, forward and backward (mg_layer_norm_*).

The reference has no counterpart: this is one of the operators of a network
that predicts or refines splats, next to ``rotary`` and ``attention``.
"""

from __future__ import annotations

import torch

from . import _lib


def _rows(x: torch.Tensor):
    """(2-D view or copy of x, row stride): rows may lie apart, a row may not."""
    n = x.shape[-1]
    if x.dim() != 2:
        x = x.reshape(-1, n)
    if x.stride(1) != 1 and n != 1:
        x = x.contiguous()
    return x, x.stride(0)


def _check_weight(w, n, index, what):
    if w.dim() != 1 or w.shape[0] != n:
        raise ValueError(f"{what} must have shape ({n},), got {tuple(w.shape)}")
    if w.get_device() != index:
        raise RuntimeError(f"{what} must be on GPU {index}, got device '{w.device}'")
    return w if w.is_contiguous() else w.contiguous()


def _forward(x, weight, bias, eps, keep):
    """y and, with ``keep``, what the backward pass needs."""
    code = _lib.type_code(x, "x")
    lib = _lib.load()
    width = x.shape[-1] if x.dim() else 0
    if width == 0:
        raise ValueError(f"layer_norm needs rows of at least one element, got {tuple(x.shape)}")
    index = x.get_device()
    wcode, w_at, b_at = code, None, None
    if weight is not None:
        weight = _check_weight(weight, width, index, "weight")
        wcode, w_at = _lib.type_code(weight, "weight"), weight.data_ptr()
    if bias is not None:
        bias = _check_weight(bias, width, index, "bias")
        if weight is not None and bias.dtype != weight.dtype:
            raise ValueError(f"weight is {weight.dtype} and bias {bias.dtype}; one type is needed")
        wcode, b_at = _lib.type_code(bias, "bias"), bias.data_ptr()
    rows, stride = _rows(x)
    n = rows.shape[0]
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    stats = mean = rstd = None
    if keep:
        stats = torch.empty(2 * n, dtype=torch.float32, device=x.device)
        mean = stats.data_ptr()
        rstd = mean + 4 * n
    _lib.launch(lib.mg_layer_norm_forward, index, n, width, code, rows.data_ptr(), stride, wcode,
                w_at, b_at, eps, y.data_ptr(), mean, rstd)
    return y, rows, stats, weight


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, rows, stats, w = _forward(x, weight, bias, eps, True)
        ctx.save_for_backward(rows, w, stats)
        ctx.x_shape = x.shape
        ctx.has_bias = None if bias is None else bias.dtype
        return y

    @staticmethod
    @_lib.differentiable_once
    def backward(ctx, dy):
        # Hooks on saved tensors may give them back in another layout.
        rows, w, stats = ctx.saved_tensors
        rows, row_stride = _rows(rows)
        stats = stats.contiguous()
        if w is not None:
            w = w.contiguous()
        lib = _lib.load()
        n, width = rows.shape
        dtype, dev, index = rows.dtype, rows.device, rows.get_device()
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        if dy.dtype != dtype:
            dy = dy.to(dtype)
        dy, dy_stride = _rows(dy)
        code = _lib.TYPE_CODES[dtype]
        wtype = w.dtype if w is not None else ctx.has_bias
        dx = torch.empty(ctx.x_shape, dtype=dtype, device=dev) if need_x else None
        make = torch.zeros if n == 0 else torch.empty
        dw = make(width, dtype=wtype, device=dev) if need_w else None
        db = make(width, dtype=wtype, device=dev) if need_b else None
        if n == 0:
            return dx, dw, db, None
        ws, size = None, 0
        if need_w or need_b:
            size = lib.mg_layer_norm_backward_workspace_bytes(n, width)
            ws = torch.empty(size, dtype=torch.uint8, device=dev)
        mean = stats.data_ptr()
        _lib.launch(lib.mg_layer_norm_backward, index, n, width, code, rows.data_ptr(),
                    row_stride, dy.data_ptr(), dy_stride,
                    code if wtype is None else _lib.TYPE_CODES[wtype],
                    None if w is None else w.data_ptr(), mean, mean + 4 * n,
                    dx.data_ptr() if need_x else None, dw.data_ptr() if need_w else None,
                    db.data_ptr() if need_b else None, ws.data_ptr() if size else None, size)
        return dx, dw, db, None


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None,
               bias: torch.Tensor | None = None, eps: float = 1e-5) -> torch.Tensor:
    """Normalise the last dimension of ``x``:
    ``(x - mean) / sqrt(var + eps) * weight + bias``.

    ``x`` is float32, bfloat16 or float16, any shape; rows may be strided.
    ``weight`` and ``bias`` (either may be None) are float32 or of x's type, and
    their gradients come in that type. Means, variances and all sums are float32;
    the result has x's type. Differentiable in all three, with the same bits from
    call to call.
    """
    if (torch.is_grad_enabled() and (
            x.requires_grad or (weight is not None and weight.requires_grad) or
            (bias is not None and bias.requires_grad))) or _lib.forward_mode():
        return _LayerNorm.apply(x, weight, bias, float(eps))
    return _forward(x, weight, bias, float(eps), False)[0]
