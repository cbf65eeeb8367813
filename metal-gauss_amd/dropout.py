"""Dropout on the GPU, onto a residual stream or by itself (mg_dropout).

The reference has no counterpart: this is one of the operators of a network
that predicts or refines splats, next to ``layer_norm`` and ``attention``.
"""

from __future__ import annotations

import operator

import torch

from . import _lib


def _run(x, residual, dtype, drop, seed, site):
    out = torch.empty_like(x, dtype=dtype, memory_format=torch.contiguous_format)
    x = x.contiguous()
    if residual is not None:
        residual = residual.contiguous()
    at = isinstance(seed, torch.Tensor)
    _lib.launch(_lib.load().mg_dropout, x.get_device(), x.numel(), _lib.TYPE_CODES[x.dtype],
                x.data_ptr(), _lib.TYPE_CODES[dtype],
                None if residual is None else residual.data_ptr(), out.data_ptr(), drop,
                0 if at else seed, seed.data_ptr() if at else None, site)
    return out


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, drop, seed, site):
        at = isinstance(seed, torch.Tensor)
        ctx.save_for_backward(seed if at else None)
        ctx.seed, ctx.site, ctx.drop, ctx.x_dtype = None if at else seed, site, drop, x.dtype
        dtype = x.dtype if residual is None else residual.dtype
        return _run(x, residual, dtype, drop, seed, site)

    @staticmethod
    @_lib.differentiable_once
    def backward(ctx, dy):
        seed, = ctx.saved_tensors
        dx = None
        if ctx.needs_input_grad[0]:
            dx = _run(dy, None, ctx.x_dtype, ctx.drop, ctx.seed if seed is None else seed,
                      ctx.site)
        return dx, dy if ctx.needs_input_grad[1] else None, None, None, None


def dropout(x: torch.Tensor, p: float, seed: int | torch.Tensor, *,
            residual: torch.Tensor | None = None, site: int = 0) -> torch.Tensor:
    """``residual + x * kept / (1 - p)``, each element of ``x`` kept with probability
    ``1 - p`` (0 in place of one that is not, whatever it holds).

    ``x`` is float32, bfloat16 or float16, of any shape; ``residual`` (None: nothing is
    added) has x's shape, is float32 or of x's type, and gives the result its type.
    ``p`` is held in steps of 2^-16, and the gain is that step's.

    Which elements are kept follows from their number in x, ``seed`` and ``site`` alone:
    16 bits each of a Philox4x32-10 block, never stored; the backward pass forms them
    again. ``seed`` is an integer below 2^64, or an int64 tensor of one element on the
    GPU, which a captured step can count on between replays (not between a call
    and its backward pass). ``site`` tells apart the calls of one step that share a
    seed. Differentiable in x and residual.
    """
    code = _lib.type_code(x, "x")
    index = x.get_device()
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"p must be between 0 and 1, got {p}")
    if residual is not None:
        if residual.shape != x.shape:
            raise ValueError(f"residual is {tuple(residual.shape)} and x {tuple(x.shape)}; one "
                             "shape is needed")
        if _lib.type_code(residual, "residual") not in (0, code):
            raise RuntimeError(f"residual must be float32 or of x's {x.dtype}, got "
                               f"{residual.dtype}")
        if residual.get_device() != index:
            raise RuntimeError(f"residual must be on {x.device}, got device '{residual.device}'")
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1:
            raise ValueError(f"seed must be one int64, got {seed.dtype} {tuple(seed.shape)}")
        if not seed.is_cuda or seed.get_device() != index:
            raise RuntimeError(f"seed must be on {x.device}, got device '{seed.device}'")
    else:
        seed = operator.index(seed)
        if not 0 <= seed < 2 ** 64:
            raise ValueError(f"seed must be an integer from 0 to 2^64 - 1, got {seed}")
    site = operator.index(site)
    if not 0 <= site < 2 ** 64:
        raise ValueError(f"site must be an integer from 0 to 2^64 - 1, got {site}")
    # Of 65536 draws: all of them for p = 1 alone.
    drop = 65536 if p == 1.0 else min(round(p * 65536.0), 65535)
    if (torch.is_grad_enabled() and (x.requires_grad or
                                     (residual is not None and residual.requires_grad))) \
            or _lib.forward_mode():
        return _Dropout.apply(x, residual, drop, seed, site)
    return _run(x, residual, x.dtype if residual is None else residual.dtype, drop, seed, site)
