"""Rotary positions of queries and keys on the GPU (mg_rotary).

The reference has no counterpart: this is one of the operators of a network
that predicts or refines splats, next to ``layer_norm`` and ``attention``.
"""

from __future__ import annotations

import ctypes
import functools
import math

import torch

from . import _lib

LAYOUTS = ("half", "interleaved")
ORDERS = ("runs", "turns")


def rotary_frequencies(dims: int, base: float = 10000.0, *, axes: int = 1,
                       scaling: str | None = None, factor: float = 1.0,
                       original_length: int | None = None, fast: float = 32.0,
                       slow: float = 1.0, device="cuda") -> torch.Tensor:
    """Radians per position of each of the ``dims // 2`` pairs, float64.

    Pair i of an axis's p = dims / 2 / axes pairs turns by ``base ** (-i / p)``;
    with several axes (a patch's column and row) the pairs are dealt to them in
    equal runs. For contexts ``factor`` times as long as those trained on:

    * ``scaling="linear"`` divides every frequency by ``factor``;
    * ``scaling="base"`` raises the base so that the slowest pair slows by
      ``factor`` and the fastest keeps its frequency;
    * ``scaling="bands"`` keeps the pairs that make at least ``fast`` turns within
      ``original_length``, divides those that make at most ``slow`` by ``factor``,
      and blends linearly in the number of turns between.
    """
    if dims < 2 or dims % (2 * axes) != 0:
        raise ValueError(f"{dims} rotated elements do not make pairs for {axes} axes")
    if scaling not in (None, "linear", "base", "bands"):
        raise ValueError(f"unknown scaling {scaling!r}; expected 'linear', 'base' or 'bands'")
    if factor <= 0.0 or base <= 0.0:
        raise ValueError(f"base {base} and factor {factor} must be positive")
    per = dims // 2 // axes
    i = torch.arange(per, dtype=torch.float64)
    if scaling == "base" and per > 1:
        base = base * factor ** (per / (per - 1))
    freq = base ** (-i / per)
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "bands":
        if original_length is None or not fast > slow:
            raise ValueError("scaling 'bands' needs original_length and fast > slow")
        turns = original_length * freq / (2.0 * math.pi)
        keep = ((turns - slow) / (fast - slow)).clamp(0.0, 1.0)
        freq = freq * keep + freq / factor * (1.0 - keep)
    return freq.repeat(axes).to(device)


def _heads(x: torch.Tensor):
    return x if x.stride(2) == 1 or x.shape[2] == 1 else x.contiguous()


@functools.lru_cache(maxsize=256)
def _table(sections: tuple, order: str):
    """The axis of each pair, a byte each."""
    if order not in ORDERS:
        raise ValueError(f"unknown order {order!r}; expected one of {ORDERS}")
    if not 1 <= len(sections) <= 256 or any(n < 0 for n in sections) \
            or not 1 <= sum(sections) <= 256:
        raise ValueError(f"sections {sections} must be numbers of pairs, up to 256 in all")
    turn = [(n, a) for a, count in enumerate(sections) for n in range(count)]
    if order == "turns":
        turn.sort()
    return ctypes.create_string_buffer(bytes(a for _, a in turn), len(turn))


def axis_table(sections, order, positions, frequencies):
    """The axis of each pair as the C calls take it, or None for equal runs."""
    if sections is None:
        if order != "runs":
            raise ValueError(f"order {order!r} needs sections")
        return None
    sections = tuple(sections)
    table = _table(sections, order)
    axes = 1 if positions.dim() == 1 else positions.shape[1]
    if len(sections) != axes or len(table) != frequencies.numel():
        raise ValueError(f"sections {sections} must be one for each of the {axes} axes and add "
                         f"up to the {frequencies.numel()} frequencies")
    return table


def _turn(q, k, positions, frequencies, layout, table, inverse):
    lib = _lib.load()
    q = _heads(q)
    T, Hq, D = q.shape
    q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    k_out, k_args, k_to = None, (None, 0, 0, 0), None
    if k is not None:
        k = _heads(k)
        k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
        k_args, k_to = (k.data_ptr(), k.stride(0), k.stride(1), k.shape[1]), k_out.data_ptr()
    fn, axis_of = (lib.mg_rotary, ()) if table is None else (lib.mg_rotary_axes, (table,))
    _lib.launch(fn, q.get_device(), T, _lib.TYPE_CODES[q.dtype], q.data_ptr(),
                q.stride(0), q.stride(1), Hq, *k_args, D, positions.data_ptr(),
                positions.dtype == torch.int64,
                1 if positions.dim() == 1 else positions.shape[1], *axis_of,
                frequencies.data_ptr(), frequencies.numel(), layout == "interleaved", inverse,
                q_out.data_ptr(), k_to)
    return q_out, k_out


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, frequencies, layout, table):
        ctx.save_for_backward(positions, frequencies)
        ctx.layout, ctx.table, ctx.dtype = layout, table, q.dtype
        ctx.set_materialize_grads(False)
        return _turn(q, k, positions, frequencies, layout, table, False)

    @staticmethod
    @_lib.differentiable_once
    def backward(ctx, dq, dk):
        # Hooks on saved tensors may give them back in another layout.
        positions, frequencies = (t.contiguous() for t in ctx.saved_tensors)
        dtype = ctx.dtype
        if dq is None and dk is None:
            return None, None, None, None, None, None
        first, second = (dq, dk) if dq is not None else (dk, None)
        first = first.to(dtype)
        second = None if second is None else second.to(dtype)
        a, b = _turn(first, second, positions, frequencies, ctx.layout, ctx.table, True)
        return (a, b, None, None, None, None) if dq is not None else \
            (None, a, None, None, None, None)


def _check(q, k, positions, frequencies, layout):
    """The GPU of all of them, and contiguous positions."""
    code = _lib.type_code(q, "q")
    if q.dim() != 3:
        raise ValueError(f"q must be (tokens, heads, dim), got {tuple(q.shape)}")
    index = q.get_device()
    if k is not None and (k.dim() != 3 or _lib.type_code(k, "k") != code or
                          k.shape[0] != q.shape[0] or k.shape[2] != q.shape[2] or
                          k.get_device() != index):
        raise ValueError(f"k must match q's type, device, tokens and head dimension; got "
                         f"{k.dtype} {tuple(k.shape)} against {q.dtype} {tuple(q.shape)}")
    if layout not in LAYOUTS:
        raise ValueError(f"unknown layout {layout!r}; expected one of {LAYOUTS}")
    if positions.dtype not in (torch.int32, torch.int64):
        raise RuntimeError(f"positions must be int32 or int64, got {positions.dtype}")
    if positions.dim() not in (1, 2) or positions.shape[0] != q.shape[0]:
        raise ValueError(f"positions must be ({q.shape[0]},) or ({q.shape[0]}, axes), got "
                         f"{tuple(positions.shape)}")
    if not positions.is_cuda or positions.get_device() != index:
        raise RuntimeError(f"positions must be on {q.device}, got device '{positions.device}'")
    if frequencies.dtype != torch.float64 or not frequencies.is_contiguous():
        _lib.dev_tensor(frequencies, "frequencies", torch.float64)
    if not frequencies.is_cuda or frequencies.get_device() != index:
        raise RuntimeError(f"frequencies must be on {q.device}, got device "
                           f"'{frequencies.device}'")
    if frequencies.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("frequencies must not require a gradient: there is none for them")
    return index, positions if positions.is_contiguous() else positions.contiguous()


def rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor,
           frequencies: torch.Tensor, *, layout: str = "half",
           sections: tuple[int, ...] | None = None, order: str = "runs"):
    """Turn pairs of each head's first ``2 * frequencies.numel()`` elements by
    ``position * frequency`` radians; the rest of the head is copied.

    ``q`` (tokens, heads, dim) and ``k`` (tokens, its own heads, dim; or None) are
    float32, bfloat16 or float16, with any strides over tokens and heads, so
    slices of one projection go as they are. ``positions`` is (tokens,) or
    (tokens, axes), int32 or int64, of any size or sign; ``frequencies`` comes from
    ``rotary_frequencies`` (float64 on the GPU). ``layout`` pairs elements (i, P + i)
    ("half") or (2i, 2i + 1) ("interleaved").

    With several axes (frame, row and column) the pairs are dealt to them in equal
    runs, or as ``sections`` says: one number of pairs for each axis (0 is taken),
    in all those of ``frequencies`` and 256 at most. ``order="runs"`` gives each axis
    neighbouring pairs; ``"turns"`` deals pair after pair to the axes in turn, an axis
    with its pairs dealt being left out, so that every axis has fast and slow ones.

    Returns new contiguous tensors (q, k), or q alone where k is None; one launch
    for both, one for both gradients. Differentiable in q and k; frequencies that
    require a gradient are refused.
    """
    _, positions = _check(q, k, positions, frequencies, layout)
    table = axis_table(sections, order, positions, frequencies)
    if (torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad))) \
            or _lib.forward_mode():
        out = _Rotary.apply(q, k, positions, frequencies, layout, table)
    else:
        out = _turn(q, k, positions, frequencies, layout, table, False)
    return out if k is not None else out[0]
