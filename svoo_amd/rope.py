"""Rotary positions on several axes on the MI355X, behind the RMS norm of queries and keys, with gradients.

A video token has a position in time, height and width, and each axis turns its own share of a head's channels
(``svoo/models/wan/attention.py:179-190``; :func:`svoo_amd.dit.rope_tables` is the same as tables).  As tensor operations the
norm and the rotation are about eight passes over the projections; here one read and one write.  Angles are made where they
are used, from a grid's sizes or from positions, in doubles, so that far positions keep their angle.
:func:`svoo_amd.heads.qkv_heads` is the inference form for bf16 and given tables, which also transposes.

Tensors are bf16, fp16 or fp32 on the GPU; sums and rotations are fp32, a result is rounded once.
"""

from __future__ import annotations

import ctypes
import math
from typing import Optional, Sequence

import torch

from . import _lib

_NORMS = {"none": 0, "row": 1, "head": 2}
_POSITIONS = {torch.int32: 1, torch.int64: 2, torch.float32: 3}


class _Call:
    """The checked arguments, as the C entries take them."""

    __slots__ = ("kind", "shape", "device", "norm", "weight", "w_args", "where", "keep")

    def __init__(self, x, axes, grid, start, positions, theta, norm, weight, interleaved, eps):
        self.kind = _lib.elem_type(x, "x")
        self.device = x.device
        if x.dim() != 4:
            raise ValueError(f"axis_rope: x of shape {tuple(x.shape)}; [B, S, H, D] expected")
        self.shape = b, s, h, d = x.shape
        if d % 2 or not 2 <= d <= 512 or h == 0:
            raise ValueError(f"axis_rope: {h} heads of {d} channels (even, up to 512)")
        if norm not in _NORMS:
            raise ValueError(f"axis_rope: norm {norm!r} ({', '.join(_NORMS)})")
        if not eps >= 0:
            raise ValueError(f"axis_rope: eps={eps}")
        self.norm = _NORMS[norm]
        if norm == "row" and h > 32 * (64 // -(-d // 8)):
            raise ValueError(f"axis_rope: a norm over rows of {h} heads of {d} (at most {32 * (64 // -(-d // 8))})")
        axes = tuple(int(n) for n in axes)
        n = len(axes)
        if not 1 <= n <= 4 or any(a < 0 or a % 2 for a in axes) or sum(axes) > d:
            raise ValueError(f"axis_rope: axes {axes} of {d} channels (one to four, even)")
        thetas = tuple(float(t) for t in theta) if isinstance(theta, Sequence) else (float(theta),) * n
        if len(thetas) != n or not all(0 < t < 1e300 for t in thetas):
            raise ValueError(f"axis_rope: theta={theta} for {n} axes")
        if weight is None:
            self.weight, self.w_args = None, (None, 2)
        else:
            w_kind = _lib.elem_type(weight, "weight")
            want = {"row": h * d, "head": d}.get(norm)
            if want is None or weight.shape != (want,) or weight.device != x.device:
                raise ValueError(f"weight: shape {tuple(weight.shape)} on {weight.device} for norm={norm!r} over {h} heads of "
                                 f"{d} on {x.device}")
            self.weight = weight.contiguous()
            self.w_args = self.weight.data_ptr(), w_kind
        ints = ctypes.c_int * n
        if (grid is None) == (positions is None):
            raise ValueError("axis_rope: a grid or positions")
        if grid is not None:
            grid = tuple(int(g) for g in grid)
            start = (0,) * n if start is None else tuple(int(v) for v in start)
            if len(grid) != n or any(not 0 < g < 2 ** 31 for g in grid) or math.prod(grid) > max(s, 1):
                raise ValueError(f"axis_rope: grid {grid} for {n} axes and {s} rows")
            if len(start) != n or any(not -2 ** 31 <= v < 2 ** 31 for v in start):
                raise ValueError(f"axis_rope: start {start} for {n} axes")
            pos = None, 0, 0
            cells, at = ints(*grid), ints(*start)
        else:
            if start is not None:
                raise ValueError("axis_rope: start goes with a grid")
            if not isinstance(positions, torch.Tensor) or positions.dtype not in _POSITIONS:
                raise TypeError(f"positions: int32, int64 or float32, got {getattr(positions, 'dtype', type(positions).__name__)}")
            if positions.shape not in ((s, n), (b, s, n), (1, s, n)) or positions.device != x.device:
                raise ValueError(f"positions: shape {tuple(positions.shape)} on {positions.device}; [{s}, {n}] or [{b}, {s}, "
                                 f"{n}] on {x.device} expected")
            kind = _POSITIONS[positions.dtype]
            positions = positions.detach().contiguous()
            pos = positions.data_ptr(), kind, s * n if positions.dim() == 3 and positions.shape[0] == b else 0
            cells = at = None
        self.where = n, ints(*axes), (ctypes.c_double * n)(*thetas), cells, at, *pos, int(not interleaved)
        self.keep = [positions]

    def rows_of(self, t):
        """``(pointer, elements between batch entries, rows and heads)``, in place where a head's columns are contiguous."""
        if t.stride(3) != 1:
            t = t.contiguous()
        self.keep.append(t)
        return t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)


def _forward(c: _Call, x, eps):
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    at, *strides = c.rows_of(x)
    _lib.launch(c.device, "svoo_axis_rope_fwd", at, c.kind, *strides, *c.shape, c.norm, *c.w_args, eps, *c.where, y.data_ptr())
    return y


def _backward(c: _Call, dy, x, eps, needs):
    if _lib.elem_type(dy, "dy") != c.kind or dy.shape != c.shape or dy.device != c.device:
        raise ValueError(f"dy: {dy.dtype} {tuple(dy.shape)} on {dy.device}, x {x.dtype} {tuple(c.shape)} on {c.device}")
    dx = torch.empty_like(dy, memory_format=torch.contiguous_format) if needs[0] else None
    need_w = needs[1] and c.weight is not None
    if dy.numel() == 0:
        return dx, torch.zeros_like(c.weight) if need_w else None
    dw, ws, size = None, None, 0
    if need_w:
        dw = torch.empty_like(c.weight)
        size = _lib.lib().svoo_axis_rope_bwd_workspace_size(*c.shape, c.norm)
        ws = _lib.workspace(size, c.device)
    if dx is None and dw is None:
        return None, None
    x_at, *x_strides = c.rows_of(x)
    _lib.launch(c.device, "svoo_axis_rope_bwd", *c.rows_of(dy), x_at, c.kind, *x_strides, *c.shape, c.norm, *c.w_args, eps,
                *c.where, _lib.ptr(dx), _lib.ptr(dw), c.w_args[1], _lib.ptr(ws), size)
    return dx, dw


class _AxisRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, positions, args, eps):
        axes, grid, start, theta, norm, interleaved = args
        y = _forward(_Call(x, axes, grid, start, positions, theta, norm, weight, interleaved, eps), x, eps)
        ctx.save_for_backward(x if norm != "none" else None, weight, positions)
        ctx.args, ctx.eps = args, eps
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, positions = ctx.saved_tensors
        axes, grid, start, theta, norm, interleaved = ctx.args
        x = dy if x is None else x  # a rotation alone does not look at x
        c = _Call(x, axes, grid, start, positions, theta, norm, weight, interleaved, ctx.eps)
        return (*_backward(c, dy, x, ctx.eps, ctx.needs_input_grad[:2]), None, None, None)


def axis_rope(x: torch.Tensor, axes: Sequence[int], *, grid: Optional[Sequence[int]] = None,
              start: Optional[Sequence[int]] = None, positions: Optional[torch.Tensor] = None, theta=10000.0,
              norm: str = "none", weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
              interleaved: bool = True) -> torch.Tensor:
    """``x [B, S, H, D]`` with its RMS norm, then its rotary positions: same shape and type, contiguous.

    ``axes``: the channels of each axis (one to four, even, D in all at most; channels behind them stay).  Pair j of an axis
    of d channels turns by ``p theta^(-2j/d)`` at position p; ``theta`` is one for all or one for each.  Pairs are neighbours
    (``interleaved``) or channel j of the first half of a head and of the second.

    Positions are those of a ``grid`` (rows in order, the last axis fastest, counted from ``start``; rows behind the grid, a
    prompt's for instance, are not turned) or given as ``positions [S, axes]`` or ``[B, S, axes]`` (int32, int64, float32).

    ``norm``: ``"none"``, ``"row"`` (over all heads of a token, Wan's) or ``"head"`` (HunyuanVideo's), with ``weight``
    ``[H * D]`` or ``[D]`` if any.  Differentiable in x and weight, once."""
    _lib.refuse_unseen("axis_rope", x, weight, positions if isinstance(positions, torch.Tensor) else None)
    if isinstance(positions, torch.Tensor) and _lib.wants_grad(positions):
        raise RuntimeError("axis_rope has no gradient for positions: detach them")
    eps = float(eps)
    if _lib.wants_grad(x, weight):
        args = tuple(axes), grid if grid is None else tuple(grid), start if start is None else tuple(start), \
            tuple(theta) if isinstance(theta, Sequence) else theta, norm, bool(interleaved)
        return _AxisRope.apply(x, weight, positions, args, eps)
    return _forward(_Call(x, axes, grid, start, positions, theta, norm, weight, interleaved, eps), x, eps)


def axis_rope_bwd(dy, x, axes, *, grid=None, start=None, positions=None, theta=10000.0, norm="none", weight=None, eps=1e-6,
                  interleaved=True, needs: Sequence[bool] = (True, True)):
    """Gradients ``(dx, dweight)`` of :func:`axis_rope` for the incoming ``dy`` (None without a weight, or where ``needs`` says
    so).  Sums over rows are fp32 in a fixed order.  A plain call: no autograd."""
    _lib.refuse_unseen("axis_rope_bwd", dy, x, weight)
    eps = float(eps)
    return _backward(_Call(x, axes, grid, start, positions, theta, norm, weight, interleaved, eps), dy, x, eps, needs)
