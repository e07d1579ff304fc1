"""Layer norm on the MI355X: plain, affine, or modulated by a scale and shift per batch entry, with gradients.

A DiT block norms its hidden states three times and modulates two of them (``svoo/models/wan/custom_models.py:23-109``);
as tensor operations that is five to seven passes over the activations, here one read and one write.  Statistics are
fp32 whatever the tensors' types (bf16, fp16, fp32), outputs are rounded once.  Rows of 1 to 16384 columns, any strides
between rows and batch entries; fewer than 2^24 batch entries (2^22 above 5120 columns) where a parameter has a row for each.

:func:`layer_norm` is differentiable.  :func:`layer_norm_fwd` and :func:`layer_norm_bwd` are its two passes as plain
calls, for programs that keep the statistics themselves or capture a training step into a graph (autograd ties a leaf's
gradient to the stream of the first graph that used it; plain calls do not).  :func:`layer_norm_fp8` writes the result
as 8-bit rows for :func:`svoo_amd.fp8.fp8_matmul` instead.
"""

from __future__ import annotations

from typing import Optional, Sequence

import torch

from . import _lib
from .fp8 import FP8_TYPES, empty_fp8, empty_scales


def _param(p, cols: int, batch: int, device, name: str):
    """``p`` as what the C entry takes: ``(pointer, type, elements between batch entries)``, with the tensor read (kept
    alive by the caller) and whether it has a row per batch entry.  Expanded rows are such rows too, 0 elements apart."""
    kind = _lib.elem_type(p, name)
    shape = p.shape
    if p.device != device:
        raise ValueError(f"{name}: on {p.device}, x on {device}")
    dims = len(shape)
    if dims == 0 or shape[-1] != cols or (dims > 1 and (shape[0] not in (1, batch) or
                                                        any(n != 1 for n in shape[1:-1]))):
        raise ValueError(f"{name}: shape {tuple(shape)}; [{cols}] or [{batch}, 1, .., {cols}] expected")
    if p.stride(-1) != 1 and cols > 1:
        p = p.contiguous()
    each = dims > 1 and shape[0] == batch and batch > 1
    return p, (p.data_ptr(), kind, p.stride(0) if each else 0), each


_NO_PARAM = (None, 2, 0)


class _Call:
    """The checked arguments of a layer norm: x as ``[batch, rows, cols]`` by its strides, and its parameters.

    x is split by batch entries where a parameter's values differ between them, and where a gradient of a parameter with
    a row per entry is wanted (``grads``, of the two parameters)."""

    __slots__ = ("x", "x_args", "cols", "eps", "device", "shape", "batch", "rows", "modulated", "params", "args", "each",
                 "keep")

    def __init__(self, x, weight, bias, scale, shift, eps, grads=(False, False)):
        self.modulated = scale is not None or shift is not None
        if self.modulated and (weight is not None or bias is not None):
            raise ValueError("layer_norm: weight and bias or scale and shift, not both")
        if not eps >= 0:
            raise ValueError(f"layer_norm: eps={eps}")
        x_type = _lib.elem_type(x, "x")
        self.shape = shape = x.shape
        dims = len(shape)
        if dims == 0 or not 1 <= shape[-1] <= 16384:
            raise ValueError(f"layer_norm: x of shape {tuple(shape)} (1..16384 columns)")
        self.x, self.cols, self.eps, self.device = x, shape[-1], eps, x.device
        batch = shape[0] if dims > 1 else 1
        if self.modulated:
            self.params, names = (scale, shift), ("scale", "shift")
        else:
            self.params, names = (weight, bias), ("weight", "bias")
        self.keep, self.args, self.each = keep, args, each = [], [_NO_PARAM, _NO_PARAM], [False, False]
        split = False
        for i, p in enumerate(self.params):
            if p is not None:
                p, args[i], each[i] = _param(p, self.cols, batch, self.device, names[i])
                keep.append(p)
                split = split or args[i][2] != 0 or (each[i] and grads[i])
        self.batch = batch if split else 1
        self.rows = x.numel() // self.cols // self.batch if self.batch else 0
        self.x_args = (*self.rows_of(x, x_type),)

    def rows_of(self, t, kind):
        """A tensor of x's shape as the C entry takes it, ``(pointer, type, batch stride, row stride)``: in place where
        its strides make rows of contiguous columns."""
        if t.is_contiguous():
            return t.data_ptr(), kind, self.rows * self.cols, self.cols
        t = t.reshape(self.batch, self.rows, self.cols)
        if t.stride(2) != 1 and self.cols > 1:
            t = t.contiguous()
        self.keep.append(t)
        return t.data_ptr(), kind, t.stride(0), t.stride(1)

    def forward(self, y, y_type, q, s, fp8_type, mean, rstd):
        _lib.launch(self.device, "svoo_layer_norm_fwd", *self.x_args, *self.args[0], *self.args[1], self.modulated,
                    self.eps, self.batch, self.rows, self.cols, y, y_type, q, s, fp8_type, mean, rstd)


def _forward(c: _Call, out_dtype, stats: bool):
    """``(y, statistics [2, rows] or None)``."""
    y = torch.empty(c.shape, dtype=out_dtype or c.x.dtype, device=c.device)
    y_type = _lib.elem_type(y, "out_dtype")
    if not stats:
        c.forward(y.data_ptr(), y_type, None, None, 0, None, None)
        return y, None
    rows = c.batch * c.rows
    st = torch.empty((2, rows), dtype=torch.float32, device=c.device)
    at = st.data_ptr()
    c.forward(y.data_ptr(), y_type, None, None, 0, at, at + 4 * rows)
    return y, st


def layer_norm_fwd(x, weight=None, bias=None, *, scale=None, shift=None, eps=1e-6, out_dtype=None):
    """``(y, mean, rstd)`` of :func:`layer_norm`, with the fp32 statistics of every row (x's shape without its columns).
    No autograd."""
    _lib.refuse_grad("layer_norm_fwd", x, weight, bias, scale, shift)
    y, st = _forward(_Call(x, weight, bias, scale, shift, eps), out_dtype, True)
    return y, st[0].view(x.shape[:-1]), st[1].view(x.shape[:-1])


def layer_norm_bwd(dy, x, mean, rstd, weight=None, bias=None, *, scale=None, shift=None, eps=1e-6,
                   needs: Sequence[bool] = (True, True, True)):
    """Gradients ``(dx, dweight, dbias)`` (``(dx, dscale, dshift)``) for the incoming ``dy``, from x and the statistics
    that :func:`layer_norm_fwd` returned.

    Pass the parameters the forward pass had: a gradient has its parameter's shape and type and is None without one, or
    where ``needs`` says so.  Sums over rows are fp32 in a fixed order: the same call gives the same bits."""
    _lib.refuse_unseen("layer_norm_bwd", dy, x, mean, rstd, weight, bias, scale, shift)
    for t, name in ((mean, "mean"), (rstd, "rstd")):
        if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or t.shape != x.shape[:-1] or t.device != x.device:
            raise ValueError(f"{name}: fp32 of shape {tuple(x.shape[:-1])} on {x.device} expected")
    mean, rstd = mean.contiguous(), rstd.contiguous()
    return _backward(dy, _Call(x, weight, bias, scale, shift, eps, needs[1:]), mean.data_ptr(), rstd.data_ptr(), needs)


def _launch_backward(device, x_args, dy_args, w_args, modulated, mean, rstd, batch, rows, cols, dx, grads, types):
    ws, size = None, 0
    if grads[0] is not None or grads[1] is not None:
        size = _lib.lib().svoo_layer_norm_bwd_workspace_size(batch, rows, cols)
        if size:
            ws = _lib.workspace(size, device)
    _lib.launch(device, "svoo_layer_norm_bwd", *x_args, *dy_args, *w_args, modulated, mean, rstd, batch, rows, cols,
                _lib.ptr(dx), _lib.ptr(grads[0]), types[0], _lib.ptr(grads[1]), types[1], _lib.ptr(ws), size)


def _sum_of_rows(t, out):
    """``out`` with the sum of the rows of ``t [B, cols]`` (fp32): a bias's gradient for ``dy = t``, whatever x and the
    statistics are, so ``t`` stands for those too.  torch's ``sum`` clears its counters by a memset, which has no place in
    a captured graph."""
    rows, cols = t.shape
    at = t.data_ptr()
    args = (at, 2, rows * cols, cols)
    _launch_backward(t.device, args, args, _NO_PARAM, False, at, at, 1, rows, cols, None, (None, out),
                     (2, _lib.elem_type(out, "")))
    return out


def _backward(dy, c: _Call, mean: int, rstd: int, needs):
    x = c.x
    dy_type = _lib.elem_type(dy, "dy")
    if dy.shape != c.shape or dy.device != c.device:
        raise ValueError(f"dy: shape {tuple(dy.shape)} on {dy.device}, x {tuple(c.shape)} on {c.device}")
    dy_args = c.rows_of(dy, dy_type)
    dx = torch.empty(c.shape, dtype=x.dtype, device=c.device) if needs[0] else None
    want = [p is not None and need for p, need in zip(c.params, needs[1:])]
    if c.batch * c.rows == 0:
        return (dx, *(torch.zeros_like(p) if w else None for p, w in zip(c.params, want)))
    # a parameter shared by the batch entries of one that is not: its sums per entry, added here
    grads = [None, None]
    types = [2, 2]
    for i, p in enumerate(c.params):
        if want[i]:
            own = c.each[i] or c.batch == 1
            grads[i] = torch.empty(p.shape if own else (c.batch, c.cols), dtype=p.dtype if own else torch.float32,
                                   device=c.device)
            types[i] = _lib.elem_type(grads[i], "")
    _launch_backward(c.device, c.x_args, dy_args, c.args[0], c.modulated, mean, rstd, c.batch, c.rows, c.cols, dx, grads,
                     types)
    for i, p in enumerate(c.params):
        if grads[i] is not None and grads[i].shape != p.shape:
            grads[i] = _sum_of_rows(grads[i], torch.empty(p.shape, dtype=p.dtype, device=c.device))
    return dx, grads[0], grads[1]


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p0, p1, modulated, eps, out_dtype):
        params = (None, None, p0, p1) if modulated else (p0, p1, None, None)
        y, st = _forward(_Call(x, *params, eps), out_dtype, True)
        ctx.save_for_backward(x, p0, p1, st)
        ctx.modulated, ctx.eps = modulated, eps
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, p0, p1, st = ctx.saved_tensors
        params = (None, None, p0, p1) if ctx.modulated else (p0, p1, None, None)
        at = st.data_ptr()
        needs = ctx.needs_input_grad[:3]
        grads = _backward(dy, _Call(x, *params, ctx.eps, needs[1:]), at, at + 4 * st.shape[1], needs)
        return (*grads, None, None, None)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, *,
               scale: Optional[torch.Tensor] = None, shift: Optional[torch.Tensor] = None, eps: float = 1e-6,
               out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``n * weight + bias``, or ``n * (1 + scale) + shift``, of ``n = (x - mean) / sqrt(var + eps)`` over the last
    dimension.

    Parameters are ``[C]``, or ``[B, C]`` / ``[B, 1, .., C]`` with one row for each entry of x's first dimension
    (modulation vectors; strided ones are read in place).  Types may differ from x's.  The result has ``out_dtype``
    (x's by default).  Differentiable in x and the parameters, once."""
    _lib.refuse_unseen("layer_norm", x, weight, bias, scale, shift)
    if _lib.wants_grad(x, weight, bias, scale, shift):
        modulated = scale is not None or shift is not None
        if modulated and (weight is not None or bias is not None):
            raise ValueError("layer_norm: weight and bias or scale and shift, not both")
        return _LayerNorm.apply(x, scale if modulated else weight, shift if modulated else bias, modulated, eps, out_dtype)
    return _forward(_Call(x, weight, bias, scale, shift, eps), out_dtype, False)[0]


def layer_norm_fp8(x, weight=None, bias=None, *, scale=None, shift=None, eps=1e-6, dtype=torch.float8_e4m3fn):
    """:func:`layer_norm` in x's type, quantised in the same pass: ``(q, s)`` bit for bit as
    ``fp8_quantize_rows(layer_norm(x, ...))`` gives them, without the 16-bit result in memory.  No backward pass."""
    _lib.refuse_grad("layer_norm_fp8", x, weight, bias, scale, shift)
    if dtype not in FP8_TYPES:
        raise TypeError(f"layer_norm_fp8: float8_e4m3fn or float8_e5m2, got {dtype}")
    c = _Call(x, weight, bias, scale, shift, eps)
    q, s = empty_fp8(x.shape[:-1], c.cols, dtype, x.device), empty_scales(x.shape[:-1], c.cols, x.device)
    c.forward(None, c.x_args[1], q.data_ptr(), s.data_ptr(), FP8_TYPES[dtype], None, None)
    return q, s


# ------------------------------------------------------------------------------------------------ gated residuals
class _Residual:
    """The checked arguments of a gated residual with or without a norm: tensors as ``[batch, rows, cols]``, the parameters
    ``(gate, weight or scale, bias or shift)``.  Rows are split by batch entries where a parameter's values differ between
    them or a gradient with a row per entry is wanted (``grads``, of the three parameters)."""

    __slots__ = ("x", "kind", "cols", "eps", "device", "shape", "batch", "rows", "modulated", "params", "args", "each", "keep")

    def __init__(self, name, x, gate, weight, bias, scale, shift, eps, grads=(False,) * 3):
        self.modulated = scale is not None or shift is not None
        if self.modulated and (weight is not None or bias is not None):
            raise ValueError(f"{name}: weight and bias or scale and shift, not both")
        if not eps >= 0:
            raise ValueError(f"{name}: eps={eps}")
        self.kind = _lib.elem_type(x, "x")
        self.shape = shape = x.shape
        if len(shape) == 0 or not 1 <= shape[-1] <= 16384:
            raise ValueError(f"{name}: x of shape {tuple(shape)} (1..16384 columns)")
        self.x, self.cols, self.eps, self.device = x, shape[-1], eps, x.device
        batch = shape[0] if len(shape) > 1 else 1
        self.params = (gate, scale, shift) if self.modulated else (gate, weight, bias)
        names = ("gate", "scale", "shift") if self.modulated else ("gate", "weight", "bias")
        self.keep, self.args, self.each = [], [_NO_PARAM] * 3, [False] * 3
        split = False
        for i, p in enumerate(self.params):
            if p is not None:
                p, self.args[i], self.each[i] = _param(p, self.cols, batch, self.device, names[i])
                self.keep.append(p)
                split = split or self.args[i][2] != 0 or (self.each[i] and grads[i])
        self.batch = batch if split else 1
        if self.batch >= 65536:
            raise ValueError(f"{name}: {self.batch} batch entries with parameters of their own (fewer than 65536)")
        self.rows = x.numel() // self.cols // self.batch if self.batch else 0

    def rows_of(self, t, name):
        """A tensor of x's shape and type as the C entries take it, ``(pointer, batch stride, row stride)``."""
        if _lib.elem_type(t, name) != self.kind or t.shape != self.shape or t.device != self.device:
            raise ValueError(f"{name}: {t.dtype} {tuple(t.shape)} on {t.device}, x {self.x.dtype} {tuple(self.shape)} on "
                             f"{self.device}")
        if t.is_contiguous():
            return t.data_ptr(), self.rows * self.cols, self.cols
        t = t.reshape(self.batch, self.rows, self.cols)
        if t.stride(2) != 1 and self.cols > 1:
            t = t.contiguous()
        self.keep.append(t)
        return t.data_ptr(), t.stride(0), t.stride(1)


def _residual_forward(c: _Residual, branch, normed: bool, stats: bool):
    """``(h, y or None, statistics [2, rows] or None)``."""
    at, *strides = c.rows_of(c.x, "x")
    b_args = c.rows_of(branch, "branch")
    h = torch.empty_like(c.x, memory_format=torch.contiguous_format)
    y = torch.empty_like(c.x, memory_format=torch.contiguous_format) if normed else None
    rows = c.batch * c.rows
    st = torch.empty((2, rows), dtype=torch.float32, device=c.device) if stats else None
    mean = st.data_ptr() if stats else None
    _lib.launch(c.device, "svoo_residual_norm_fwd", at, c.kind, *strides, *b_args, *c.args[0], *c.args[1], *c.args[2],
                c.modulated, c.eps, c.batch, c.rows, c.cols, h.data_ptr(), _lib.ptr(y), mean, mean + 4 * rows if stats else None)
    return h, y, st


def _residual_backward(c: _Residual, dh, dy, h, branch, mean, rstd, needs):
    """``(dx, dbranch, dgate, dweight, dbias)`` as ``needs`` says; dy, h and the statistics are None for a residual alone."""
    params = c.params
    want = [p is not None and bool(n) for p, n in zip(params, needs[2:])]
    new = [torch.empty_like(c.x, memory_format=torch.contiguous_format) if n else None for n in needs[:2]]
    if c.batch * c.rows == 0:
        return (*new, *(torch.zeros_like(p) if w else None for p, w in zip(params, want)))
    sums = [torch.empty_like(p, memory_format=torch.contiguous_format) if w else None for p, w in zip(params, want)]
    if not any(needs[:2]) and not any(want):
        return (*new, *sums)
    size, ws = 0, None
    if any(want):
        size = _lib.lib().svoo_residual_norm_bwd_workspace_size(c.batch, c.rows, c.cols)
        ws = _lib.workspace(size, c.device)
    none = (None, 0, 0)
    _lib.launch(c.device, "svoo_residual_norm_bwd", *(none if dh is None else c.rows_of(dh, "dh")),
                *(none if dy is None else c.rows_of(dy, "dy")), c.kind, _lib.ptr(h),
                *(c.rows_of(branch, "branch") if want[0] else none), *c.args[0], *c.args[1], c.modulated, mean, rstd, c.batch,
                c.rows, c.cols, *(_lib.ptr(t) for t in new),
                *(v for i, t in enumerate(sums) for v in (_lib.ptr(t), 2 if t is None else _lib.elem_type(t, ""), c.each[i])),
                _lib.ptr(ws), size)
    return (*new, *sums)


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, branch, gate, p0, p1, modulated, eps):
        norm = (None, None, p0, p1) if modulated else (p0, p1, None, None)
        h, y, st = _residual_forward(_Residual("residual_norm", x, gate, *norm, eps), branch, True, True)
        ctx.save_for_backward(h, branch if gate is not None and gate.requires_grad else None, gate, p0, p1, st)
        ctx.modulated, ctx.eps = modulated, eps
        return h, y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh, dy):
        h, branch, gate, p0, p1, st = ctx.saved_tensors
        needs = ctx.needs_input_grad[:5]
        norm = (None, None, p0, p1) if ctx.modulated else (p0, p1, None, None)
        c = _Residual("residual_norm", h, gate, *norm, ctx.eps, needs[2:])
        at = st.data_ptr()
        return (*_residual_backward(c, dh, dy, h, branch, at, at + 4 * st.shape[1], needs), None, None)


class _GatedResidual(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, branch, gate):
        c = _Residual("gated_residual", x, gate, None, None, None, None, 0.0)
        h = _residual_forward(c, branch, False, False)[0]
        ctx.save_for_backward(branch if gate is not None and gate.requires_grad else None, gate)
        return h

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh):
        branch, gate = ctx.saved_tensors
        need_x, need_b, need_g = ctx.needs_input_grad
        dx = dh if need_x else None
        if gate is None:
            return dx, dh if need_b else None, None
        c = _Residual("gated_residual", dh, gate, None, None, None, None, 0.0, (need_g, False, False))
        _, db, dg, _, _ = _residual_backward(c, dh, None, None, branch, None, None, (False, need_b, need_g, False, False))
        return dx, db, dg


def residual_norm(x: torch.Tensor, branch: torch.Tensor, gate: Optional[torch.Tensor] = None,
                  weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, *,
                  scale: Optional[torch.Tensor] = None, shift: Optional[torch.Tensor] = None, eps: float = 1e-6):
    """``(h, y)``: ``h = x + gate * branch``, rounded to x's type, and :func:`layer_norm` of h in the same pass.

    ``branch`` has x's shape and type; ``gate`` (1 without one) and the norm's parameters are as those of
    :func:`layer_norm`.  Differentiable in all of them, once."""
    _lib.refuse_unseen("residual_norm", x, branch, gate, weight, bias, scale, shift)
    if _lib.wants_grad(x, branch, gate, weight, bias, scale, shift):
        modulated = scale is not None or shift is not None
        if modulated and (weight is not None or bias is not None):
            raise ValueError("residual_norm: weight and bias or scale and shift, not both")
        return _ResidualNorm.apply(x, branch, gate, scale if modulated else weight, shift if modulated else bias, modulated,
                                   eps)
    c = _Residual("residual_norm", x, gate, weight, bias, scale, shift, eps)
    return _residual_forward(c, branch, True, False)[:2]


def gated_residual(x: torch.Tensor, branch: torch.Tensor, gate: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x + gate * branch``, rounded once to x's type, without a norm: a block's end.  Differentiable, once."""
    _lib.refuse_unseen("gated_residual", x, branch, gate)
    if _lib.wants_grad(x, branch, gate):
        return _GatedResidual.apply(x, branch, gate)
    return _residual_forward(_Residual("gated_residual", x, gate, None, None, None, None, 0.0), branch, False, False)[0]


def residual_norm_fwd(x, branch, gate=None, weight=None, bias=None, *, scale=None, shift=None, eps=1e-6):
    """``(h, y, mean, rstd)`` of :func:`residual_norm`, with the fp32 statistics of every row of h.  No autograd."""
    _lib.refuse_grad("residual_norm_fwd", x, branch, gate, weight, bias, scale, shift)
    c = _Residual("residual_norm_fwd", x, gate, weight, bias, scale, shift, eps)
    h, y, st = _residual_forward(c, branch, True, True)
    return h, y, st[0].view(x.shape[:-1]), st[1].view(x.shape[:-1])


def residual_norm_bwd(dh, dy, h, branch, mean, rstd, gate=None, weight=None, bias=None, *, scale=None, shift=None, eps=1e-6,
                      needs: Sequence[bool] = (True,) * 5):
    """Gradients ``(dx, dbranch, dgate, dweight, dbias)`` (dscale and dshift in the last two places) for the gradients that
    arrive at h (or None) and y, from what :func:`residual_norm_fwd` took and returned; None without a parameter or where
    ``needs`` says so.  Sums over rows are fp32 in a fixed order."""
    _lib.refuse_unseen("residual_norm_bwd", dh, dy, h, branch, mean, rstd, gate, weight, bias, scale, shift)
    for t, name in ((mean, "mean"), (rstd, "rstd")):
        if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or t.shape != h.shape[:-1] or t.device != h.device:
            raise ValueError(f"{name}: fp32 of shape {tuple(h.shape[:-1])} on {h.device} expected")
    mean, rstd = mean.contiguous(), rstd.contiguous()
    c = _Residual("residual_norm_bwd", h, gate, weight, bias, scale, shift, eps, needs[2:])
    return _residual_backward(c, dh, dy, h.contiguous(), branch, mean.data_ptr(), rstd.data_ptr(), needs)
