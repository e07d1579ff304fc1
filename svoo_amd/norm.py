"""Layer norm on the MI355X: plain, affine, or modulated by a scale and shift per batch entry, with gradients.

A DiT block norms its hidden states three times and modulates two of them (``svoo/models/wan/custom_models.py:23-109``);
as tensor operations that is five to seven passes over the activations, here one read and one write.  Statistics are
fp32 whatever the tensors' types (bf16, fp16, fp32), outputs are rounded once.  Rows of 1 to 16384 columns, any strides
between rows and batch entries.

:func:`layer_norm` is differentiable.  :func:`layer_norm_fwd` and :func:`layer_norm_bwd` are its two passes as plain
calls, for programs that keep the statistics themselves or capture a training step into a graph (autograd ties a leaf's
gradient to the stream of the first graph that used it; plain calls do not).  :func:`layer_norm_fp8` writes the result
as 8-bit rows for :func:`svoo_amd.fp8.fp8_matmul` instead.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from .fp8 import FP8_TYPES, empty_fp8, empty_scales


def _param(p, cols: int, batch: int, device, name: str):
    """``p`` as ``(rows [1 or batch, cols], one row per batch entry?)``."""
    if p is None:
        return None, False
    _lib.elem_type(p, name)
    if p.device != device:
        raise ValueError(f"{name}: on {p.device}, x on {device}")
    if p.dim() == 0 or p.shape[-1] != cols or any(n != 1 for n in p.shape[1:-1]) or \
            (p.dim() > 1 and p.shape[0] not in (1, batch)):
        raise ValueError(f"{name}: shape {tuple(p.shape)}; [{cols}] or [{batch}, 1, .., {cols}] expected")
    rows = p.reshape(-1, cols)
    if rows.stride(1) != 1:
        rows = rows.contiguous()
    return rows, p.dim() > 1 and p.shape[0] == batch and batch > 1


class _Call:
    """The checked arguments of a layer norm: x as ``[batch, rows, cols]`` and its parameters as rows."""

    def __init__(self, x, weight, bias, scale, shift, eps):
        if (weight is not None or bias is not None) and (scale is not None or shift is not None):
            raise ValueError("layer_norm: weight and bias or scale and shift, not both")
        if not eps >= 0:
            raise ValueError(f"layer_norm: eps={eps}")
        self.x_type = _lib.elem_type(x, "x")
        if x.dim() == 0 or not 1 <= x.shape[-1] <= 16384:
            raise ValueError(f"layer_norm: x of shape {tuple(x.shape)} (1..16384 columns)")
        self.modulated = scale is not None or shift is not None
        self.names = ("scale", "shift") if self.modulated else ("weight", "bias")
        self.params = (scale, shift) if self.modulated else (weight, bias)
        self.cols, self.eps, self.device, self.shape = x.shape[-1], float(eps), x.device, x.shape
        batch = x.shape[0] if x.dim() > 1 else 1
        (self.w, self.w_each), (self.b, self.b_each) = (
            _param(p, self.cols, batch, x.device, n) for p, n in zip(self.params, self.names))
        self.batch = batch if self.w_each or self.b_each else 1
        self.x = self.rows_of(x)
        self.rows = self.x.shape[1]

    def rows_of(self, t):
        """A tensor of x's shape as ``[batch, rows, cols]`` with contiguous columns, in place where its strides allow."""
        n = t.numel() // self.cols // self.batch if self.batch else 0
        t = t.reshape(self.batch, n, self.cols)
        return t if t.stride(2) == 1 else t.contiguous()

    def param_args(self, p, each):
        return (_lib.ptr(p), 2 if p is None else _lib.elem_type(p, ""), p.stride(0) if each else 0)

    def forward(self, y, y_type, q, s, fp8_type, mean, rstd):
        _lib.launch(self.device, "svoo_layer_norm_fwd", self.x.data_ptr(), self.x_type, self.x.stride(0), self.x.stride(1),
                    *self.param_args(self.w, self.w_each), *self.param_args(self.b, self.b_each), int(self.modulated),
                    self.eps, self.batch, self.rows, self.cols, _lib.ptr(y), y_type, _lib.ptr(q), _lib.ptr(s), fp8_type,
                    _lib.ptr(mean), _lib.ptr(rstd))


def _forward(c: _Call, x, out_dtype, stats: bool):
    out_dtype = x.dtype if out_dtype is None else out_dtype
    y = torch.empty(x.shape, dtype=out_dtype, device=x.device)
    y_type = _lib.elem_type(y, "out_dtype")
    mean, rstd = (torch.empty(2, *x.shape[:-1], dtype=torch.float32, device=x.device) if stats else (None, None))
    c.forward(y, y_type, None, None, 0, mean, rstd)
    return y, mean, rstd


def layer_norm_fwd(x, weight=None, bias=None, *, scale=None, shift=None, eps=1e-6, out_dtype=None):
    """``(y, mean, rstd)`` of :func:`layer_norm`, with the fp32 statistics of every row (x's shape without its columns).
    No autograd."""
    _lib.refuse_grad("layer_norm_fwd", x, weight, bias, scale, shift)
    return _forward(_Call(x, weight, bias, scale, shift, eps), x, out_dtype, True)


def layer_norm_bwd(dy, x, mean, rstd, weight=None, bias=None, *, scale=None, shift=None, eps=1e-6,
                   needs: Tuple[bool, bool, bool] = (True, True, True)):
    """Gradients ``(dx, dweight, dbias)`` (``(dx, dscale, dshift)``) for the incoming ``dy``, from x and the statistics
    that :func:`layer_norm_fwd` returned.

    Pass the parameters the forward pass had: a gradient has its parameter's shape and type and is None without one, or
    where ``needs`` says so.  Sums over rows are fp32 in a fixed order: the same call gives the same bits."""
    c = _Call(x, weight, bias, scale, shift, eps)
    dy_type = _lib.elem_type(dy, "dy")
    if dy.shape != x.shape or dy.device != x.device:
        raise ValueError(f"dy: shape {tuple(dy.shape)} on {dy.device}, x {tuple(x.shape)} on {x.device}")
    for t, name in ((mean, "mean"), (rstd, "rstd")):
        if t.dtype != torch.float32 or t.shape != x.shape[:-1] or t.device != x.device:
            raise ValueError(f"{name}: fp32 of shape {tuple(x.shape[:-1])} on {x.device} expected")
    mean, rstd = mean.contiguous(), rstd.contiguous()
    dy = c.rows_of(dy)
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if needs[0] else None
    want = [p is not None and need for p, need in zip(c.params, needs[1:])]
    if c.batch * c.rows == 0:
        return (dx, *(torch.zeros_like(p) if w else None for p, w in zip(c.params, want)))
    # a parameter shared by the batch entries of one that is not: its sums per entry, added here
    grads = [None] * 2
    for i, each in enumerate((c.w_each, c.b_each)):
        if want[i]:
            dtype = c.params[i].dtype if each or c.batch == 1 else torch.float32
            grads[i] = torch.empty(c.batch, c.cols, dtype=dtype, device=x.device)
    ws = None
    if any(want):
        ws = _lib.workspace(_lib.lib().svoo_layer_norm_bwd_workspace_size(c.batch, c.rows, c.cols), x.device)
    types = [2 if g is None else _lib.elem_type(g, "") for g in grads]
    _lib.launch(c.device, "svoo_layer_norm_bwd", c.x.data_ptr(), c.x_type, c.x.stride(0), c.x.stride(1), dy.data_ptr(),
                dy_type, dy.stride(0), dy.stride(1), *c.param_args(c.w, c.w_each), int(c.modulated), mean.data_ptr(),
                rstd.data_ptr(), c.batch, c.rows, c.cols, _lib.ptr(dx), _lib.ptr(grads[0]), types[0],
                _lib.ptr(grads[1]), types[1], _lib.ptr(ws), ws.numel() if ws is not None else 0)
    out = [None if g is None else (g if g.shape[0] == p.numel() // c.cols else g.sum(0)).to(p.dtype).view(p.shape)
           for g, p in zip(grads, c.params)]
    return (dx, *out)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p0, p1, modulated, eps, out_dtype):
        params = (None, None, p0, p1) if modulated else (p0, p1, None, None)
        y, mean, rstd = _forward(_Call(x, *params, eps), x, out_dtype, True)
        ctx.save_for_backward(x, p0, p1, mean, rstd)
        ctx.modulated, ctx.eps = modulated, eps
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, p0, p1, mean, rstd = ctx.saved_tensors
        kw = dict(scale=p0, shift=p1) if ctx.modulated else dict(weight=p0, bias=p1)
        grads = layer_norm_bwd(dy, x, mean, rstd, eps=ctx.eps, needs=ctx.needs_input_grad[:3], **kw)
        return (*grads, None, None, None)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, *,
               scale: Optional[torch.Tensor] = None, shift: Optional[torch.Tensor] = None, eps: float = 1e-6,
               out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``n * weight + bias``, or ``n * (1 + scale) + shift``, of ``n = (x - mean) / sqrt(var + eps)`` over the last
    dimension.

    Parameters are ``[C]``, or ``[B, C]`` / ``[B, 1, .., C]`` with one row for each entry of x's first dimension
    (modulation vectors; strided ones are read in place).  Types may differ from x's.  The result has ``out_dtype``
    (x's by default).  Differentiable in x and the parameters, once."""
    tensors = [t for t in (x, weight, bias, scale, shift) if t is not None]
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        modulated = scale is not None or shift is not None
        if modulated and (weight is not None or bias is not None):
            raise ValueError("layer_norm: weight and bias or scale and shift, not both")
        return _LayerNorm.apply(x, scale if modulated else weight, shift if modulated else bias, modulated, eps, out_dtype)
    return _forward(_Call(x, weight, bias, scale, shift, eps), x, out_dtype, False)[0]


def layer_norm_fp8(x, weight=None, bias=None, *, scale=None, shift=None, eps=1e-6, dtype=torch.float8_e4m3fn):
    """:func:`layer_norm` in x's type, quantised in the same pass: ``(q, s)`` bit for bit as
    ``fp8_quantize_rows(layer_norm(x, ...))`` gives them, without the 16-bit result in memory.  No backward pass."""
    _lib.refuse_grad("layer_norm_fp8", x, weight, bias, scale, shift)
    if dtype not in FP8_TYPES:
        raise TypeError(f"layer_norm_fp8: float8_e4m3fn or float8_e5m2, got {dtype}")
    c = _Call(x, weight, bias, scale, shift, eps)
    q, s = empty_fp8(x.shape[:-1], c.cols, dtype, x.device), empty_scales(x.shape[:-1], c.cols, x.device)
    c.forward(None, c.x_type, q, s, FP8_TYPES[dtype], None, None)
    return q, s
