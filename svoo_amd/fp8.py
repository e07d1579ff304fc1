"""8-bit matrices with a power-of-two scale per block of 128, their product, and a linear layer on them with gradients.

A block's scale is ``2^e`` with the smallest e that brings its largest magnitude within the type's range (448 for e4m3,
57344 for e5m2), kept as an e8m0 byte (``torch.float8_e8m0fnu``).  Such a scale is exact to multiply by, and gfx950's
matrix instructions apply it on the fly, so a product's sums stay inside the matrix unit over the whole contracted
dimension.  A floating-point format loses no precision to it, only up to one binade of its range.  The accumulator is
fp32; what the 8-bit instructions cut off before they add to it is stated at :func:`fp8_matmul`.

Values of a matrix ``[.., K]`` are stored as ``[.., 128 ceil(K / 128)]`` (zeros past K) with scales ``[.., ceil(K / 128)]``:

* :func:`fp8_quantize_rows`    a scale per 128 columns of each row (activations, gradients)
* :func:`fp8_quantize_blocks`  a scale per 128 x 128 block (weights), also of the transpose
* :func:`fp8_quantize_both`    rows, and the transposed matrix's rows: what a training step contracts both ways
* :func:`fp8_dequantize`       the values back
* :func:`fp8_matmul`           ``a b^T + bias``, with the tanh GELU if asked for
* :func:`fp8_linear`           ``x W^T + b`` from 16 or 32-bit tensors, differentiable
* :class:`Fp8Linear`           a ``torch.nn.Linear``'s stand-in for inference, its weight laid out once
* :class:`Fp8TrainLinear`      a ``torch.nn.Linear`` that computes by :func:`fp8_linear`

NaN stays NaN and infinities become NaN in e4m3 (e5m2 keeps them); they do not count towards a block's scale.
"""

from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from . import _lib

FP8_TYPES = {torch.float8_e4m3fn: 0, torch.float8_e5m2: 1}
SCALE_DTYPE = torch.float8_e8m0fnu
BLOCK = 128
_BOTH, _E4M3 = tuple(FP8_TYPES), (torch.float8_e4m3fn,)
_ACTS = {"none": 0, "gelu_tanh": 1}


def _blocks(n: int) -> int:
    return -(-n // BLOCK)


def empty_fp8(lead, cols: int, dtype, device) -> torch.Tensor:
    """Storage for the 8-bit values of ``[*lead, cols]``."""
    return torch.empty((*lead, _blocks(cols) * BLOCK), dtype=dtype, device=device)


def empty_scales(lead, cols: int, device) -> torch.Tensor:
    """Scales ``[*lead, ceil(cols / 128)]`` of rows, stored with neighbouring rows side by side."""
    kb = _blocks(cols)
    if len(lead) == 1:
        return torch.empty_strided((lead[0], kb), (1, max(lead[0], 1)), dtype=SCALE_DTYPE, device=device)
    return torch.empty(kb, math.prod(lead), dtype=SCALE_DTYPE, device=device).t().view(*lead, kb)


def _square_scales(rows: int, cols: int, device) -> torch.Tensor:
    return torch.empty(_blocks(rows), _blocks(cols), dtype=SCALE_DTYPE, device=device)


def _fp8_type(dtype, name: str) -> int:
    if dtype not in FP8_TYPES:
        raise TypeError(f"{name}: float8_e4m3fn or float8_e5m2, got {dtype}")
    return FP8_TYPES[dtype]


def _matrix(x, name: str):
    """``x [.., K]`` as ``(rows [M, K] with contiguous columns, its type)``, in place where the strides allow."""
    kind = _lib.elem_type(x, name)
    dims = x.dim()
    if dims == 0 or x.shape[-1] == 0:
        raise ValueError(f"{name}: shape {tuple(x.shape)}")
    if dims != 2:
        x = x.reshape(x.numel() // x.shape[-1], x.shape[-1])
    return (x if x.stride(1) == 1 or x.shape[1] == 1 else x.contiguous()), kind


def fp8_quantize_rows(x: torch.Tensor, dtype=torch.float8_e4m3fn) -> Tuple[torch.Tensor, torch.Tensor]:
    """``x [.., K]`` to ``(q [.., Kp], s [.., Kb])``: a scale per 128 columns of each row.  No backward pass."""
    _lib.refuse_grad("fp8_quantize_rows", x)
    fp8 = _fp8_type(dtype, "fp8_quantize_rows")
    rows, kind = _matrix(x, "x")
    m, k = rows.shape
    q, s = empty_fp8(x.shape[:-1], k, dtype, x.device), empty_scales(x.shape[:-1], k, x.device)
    _lib.launch(x.device, "svoo_fp8_quantize_rows", rows.data_ptr(), kind, rows.stride(0), m, k, fp8, q.data_ptr(),
                s.data_ptr())
    return q, s


def _tiles(rows, kind, dtype, square, plain, turned, sums=None):
    """``svoo_fp8_quantize_tiles`` of ``rows [M, K]``: ``(q, s)`` if ``plain``, ``(qt, st)`` if ``turned``, column sums
    into ``sums``."""
    m, k = rows.shape
    dev = rows.device
    q = s = qt = st = ws = None
    if plain:
        q = empty_fp8((m,), k, dtype, dev)
        s = _square_scales(m, k, dev) if square else empty_scales((m,), k, dev)
    if turned:
        qt = empty_fp8((k,), m, dtype, dev)
        st = _square_scales(k, m, dev) if square else empty_scales((k,), m, dev)
    if sums is not None:
        ws = _lib.workspace(_lib.lib().svoo_fp8_quantize_tiles_workspace_size(m, k), dev)
    _lib.launch(dev, "svoo_fp8_quantize_tiles", rows.data_ptr(), kind, rows.stride(0), m, k, FP8_TYPES[dtype],
                int(square), _lib.ptr(q), _lib.ptr(s), _lib.ptr(qt), _lib.ptr(st), _lib.ptr(sums),
                2 if sums is None else _lib.elem_type(sums, "sums"), _lib.ptr(ws), ws.numel() if ws is not None else 0)
    return q, s, qt, st


def fp8_quantize_blocks(w: torch.Tensor, dtype=torch.float8_e4m3fn, *, transposed: bool = False):
    """``w [N, K]`` to ``(q [N, Kp], s [Nb, Kb])``: a scale per 128 x 128 block; with ``transposed`` also
    ``(qt [K, Np], st [Kb, Nb])``, the same values and scales of the transpose.  No backward pass."""
    _lib.refuse_grad("fp8_quantize_blocks", w)
    _fp8_type(dtype, "fp8_quantize_blocks")
    if w.dim() != 2:
        raise ValueError(f"fp8_quantize_blocks: a matrix, got shape {tuple(w.shape)}")
    rows, kind = _matrix(w, "w")
    out = _tiles(rows, kind, dtype, True, True, transposed)
    return out if transposed else out[:2]


def fp8_quantize_both(x: torch.Tensor, dtype=torch.float8_e4m3fn):
    """``x [M, K]`` to ``(q [M, Kp], s [M, Kb], qt [K, Mp], st [K, Mb])``: its rows and its transpose's rows, each with
    a scale per 128 of its own columns, from one read.  No backward pass."""
    _lib.refuse_grad("fp8_quantize_both", x)
    _fp8_type(dtype, "fp8_quantize_both")
    if x.dim() != 2:
        raise ValueError(f"fp8_quantize_both: a matrix, got shape {tuple(x.shape)}")
    rows, kind = _matrix(x, "x")
    return _tiles(rows, kind, dtype, False, True, True)


class _Operand:
    """Checked 8-bit values and scales, as the C entries take them."""

    __slots__ = ("lead", "kp", "rows", "fp8", "tall", "args", "keep")

    def __init__(self, q, s, name: str, dtypes, square: bool, side_by_side: bool = False):
        """``square``: one scale may cover 128 rows.  ``side_by_side``: row scales are wanted with neighbouring rows in
        neighbouring bytes, and laid out so if they are not."""
        if not isinstance(q, torch.Tensor) or not isinstance(s, torch.Tensor):
            raise TypeError(f"{name}: tensors of values and scales, got {type(q).__name__}, {type(s).__name__}")
        if q.dtype not in dtypes:
            raise TypeError(f"{name}: {' or '.join(str(d)[6:] for d in dtypes)}, got {q.dtype}")
        if s.dtype != SCALE_DTYPE:
            raise TypeError(f"{name}'s scales: float8_e8m0fnu, got {s.dtype}")
        if not q.is_cuda:
            _lib.require_gpu_tensor(q, name)
        if s.device != q.device:
            raise ValueError(f"{name}'s scales: on {s.device}, values on {q.device}")
        shape, s_shape = q.shape, s.shape
        dims = len(shape)
        self.lead, kp = shape[:-1], shape[-1] if dims else 0
        if kp == 0 or kp % BLOCK:
            raise ValueError(f"{name}: shape {tuple(shape)}; columns in whole blocks of {BLOCK} expected")
        kb = kp // BLOCK
        if s_shape == (*self.lead, kb):
            self.tall = 1
        elif square and dims == 2 and s_shape == (_blocks(shape[0]), kb):
            self.tall = BLOCK
        else:
            raise ValueError(f"{name}'s scales: shape {tuple(s_shape)} for values {tuple(shape)}")
        if dims != 2:
            n = math.prod(self.lead)
            q, s = q.reshape(n, kp), s.view(torch.uint8).reshape(n, kb)
        self.kp, self.rows, self.fp8 = kp, q.shape[0], FP8_TYPES[q.dtype]
        row, at = q.stride(0) if self.rows > 1 else kp, q.data_ptr()
        if q.stride(1) != 1 or at % 16 or row % 16 or row < kp:
            q = q.view(torch.uint8).clone(memory_format=torch.contiguous_format)
            row, at = kp, q.data_ptr()
        if side_by_side and self.tall == 1 and self.rows > 1 and s.stride(0) != 1:
            s = s.view(torch.uint8).t().contiguous().t()
        self.keep = q, s
        self.args = at, row, s.data_ptr(), s.stride(0) if s.shape[0] > 1 else 1, s.stride(1) if kb > 1 else s.shape[0]


def fp8_dequantize(q: torch.Tensor, s: torch.Tensor, cols: Optional[int] = None, out_dtype=torch.bfloat16) -> torch.Tensor:
    """The values ``[.., cols]`` (all stored columns by default) that 8-bit values and their scales stand for, rounded to
    ``out_dtype``.  ``s`` has a row for each row of q, or for each 128 of a matrix's rows."""
    _lib.refuse_unseen("fp8_dequantize", q)
    o = _Operand(q, s, "q", _BOTH, True)
    cols = o.kp if cols is None else int(cols)
    if not o.kp - BLOCK < cols <= o.kp:
        raise ValueError(f"fp8_dequantize: cols={cols} of {o.kp} stored")
    y = torch.empty(*o.lead, cols, dtype=out_dtype, device=q.device)
    kind = _lib.elem_type(y, "out_dtype")
    _lib.launch(q.device, "svoo_fp8_dequantize", *o.args, o.tall, o.rows, cols, o.fp8, y.data_ptr(), kind)
    return y


def fp8_matmul(a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor,
               bias: Optional[torch.Tensor] = None, activation: str = "none", out_dtype=torch.bfloat16) -> torch.Tensor:
    """``act(a b^T + bias)`` of ``a [.., Kp]`` (e4m3 or e5m2, a scale per row and block) and ``b [N, Kp]`` (e4m3, a scale
    per row or per 128 rows and block), rounded once to ``out_dtype``: ``[.., N]``.

    With a 16-bit ``out_dtype`` the matrix instructions add eight products at a time, each cut 13 bits below the largest,
    before they go to the fp32 accumulator: about 2^-15 of a random sum's size, a fiftieth of bf16's own rounding and a
    sixth of fp16's, so one bf16 result in fifty and one fp16 result in ten is the neighbour of what fp32 sums round to.
    With ``out_dtype=torch.float32`` sums are fp32 throughout, at half the rate, of the operands' values as bf16 has them
    (below 2^-126 in steps of 2^-133, infinite from 2^128 on).

    ``activation``: ``"none"`` or ``"gelu_tanh"``.  The same call gives the same bits; a row's bits may depend on how many
    others are in the call (sums in another order, the GELU by other instructions).  No backward pass."""
    _lib.refuse_grad("fp8_matmul", bias)
    if activation not in _ACTS:
        raise ValueError(f"fp8_matmul: activation {activation!r} ({', '.join(_ACTS)})")
    oa = _Operand(a, a_scale, "a", _BOTH, False, True)
    ob = _Operand(b, b_scale, "b", _E4M3, True, True)
    if b.dim() != 2 or oa.kp != ob.kp or b.device != a.device:
        raise ValueError(f"fp8_matmul: a {tuple(a.shape)} on {a.device}, b {tuple(b.shape)} on {b.device}")
    m, n = oa.rows, ob.rows
    bias_type = 2
    if bias is not None:
        bias_type = _lib.elem_type(bias, "bias")
        if tuple(bias.shape) != (n,) or bias.device != a.device:
            raise ValueError(f"bias: shape {tuple(bias.shape)} on {bias.device}; [{n}] on {a.device} expected")
        bias = bias.contiguous()
    c = torch.empty((*oa.lead, n), dtype=out_dtype, device=a.device)
    kind = _lib.elem_type(c, "out_dtype")
    need = _lib.lib().svoo_fp8_matmul_workspace_size(m, n, oa.kp, kind)
    ws = _lib.workspace(need, a.device) if need else None
    _lib.launch(a.device, "svoo_fp8_matmul", *oa.args, oa.fp8, *ob.args, ob.tall, _lib.ptr(bias), bias_type,
                _ACTS[activation], m, n, oa.kp, c.data_ptr(), kind, _lib.ptr(ws), need)
    return c


def _linear(x, weight, bias, need_x: bool, need_w: bool):
    """``(y, (wqt, wst, qt, st))``: the layer's output, and the transposed weight and rows that the gradients of x and of
    the weight will read (None where they will not)."""
    rows, kind = _matrix(x, "x")
    w, w_kind = _matrix(weight, "weight")
    wq, ws, wqt, wst = _tiles(w, w_kind, torch.float8_e4m3fn, True, True, need_x)
    if need_w:
        q, s, qt, st = _tiles(rows, kind, torch.float8_e4m3fn, False, True, True)
    else:
        (q, s), qt, st = fp8_quantize_rows(rows), None, None
    y = fp8_matmul(q, s, wq, ws, bias, out_dtype=x.dtype)
    return y.view(*x.shape[:-1], w.shape[0]), (wqt, wst, qt, st)


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, grad_dtype):
        y, kept = _linear(x, weight, bias, *ctx.needs_input_grad[:2])
        ctx.save_for_backward(*kept)
        ctx.meta = x.shape, x.dtype, weight.shape, weight.dtype, None if bias is None else bias.dtype, grad_dtype
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x_shape, x_dtype, w_shape, w_dtype, b_dtype, grad_dtype = ctx.meta
        wqt, wst, qt, st = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        need_b = need_b and b_dtype is not None
        rows, kind = _matrix(dy, "dy")
        dx = dw = db = None
        if rows.shape[0] == 0:
            dx = torch.empty(x_shape, dtype=x_dtype, device=dy.device) if need_x else None
            dw = torch.zeros(w_shape, dtype=w_dtype, device=dy.device) if need_w else None
            db = torch.zeros(w_shape[0], dtype=b_dtype, device=dy.device) if need_b else None
            return dx, dw, db, None
        if need_b:
            db = torch.empty(w_shape[0], dtype=b_dtype, device=dy.device)
        q, s, gt, gs = _tiles(rows, kind, grad_dtype, False, need_x, need_w, db)
        if need_x:
            dx = fp8_matmul(q, s, wqt, wst, out_dtype=x_dtype).view(x_shape)
        if need_w:
            dw = fp8_matmul(gt, gs, qt, st, out_dtype=w_dtype)
        return dx, dw, db, None


def fp8_linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
               grad_dtype=torch.float8_e4m3fn) -> torch.Tensor:
    """``x [.., K] @ weight [N, K]^T + bias`` with 8-bit operands: x in rows of 128, the weight in 128 x 128 blocks, both
    e4m3.  Differentiable, once: ``dx`` from the incoming gradient's rows (``grad_dtype``: e4m3, or e5m2 for gradients
    of a wide range) and the weight, ``dweight`` from the gradient's and x's columns in blocks of 128 rows, ``dbias`` in
    fp32 sums of the unquantised gradient.  Results have the type of x, of weight and of bias; the three products are summed
    as :func:`fp8_matmul` sums for that type.

    Kept for the backward pass: 8-bit copies of x and of the weight (not made where no gradient can be asked for)."""
    _lib.refuse_unseen("fp8_linear", x, weight, bias)
    _fp8_type(grad_dtype, "fp8_linear")
    _lib.elem_type(weight, "weight")
    if weight.dim() != 2 or 0 in weight.shape or x.dim() == 0 or x.shape[-1] != weight.shape[1] or \
            weight.device != x.device:
        raise ValueError(f"fp8_linear: x {tuple(x.shape)} on {x.device}, weight {tuple(weight.shape)} on {weight.device}")
    if _lib.wants_grad(x, weight, bias):
        return _Linear.apply(x, weight, bias, grad_dtype)
    return _linear(x, weight, bias, False, False)[0]


class Fp8Linear(torch.nn.Module):
    """A linear layer for inference on 8-bit operands: the weight laid out once, x quantised in rows at every call.

    Buffers hold bytes, so ``module.to(dtype)`` leaves them alone (it changes the bias, in whatever of bf16, fp16 and
    fp32).  The output has x's type."""

    def __init__(self, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: str = "none"):
        super().__init__()
        if activation not in _ACTS:
            raise ValueError(f"Fp8Linear: activation {activation!r} ({', '.join(_ACTS)})")
        q, s = fp8_quantize_blocks(weight.detach())
        self.out_features, self.in_features = weight.shape
        self.activation = activation
        self.register_buffer("weight_q", q.view(torch.uint8))
        self.register_buffer("weight_scale", s.view(torch.uint8))
        self.register_buffer("bias", None if bias is None else bias.detach().clone())

    @classmethod
    def from_linear(cls, linear: torch.nn.Linear, activation: str = "none") -> "Fp8Linear":
        return cls(linear.weight, linear.bias, activation)

    def forward_quantized(self, q: torch.Tensor, s: torch.Tensor, out_dtype=torch.bfloat16) -> torch.Tensor:
        """The layer on rows that are quantised already (:func:`svoo_amd.norm.layer_norm_fp8`)."""
        return fp8_matmul(q, s, self.weight_q.view(torch.float8_e4m3fn), self.weight_scale.view(SCALE_DTYPE),
                          bias=self.bias, activation=self.activation, out_dtype=out_dtype)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.dim() == 0 or x.shape[-1] != self.in_features:
            raise ValueError(f"Fp8Linear: x {tuple(x.shape)} for {self.in_features} inputs")
        return self.forward_quantized(*fp8_quantize_rows(x), out_dtype=x.dtype)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}, " \
               f"activation={self.activation}"


class Fp8TrainLinear(torch.nn.Linear):
    """A ``torch.nn.Linear`` that computes by :func:`fp8_linear`: parameters as the optimiser keeps them (bf16, fp16 or
    fp32), quantised at every call."""

    grad_dtype = torch.float8_e4m3fn

    @classmethod
    def from_linear(cls, linear: torch.nn.Linear, grad_dtype=torch.float8_e4m3fn) -> "Fp8TrainLinear":
        """A layer that shares ``linear``'s parameters."""
        _fp8_type(grad_dtype, "Fp8TrainLinear")
        new = cls(linear.in_features, linear.out_features, bias=linear.bias is not None, device="meta")
        new.weight, new.bias, new.grad_dtype = linear.weight, linear.bias, grad_dtype
        return new.train(linear.training)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return fp8_linear(x, self.weight, self.bias, self.grad_dtype)
