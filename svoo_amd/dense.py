"""Dense attention on the MI355X with a backward pass, over heads that may share keys and values.

The sparse attention of this package has no gradients, and the layers and timesteps that run dense need some in training:
self-attention over a clip, cross-attention to a padded prompt.  The forward pass keeps the log-sum-exp of every query; the
backward pass computes the probabilities from it again, in two kernels that each own the rows they write, so that the same
call gives the same bits.

Tensors are ``[B, H, S, D]`` in bf16 or fp16 on the GPU, with any strides (rows that are not contiguous or not at 16-byte
addresses, and head dims that are no multiple of 8, are copied first); D is at most 128.  Scores, statistics and sums are
fp32; probabilities and their gradients are rounded to the tensors' type before they are multiplied.  fp16's are multiplied by
powers of two: probabilities keep all their bits down to 2^-26 of the largest of a row (18 below the highest score) in the
forward pass and to 2^-28 in the backward pass, and lose them over the ten bits below.  fp32 tensors are refused: they would
lose two thirds of their digits.

:func:`dense_attention` is differentiable; :func:`dense_attention_fwd` and :func:`dense_attention_bwd` are its two passes as
plain calls, for programs that capture a training step into a graph.
"""

from __future__ import annotations

import math
from typing import Optional, Sequence

import torch

from . import _lib

_TYPES = {torch.bfloat16: 0, torch.float16: 1}


def _kind(t, name: str) -> int:
    if not isinstance(t, torch.Tensor) or t.dtype not in _TYPES:
        raise TypeError(f"{name}: dense attention takes bfloat16 or float16 tensors, got "
                        f"{getattr(t, 'dtype', type(t).__name__)}")
    _lib.require_gpu_tensor(t, name)
    return _TYPES[t.dtype]


def _lens(t, name: str, batch: int, device):
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.shape != (batch,) or t.device != device:
        raise ValueError(f"{name}: int32 of shape ({batch},) on {device} expected")
    return t.contiguous()


class _Call:
    """The checked arguments of an attention: sizes, and operands as the C entries take them."""

    __slots__ = ("kind", "dtype", "device", "batch", "heads", "kv_heads", "sq", "sk", "d", "dp", "scale", "q_lens", "k_lens",
                 "keep")

    def __init__(self, q, k, v, scale, q_lens, k_lens):
        self.kind = _kind(q, "q")
        self.dtype, self.device = q.dtype, q.device
        for t, name in ((k, "k"), (v, "v")):
            if _kind(t, name) != self.kind or t.device != self.device:
                raise ValueError(f"{name}: {t.dtype} on {t.device}, q {q.dtype} on {q.device}")
        if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape or q.shape[0] != k.shape[0] or q.shape[3] != k.shape[3]:
            raise ValueError(f"dense_attention: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}; [B, H, S, D], "
                             "[B, Hk, Sk, D] twice expected")
        self.batch, self.heads, self.sq, self.d = q.shape
        self.kv_heads, self.sk = k.shape[1], k.shape[2]
        if not 1 <= self.d <= 128:
            raise ValueError(f"dense_attention: head dim {self.d} (1..128)")
        if self.heads and (self.kv_heads == 0 or self.heads % self.kv_heads):
            raise ValueError(f"dense_attention: {self.heads} query heads over {self.kv_heads} key heads")
        self.scale = self.d ** -0.5 if scale is None else float(scale)
        if not 0 < self.scale < math.inf:
            raise ValueError(f"dense_attention: scale={scale} (above 0)")
        self.q_lens, self.k_lens = _lens(q_lens, "q_lens", self.batch, q.device), _lens(k_lens, "k_lens", self.batch, q.device)
        self.dp = -(-self.d // 8) * 8
        self.keep = []

    def rows(self, t):
        """``(pointer, elements between batch entries, heads and rows)`` of an operand, copied where it cannot be read in
        place."""
        if self.dp == self.d:
            at, (b, h, r, c) = t.data_ptr(), t.stride()
            if c == 1 and not (at | 2 * (b | h | r)) % 16 and r < 1 << 23:
                return at, b, h, r
        else:
            t = torch.nn.functional.pad(t, (0, self.dp - self.d))
        b, h, r, c = (s if n > 1 else 0 for s, n in zip(t.stride(), t.shape))  # strides of single entries do not count
        if (c != 1 and self.dp > 1) or (t.data_ptr() | 2 * (b | h | r)) % 16 or r >= 1 << 23:
            t = t.contiguous()
            if t.data_ptr() % 16:  # contiguous as it was, at another address
                t = t.clone()
            b, h, r, _ = t.stride()
        self.keep.append(t)
        return t.data_ptr(), b, h, r

    def empty(self, heads: int, rows: int):
        """A result ``[B, H, S, D]``, contiguous as ``[B, S, H, D]``: a block's ``transpose(1, 2).flatten(2)`` is free."""
        d = self.dp
        return torch.empty_strided((self.batch, heads, rows, d), (rows * heads * d, d, heads * d, 1), dtype=self.dtype,
                                   device=self.device)

    def cut(self, t):
        if t is None or self.dp == self.d:
            return t
        return t.transpose(1, 2)[..., :self.d].contiguous().transpose(1, 2)

    def sizes(self):
        return self.kind, self.batch, self.heads, self.kv_heads, self.sq, self.sk, self.dp


def _forward(c: _Call, q, k, v, train: bool):
    """``(o, rest or None, lse)``."""
    o = c.empty(c.heads, c.sq)
    rest = c.empty(c.heads, c.sq) if train else None
    lse = torch.empty(c.batch, c.heads, c.sq, dtype=torch.float32, device=c.device)
    if c.sk == 0:
        return c.cut(o.zero_()), c.cut(rest.zero_()) if train else None, lse.fill_(-math.inf)
    if o.numel():
        need = _lib.lib().svoo_dense_attention_fwd_workspace_size(c.batch, c.heads, c.sq, c.sk, c.dp)
        ws = _lib.workspace(need, c.device) if need else None
        _lib.launch(c.device, "svoo_dense_attention_fwd", *c.rows(q), *c.rows(k), *c.rows(v), *c.sizes(), c.scale,
                    _lib.ptr(c.q_lens), _lib.ptr(c.k_lens), o.data_ptr(), _lib.ptr(rest), lse.data_ptr(), _lib.ptr(ws), need)
    return c.cut(o), c.cut(rest), lse


def _backward(c: _Call, dy, q, k, v, o, rest, lse, needs):
    out = [c.empty(h, s) if need else None
           for h, s, need in ((c.heads, c.sq, needs[0]), (c.kv_heads, c.sk, needs[1]), (c.kv_heads, c.sk, needs[2]))]
    if c.batch == 0 or c.heads == 0 or c.sq == 0 or c.sk == 0:
        return [None if t is None else c.cut(t.zero_()) for t in out]
    if any(needs):
        want_kv = bool(needs[1] or needs[2])
        need = _lib.lib().svoo_dense_attention_bwd_workspace_size(*c.sizes(), bool(needs[0]), want_kv)
        ws = _lib.workspace(need, c.device)
        if rest is not None:  # read as it was written
            rest = rest.transpose(1, 2)
            if c.dp != c.d or not rest.is_contiguous() or rest.data_ptr() % 16:
                rest = torch.nn.functional.pad(rest, (0, c.dp - c.d)).clone(memory_format=torch.contiguous_format)
        _lib.launch(c.device, "svoo_dense_attention_bwd", *c.rows(dy), *c.rows(q), *c.rows(k), *c.rows(v), *c.rows(o),
                    _lib.ptr(rest), lse.data_ptr(), *c.sizes(), c.scale, _lib.ptr(c.q_lens), _lib.ptr(c.k_lens), *(_lib.ptr(t) for t in out),
                    ws.data_ptr(), ws.numel())
    return [c.cut(t) for t in out]


class _DenseAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, scale, q_lens, k_lens):
        c = _Call(q, k, v, scale, q_lens, k_lens)
        o, rest, lse = _forward(c, q, k, v, True)
        ctx.save_for_backward(q, k, v, o, rest, lse, c.q_lens, c.k_lens)
        ctx.scale = c.scale
        return o

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        q, k, v, o, rest, lse, q_lens, k_lens = ctx.saved_tensors
        c = _Call(q, k, v, ctx.scale, q_lens, k_lens)
        return (*_backward(c, dy, q, k, v, o, rest, lse, ctx.needs_input_grad[:3]), None, None, None)


def dense_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, scale: Optional[float] = None,
                    q_lens: Optional[torch.Tensor] = None, k_lens: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``softmax(scale q k^T) v`` of ``q [B, H, Sq, D]`` over ``k, v [B, Hk, Sk, D]``; H is a multiple of Hk, and query head h
    reads key head ``h // (H / Hk)``.  ``scale`` is ``D ** -0.5`` by default.

    ``q_lens`` and ``k_lens`` (int32 ``[B]``, on the GPU; read there, values outside 0..S count as the nearest) are the valid
    rows of each batch entry: what lies behind them is not read, whatever it holds, results there are 0, and so are the
    results of queries without keys.  Keys whose score is -inf (a channel that masks them) have the probability 0, wherever they
    lie; a query whose every score is -inf is NaN.  The result is ``[B, H, Sq, D]``, contiguous as ``[B, Sq, H, D]``.  Differentiable in
    q, k and v, once."""
    _lib.refuse_unseen("dense_attention", q, k, v)
    if _lib.wants_grad(q, k, v):
        return _DenseAttention.apply(q, k, v, scale, q_lens, k_lens)
    return _forward(_Call(q, k, v, scale, q_lens, k_lens), q, k, v, False)[0]


def dense_attention_fwd(q, k, v, *, scale=None, q_lens=None, k_lens=None):
    """``(o, rest, lse)`` of :func:`dense_attention`, with what rounding o left (its shape and type; the backward pass needs o's
    product with the incoming gradient to more digits) and the fp32 log-sum-exp of every query's scaled scores
    ``[B, H, Sq]`` (-inf without keys and behind ``q_lens``).  No autograd."""
    _lib.refuse_grad("dense_attention_fwd", q, k, v)
    return _forward(_Call(q, k, v, scale, q_lens, k_lens), q, k, v, True)


def dense_attention_bwd(dy, q, k, v, o, rest, lse, *, scale=None, q_lens=None, k_lens=None,
                        needs: Sequence[bool] = (True, True, True)):
    """Gradients ``(dq, dk, dv)`` for the incoming ``dy``, from what :func:`dense_attention_fwd` took and returned
    (``rest`` may be None, at a loss of digits); None where ``needs`` says so."""
    _lib.refuse_unseen("dense_attention_bwd", dy, q, k, v, o, rest, lse)
    c = _Call(q, k, v, scale, q_lens, k_lens)
    for t, name in ((dy, "dy"), (o, "o"), (rest, "rest")):
        if t is None and name == "rest":
            continue
        _kind(t, name)
        if t.shape != q.shape or t.dtype != q.dtype or t.device != q.device:
            raise ValueError(f"{name}: {t.dtype} {tuple(t.shape)} on {t.device}, q {q.dtype} {tuple(q.shape)} on {q.device}")
    if not isinstance(lse, torch.Tensor) or lse.dtype != torch.float32 or lse.shape != q.shape[:3] or lse.device != q.device:
        raise ValueError(f"lse: fp32 of shape {tuple(q.shape[:3])} on {q.device} expected")
    return tuple(_backward(c, dy, q, k, v, o, rest, lse.contiguous(), needs))
