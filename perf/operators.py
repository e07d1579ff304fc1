"""The dense half of a DiT block as measurable cases: layer norm, 8-bit products and what trains them.

``own`` false computes every operator from elementary torch operations; true calls ``svoo_amd.norm`` and
``svoo_amd.fp8``.  ``kind`` names the operator:

* ``norm``         layer norm, affine (``weight``, ``bias``) or modulated (``1 + scale``, ``shift`` per batch entry)
* ``norm_grad``    the same with its backward pass: y, dx and the gradients of the two parameters
* ``round_trip``   quantising to 8 bits with a power-of-two scale per block and reading the values back
* ``linear``       ``x W^T + b`` on 8-bit operands: x quantised in the call (rows of 128), W laid out before
                   (128 x 128 blocks), optionally with the tanh GELU
* ``linear_grad``  a training step of such a layer: y, dx, dW and db from 16-bit x, W and dy
* ``ffn``          a DiT block's feed-forward path: modulated norm straight to 8 bits, product with GELU, product

A block's scale is the smallest power of two that brings its largest magnitude within the type's range (448 for
e4m3, 57344 for e5m2); values are rounded to nearest even.  Blocks run along the contracted dimension.
"""

import math

import torch

own = False

_DEV = "cuda:0"
_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_FP8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
_TOP = {"e4m3": 448.0, "e5m2": 57344.0}
_EPS = 1e-6


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # One token's row: the norm of a conditioning vector, where a launch is all there is.
        dict(name="norm_one_row", kind="norm", batch=1, rows=1, cols=1536, dtype="bf16", form="affine"),
        # norm1 / norm3 of a 1.3B block at 480p (21 x 30 x 52 tokens, dim 1536), modulated in fp32: the ordinary call.
        dict(name="norm_480p", kind="norm", batch=1, rows=32760, cols=1536, dtype="bf16", form="modulated"),
        # Fine-tuning on a batch of two short ragged sequences with a width that is no multiple of anything, in fp16.
        dict(name="norm_grad_odd", kind="norm_grad", batch=2, rows=513, cols=999, dtype="fp16", form="affine"),
        # A training step of the 14B model's modulated norm at 720p (21 x 45 x 80 tokens, dim 5120): the largest norm.
        dict(name="norm_grad_720p", kind="norm_grad", batch=1, rows=75600, cols=5120, dtype="bf16", form="modulated"),
        # The FFN's inner activations of the 1.3B model stored in 8 bits and read back.
        dict(name="round_trip_rows", kind="round_trip", rows=32760, cols=8960, dtype="bf16", block="rows", fp8="e4m3"),
        # A weight matrix of a checkpoint in fp32 with odd sides, in 128 x 128 blocks of the wide-range type.
        dict(name="round_trip_weight", kind="round_trip", rows=1111, cols=5001, dtype="fp32", block="square", fp8="e5m2"),
        # The time projection of a denoising step: one token, 1536 -> 6 x 1536.
        dict(name="linear_one_token", kind="linear", rows=1, k=1536, n=9216, dtype="bf16", bias=True, act="none"),
        # The text embedder's first layer: 512 text tokens, 4096 -> 1536, with its GELU.
        dict(name="linear_text", kind="linear", rows=512, k=4096, n=1536, dtype="bf16", bias=True, act="gelu_tanh"),
        # An attention projection of the 14B model at 720p: the largest product.
        dict(name="linear_720p", kind="linear", rows=75600, k=5120, n=5120, dtype="bf16", bias=True, act="none"),
        # Training a small adapter on a ragged batch in fp16, no side a multiple of a tile.
        dict(name="linear_grad_odd", kind="linear_grad", rows=1013, k=1000, n=333, dtype="fp16", bias=True, fp8="e5m2"),
        # Training the 1.3B model's FFN expansion at 480p.
        dict(name="linear_grad_480p", kind="linear_grad", rows=32760, k=1536, n=8960, dtype="bf16", bias=True,
             fp8="e4m3"),
        # The feed-forward half of a 1.3B block at 480p, as the DiT runs it.
        dict(name="ffn_480p", kind="ffn", batch=1, rows=32760, k=1536, n=8960, dtype="bf16"),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "norm_grad", "norm_grad", "round_trip", "linear", "linear", "linear",
                       "linear_grad", "linear_grad", "ffn"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind in ("norm", "norm_grad"):
        cols = _spread(rng, 24, 8192)
        if rng.random() < 0.5:
            cols = max(64, cols // 64 * 64)
        batch = rng.choice([1, 1, 2, 3])
        rows = _spread(rng, 1, max(2.0, min(75600.0, 2.0e8 / (cols * batch))))
        return dict(kind=kind, batch=batch, rows=rows, cols=cols, dtype=dtype, form=rng.choice(["affine", "modulated"]))
    if kind == "round_trip":
        cols = _spread(rng, 40, 9000)
        rows = _spread(rng, 1, min(75600.0, 2.0e8 / cols))
        return dict(kind=kind, rows=rows, cols=cols, dtype=dtype, block=rng.choice(["rows", "square"]),
                    fp8=rng.choice(["e4m3", "e5m2"]))
    k, n = (_spread(rng, 100, 9000) for _ in range(2))
    if rng.random() < 0.5:
        k, n = max(128, k // 128 * 128), max(128, n // 128 * 128)
    most = min(75600.0, (8.0e11 if kind == "linear" else 2.5e11) / (k * n))
    rows = _spread(rng, 1, max(2.0, most))
    if kind == "ffn":
        return dict(kind=kind, batch=1, rows=rows, k=k, n=n, dtype=rng.choice(["bf16", "fp16"]))
    c = dict(kind=kind, rows=rows, k=k, n=n, dtype=dtype, bias=rng.random() < 0.8)
    if kind == "linear":
        c["act"] = rng.choice(["none", "none", "gelu_tanh"])
    else:
        c["fp8"] = rng.choice(["e4m3", "e5m2"])
    return c


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=_DEV).manual_seed(seed)


def _activations(g, rows, cols, dtype, level=1.0):
    """Rows of a residual stream: unit noise on channels of unequal size, a few of them far larger."""
    x = torch.randn(rows, cols, generator=g, device=_DEV)
    chan = torch.exp(0.5 * torch.randn(cols, generator=g, device=_DEV))
    far = torch.rand(cols, generator=g, device=_DEV) < 0.01
    x *= level * torch.where(far, 8.0 * chan, chan)
    return x.to(dtype)


def _weights(g, n, k, dtype):
    return (torch.randn(n, k, generator=g, device=_DEV) / math.sqrt(k)).to(dtype)


def _small(g, n, dtype):
    return (0.1 * torch.randn(n, generator=g, device=_DEV)).to(dtype)


def prepare(case, seed):
    g = _gen(seed)
    dtype = _DTYPES[case["dtype"]]
    kind = case["kind"]
    st = {"case": case}
    if kind in ("norm", "norm_grad"):
        b, s, c = case["batch"], case["rows"], case["cols"]
        st["x"] = (_activations(g, b * s, c, torch.float32) + 0.3).to(dtype).view(b, s, c)
        if case["form"] == "affine":
            st["p"] = (1 + _small(g, c, torch.float32)).to(dtype), _small(g, c, dtype)
        else:
            mod = 0.3 * torch.randn(b, 6, c, generator=g, device=_DEV)  # a block's six modulation vectors, in fp32
            st["p"] = mod[:, 1:2], mod[:, 0:1]
        if kind == "norm_grad":
            st["dy"] = _activations(g, b * s, c, dtype, 1e-2).view(b, s, c)
            if own:
                st["leaves"] = [t.detach().requires_grad_() for t in (st["x"],) + tuple(st["p"])]
    elif kind == "round_trip":
        make = _activations if case["block"] == "rows" else _weights
        st["x"] = make(g, case["rows"], case["cols"], dtype)
    elif kind == "linear":
        st["x"] = _activations(g, case["rows"], case["k"], dtype)
        st["w"] = _layout(_weights(g, case["n"], case["k"], dtype))
        st["b"] = _small(g, case["n"], dtype) if case["bias"] else None
    elif kind == "linear_grad":
        st["x"] = _activations(g, case["rows"], case["k"], dtype)
        st["w"] = _weights(g, case["n"], case["k"], dtype)
        st["b"] = _small(g, case["n"], dtype) if case["bias"] else None
        st["dy"] = _activations(g, case["rows"], case["n"], dtype, 1e-2)
        if own:
            st["leaves"] = [None if t is None else t.detach().requires_grad_() for t in (st["x"], st["w"], st["b"])]
    else:
        b, s, k, n = case["batch"], case["rows"], case["k"], case["n"]
        st["x"] = _activations(g, b * s, k, dtype).view(b, s, k)
        mod = 0.3 * torch.randn(b, 6, k, generator=g, device=_DEV)
        st["p"] = mod[:, 4:5], mod[:, 3:4]
        st["w"] = _layout(_weights(g, n, k, dtype)), _layout(_weights(g, k, n, dtype))
        st["b"] = _small(g, n, dtype), _small(g, k, dtype)
    return st


def _layout(w):
    """A weight as a program keeps it: 8-bit values and a scale per 128 x 128 block."""
    if own:
        from svoo_amd import fp8

        return fp8.fp8_quantize_blocks(w)
    return _quantize(w, 128, "e4m3")


# ------------------------------------------------------------------------------------------------ plain forms
def _norm_plain(x, p, form):
    x = x.float()
    mean = x.mean(-1, keepdim=True)
    d = x - mean
    rstd = torch.rsqrt((d * d).mean(-1, keepdim=True) + _EPS)
    n = d * rstd
    w, b = (t.float() for t in p)
    w = w if form == "affine" else 1 + w
    return n * w + b, n, rstd, w


def _power(e):
    """2^e exactly, by way of a double's bits (a device's exp2 and pow need not be exact at whole numbers)."""
    return ((e.long() + 1023) << 52).view(torch.float64).float()


def _quantize(x, block_rows, fp8):
    """8-bit values and int32 exponents of the (block_rows x 128) blocks of a matrix."""
    x = x.float()
    m, k = x.shape
    mb, kb = -(-m // block_rows), -(-k // 128)
    padded = torch.zeros(mb * block_rows, kb * 128, device=x.device)
    padded[:m, :k] = x
    blocks = padded.view(mb, block_rows, kb, 128)
    frac, e = torch.frexp(blocks.abs().amax((1, 3), keepdim=True))
    e = e - (9 if fp8 == "e4m3" else 16) + (frac > 0.875).to(e.dtype)
    e = torch.where(frac == 0, torch.zeros_like(e), e.clamp(-127, 127))
    q = (blocks * _power(-e)).view(mb * block_rows, kb * 128)[:m, :k].to(_FP8[fp8])
    return q, e.view(mb, kb)


def _dequantize(q, e):
    m, k = q.shape
    s = _power(e).repeat_interleave(128, 1)[:, :k]
    if s.shape[0] != m:
        s = s.repeat_interleave(128, 0)[:m]
    return q.float() * s


def _rounded(x, block_rows, fp8="e4m3"):
    return _dequantize(*_quantize(x, block_rows, fp8))


def _gelu(x):
    return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x * x * x)))


def _linear_plain(x, w, b, act):
    y = _rounded(x, 1) @ _dequantize(*w).t()
    if b is not None:
        y = y + b.float()
    return _gelu(y) if act == "gelu_tanh" else y


def _run_plain(st):
    case, x = st["case"], st["x"]
    kind, dtype = case["kind"], x.dtype
    if kind == "norm":
        return _norm_plain(x, st["p"], case["form"])[0].to(dtype)
    if kind == "norm_grad":
        y, n, rstd, w = _norm_plain(x, st["p"], case["form"])
        dy = st["dy"].float()
        g = dy * w
        dx = rstd * (g - g.mean(-1, keepdim=True) - n * (g * n).mean(-1, keepdim=True))
        over = (0, 1) if case["form"] == "affine" else 1
        dw = (dy.double() * n).sum(over, keepdim=case["form"] != "affine")  # long sums
        db = dy.double().sum(over, keepdim=case["form"] != "affine")
        return y.to(dtype), dx.to(dtype), dw.to(st["p"][0].dtype), db.to(st["p"][1].dtype)
    if kind == "round_trip":
        return _rounded(x, 1 if case["block"] == "rows" else 128, case["fp8"]).to(dtype)
    if kind == "linear":
        return _linear_plain(x, st["w"], st["b"], case["act"]).to(dtype)
    if kind == "linear_grad":
        w, b, dy = st["w"], st["b"], st["dy"]
        wq = _rounded(w, 128)
        y = _rounded(x, 1) @ wq.t()
        y = y if b is None else y + b.float()
        dx = _rounded(dy, 1, case["fp8"]) @ wq
        dw = _rounded(dy.t(), 1, case["fp8"]) @ _rounded(x.t(), 1).t()
        out = [y.to(dtype), dx.to(dtype), dw.to(dtype)]
        return out if b is None else out + [dy.double().sum(0).to(dtype)]
    h = _norm_plain(x, st["p"], "modulated")[0].to(dtype)
    h = _linear_plain(h.flatten(0, 1), st["w"][0], st["b"][0], "gelu_tanh").to(dtype)
    return _linear_plain(h, st["w"][1], st["b"][1], "none").to(dtype).view(x.shape)


# ------------------------------------------------------------------------------------------------ the framework's
def _run_own(st):
    from svoo_amd import fp8, norm

    case, x = st["case"], st["x"]
    kind = case["kind"]
    names = ("weight", "bias") if case.get("form") == "affine" else ("scale", "shift")
    if kind == "norm":
        return norm.layer_norm(x, eps=_EPS, **dict(zip(names, st["p"])))
    if kind == "norm_grad":
        x, *p = st["leaves"]
        y = norm.layer_norm(x, eps=_EPS, **dict(zip(names, p)))
        return (y.detach(),) + torch.autograd.grad(y, [x] + p, st["dy"])
    if kind == "round_trip":
        make = fp8.fp8_quantize_rows if case["block"] == "rows" else fp8.fp8_quantize_blocks
        q, s = make(x, dtype=_FP8[case["fp8"]])
        return fp8.fp8_dequantize(q, s, cols=x.shape[1], out_dtype=x.dtype)
    if kind == "linear":
        q, s = fp8.fp8_quantize_rows(x)
        return fp8.fp8_matmul(q, s, *st["w"], bias=st["b"], activation=case["act"], out_dtype=x.dtype)
    if kind == "linear_grad":
        leaves = st["leaves"]
        y = fp8.fp8_linear(*leaves, grad_dtype=_FP8[case["fp8"]])
        return [y.detach(), *torch.autograd.grad(y, [t for t in leaves if t is not None], st["dy"])]
    q, s = norm.layer_norm_fp8(x, eps=_EPS, scale=st["p"][0], shift=st["p"][1])
    h = fp8.fp8_matmul(q, s, *st["w"][0], bias=st["b"][0], activation="gelu_tanh", out_dtype=x.dtype)
    q, s = fp8.fp8_quantize_rows(h)
    return fp8.fp8_matmul(q, s, *st["w"][1], bias=st["b"][1], out_dtype=x.dtype)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------------------------------ work
def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    kind = case["kind"]
    if kind in ("norm", "norm_grad"):
        b, m, c = case["batch"], case["batch"] * case["rows"], case["cols"]
        p = 2 * c * e if case["form"] == "affine" else 2 * b * c * 4
        if kind == "norm":
            return {"bytes": 2 * m * c * e + p, "flops": 8 * m * c}
        return {"bytes": 4 * m * c * e + 2 * p, "flops": 22 * m * c}
    if kind == "round_trip":
        m, c = case["rows"], case["cols"]
        return {"bytes": 2 * m * c * e, "flops": 4 * m * c}
    m, k, n = case.get("batch", 1) * case["rows"], case["k"], case["n"]
    if kind == "linear":
        return {"bytes": m * k * e + n * k + m * n * e + (n * e if case["bias"] else 0), "flops": 2 * m * n * k}
    if kind == "linear_grad":
        return {"bytes": 2 * (m * k + m * n + n * k) * e + (2 * n * e if case["bias"] else 0), "flops": 6 * m * n * k}
    return {"bytes": 2 * m * k * e + 2 * n * k + (n + k) * e + 8 * k, "flops": 4 * m * n * k}


# ------------------------------------------------------------------------------------------------ in 64 bits
def _pow64(e):
    """2^e for whole e in doubles, from its bits."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _round64(v, digits, lowest):
    """v rounded to nearest even at ``digits`` significant bits, no step below 2^(lowest - digits + 1)."""
    a = v.abs()
    a = torch.where(a > 0, a, torch.ones_like(a))
    p = a.log2().round()  # within one of the exponent, then set right: a device's log2 need not be exact
    p = torch.where(_pow64(p) > a, p - 1, p)
    p = torch.where(_pow64(p + 1) <= a, p + 1, p).clamp(min=lowest)
    step = _pow64(p - (digits - 1))
    return torch.round(v / step) * step


def _fp8_64(x, tall, fp8):
    """What quantising leaves of x, in blocks of ``tall`` rows by 128 columns: every block by itself, cut from x."""
    digits, lowest = (4, -6) if fp8 == "e4m3" else (3, -14)
    out = torch.empty_like(x)
    for c in range(0, x.shape[1], 128):
        strip = x[:, c:c + 128]
        if tall == 1:
            top = strip.abs().amax(1, keepdim=True)
        else:
            top = torch.cat([strip[r:r + tall].abs().amax().expand(strip[r:r + tall].shape[0], 1)
                             for r in range(0, x.shape[0], tall)])
        e = torch.where(top > 0, top / _TOP[fp8], torch.ones_like(top)).log2().round()
        e = torch.where(top > _TOP[fp8] * _pow64(e), e + 1, e)
        e = torch.where(top <= _TOP[fp8] * _pow64(e - 1), e - 1, e)
        e = torch.where(top > 0, e.clamp(-127, 127), torch.zeros_like(top))
        s = _pow64(e)
        out[:, c:c + 128] = _round64(strip / s, digits, lowest) * s
    return out


def _as_type64(v, dtype):
    digits, lowest = {"bf16": (8, -126), "fp16": (11, -14), "fp32": (24, -126)}[dtype]
    return _round64(v, digits, lowest)


def _norm64(x, p, form):
    var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
    n = (x - mean) / (var + _EPS).sqrt()
    gain = p[0] if form == "affine" else p[0] + 1
    return n, gain, (var + _EPS).sqrt(), torch.addcmul(p[1], n, gain)


def exact(case, seed):
    g = _gen(seed)
    kind, name = case["kind"], case["dtype"]
    dtype = _DTYPES[name]
    if kind in ("norm", "norm_grad"):
        b, s, c = case["batch"], case["rows"], case["cols"]
        x = (_activations(g, b * s, c, torch.float32) + 0.3).to(dtype).view(b, s, c).double()
        if case["form"] == "affine":
            p = [(1 + _small(g, c, torch.float32)).to(dtype).double(), _small(g, c, dtype).double()]
        else:
            mod = 0.3 * torch.randn(b, 6, c, generator=g, device=_DEV)
            p = [mod[:, 1:2].double(), mod[:, 0:1].double()]
        n, gain, sd, y = _norm64(x, p, case["form"])
        if kind == "norm":
            return y
        del x
        dy = _activations(g, b * s, c, dtype, 1e-2).view(b, s, c).double()
        t = dy * gain
        # dx = (I - 11'/C - nn'/C) t / sd, the projection off the constant and off n
        dx = t - (t * n).mean(-1, keepdim=True) * n
        dx = (dx - t.mean(-1, keepdim=True)) / sd
        rows = "bsc->c" if case["form"] == "affine" else "bsc->bc"
        keep = (lambda v: v) if case["form"] == "affine" else (lambda v: v.unsqueeze(1))
        return y, dx, keep(torch.einsum(rows, dy * n)), keep(torch.einsum(rows, dy))
    if kind == "round_trip":
        rows = case["block"] == "rows"
        x = (_activations if rows else _weights)(g, case["rows"], case["cols"], dtype).double()
        return _fp8_64(x, 1 if rows else 128, case["fp8"])

    def layer(x, w, b, act):
        y = torch.mm(x, w.t())
        y = y if b is None else y + b.double()
        if act == "gelu_tanh":
            u = (y + 0.044715 * y.pow(3)) * math.sqrt(8 / math.pi)
            y = y * torch.sigmoid(u)  # (1 + tanh(u / 2)) / 2 = sigmoid(u)
        return y

    k, n = case["k"], case["n"]
    m = case.get("batch", 1) * case["rows"]
    x = _activations(g, m, k, dtype).double()
    if kind == "ffn":
        b = case["batch"]
        mod = (0.3 * torch.randn(b, 6, k, generator=g, device=_DEV)).double()
        w1 = _fp8_64(_weights(g, n, k, dtype).double(), 128, "e4m3")
        w2 = _fp8_64(_weights(g, k, n, dtype).double(), 128, "e4m3")
        b1, b2 = _small(g, n, dtype), _small(g, k, dtype)
        h = _norm64(x.view(b, -1, k), (mod[:, 4:5], mod[:, 3:4]), "modulated")[3].flatten(0, 1)
        h = layer(_fp8_64(_as_type64(h, name), 1, "e4m3"), w1, b1, "gelu_tanh")
        return layer(_fp8_64(_as_type64(h, name), 1, "e4m3"), w2, b2, "none").view(b, -1, k)
    w = _fp8_64((w16 := _weights(g, n, k, dtype)).double(), 128, "e4m3")
    del w16
    b = _small(g, n, dtype) if case["bias"] else None
    y = layer(_fp8_64(x, 1, "e4m3"), w, b, case.get("act", "none"))
    if kind == "linear":
        return y
    dy = _activations(g, m, n, dtype, 1e-2).double()
    dx = torch.mm(_fp8_64(dy, 1, case["fp8"]), w)
    dyc = _fp8_64(dy.t().contiguous(), 1, case["fp8"])
    dw = torch.mm(dyc, _fp8_64(x.t().contiguous(), 1, "e4m3").t())
    return [y, dx, dw] + ([] if b is None else [dy.sum(0)])
