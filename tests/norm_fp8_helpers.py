"""Definitions in 64 bits of the layer norm and of the 8-bit blocks, and the error bounds their kernels are held to."""

import math

import torch

U32 = 2.0 ** -24  # half a step of fp32, relative
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: U32}  # half a step of each type (eps / 2)
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}  # half its smallest step
TOP = {torch.float8_e4m3fn: 448.0, torch.float8_e5m2: 57344.0}
DIGITS = {torch.float8_e4m3fn: (4, -6), torch.float8_e5m2: (3, -14)}


def say(*a):
    print("[case]", *a, flush=True)


def within(got, want, bound):
    """Every element of ``got`` within ``bound`` and its own rounding of ``want`` (float64)."""
    limit = bound + HALF[got.dtype] * (want.abs() + bound) + TINY[got.dtype]
    err = (got.double() - want).abs()
    worst = (err / limit).max().item() if err.numel() else 0.0
    print("   worst share of its bound %.3f" % worst, flush=True)
    assert worst <= 1.0, worst


def pow2(e):
    """2^e for whole e as a double, from its bits."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def norm64(x, w, b, eps):
    """``(n, rstd, y)`` of a layer norm with gain w and offset b (broadcastable), all float64."""
    mean = x.mean(-1, keepdim=True)
    d = x - mean
    rstd = 1 / ((d * d).mean(-1, keepdim=True) + eps).sqrt()
    n = d * rstd
    return n, rstd, n * w + b


def block_exponents64(x, tall, dtype):
    """Exponents ``[ceil(M / tall), ceil(K / 128)]`` of a float64 matrix's blocks, over finite values."""
    x = torch.where(x.isfinite(), x.abs(), torch.zeros_like(x))
    rows = []
    for r in range(0, x.shape[0], tall):
        rows.append(torch.stack([x[r:r + tall, c:c + 128].max() for c in range(0, x.shape[1], 128)]) if tall > 1 else
                    torch.cat([x[r, c:c + 128].max()[None] for c in range(0, x.shape[1], 128)]))
    top = torch.stack(rows)
    e = torch.zeros_like(top)
    for i, v in enumerate(top.flatten().tolist()):
        if v > 0:
            m, p = math.frexp(v / TOP[dtype])  # exact: the divisor is 7 2^k and v has 24 digits, so compare products
            k = p - 1
            while v > TOP[dtype] * 2.0 ** k:
                k += 1
            while v <= TOP[dtype] * 2.0 ** (k - 1):
                k -= 1
            e.view(-1)[i] = max(k, -127)
    return e


def round8(v, dtype):
    """float64 values rounded to nearest even in an 8-bit type, within its range."""
    digits, lowest = DIGITS[dtype]
    _, p = torch.frexp(v)
    step = pow2((p - 1).clamp(min=lowest) - (digits - 1))
    return torch.round(v / step) * step


def spread(e, tall, m, k):
    return pow2(e).repeat_interleave(128, 1)[:, :k].repeat_interleave(tall, 0)[:m]


def fp8_values64(x, tall, dtype):
    """What quantising leaves of a float64 matrix: ``(values, exponents)``."""
    e = block_exponents64(x, tall, dtype)
    s = spread(e, tall, *x.shape)
    v = round8(torch.where(x.isfinite(), x, torch.zeros_like(x)) / s, dtype) * s
    return torch.where(x.isfinite(), v, x), e


def gelu64(y):
    return 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))


def product_bound(a, b, wide):
    """Elementwise bound on ``|c - a b^T|`` of a product of float64 matrices ``a [M, K], b [N, K]`` before its rounding.

    fp32 accumulation: one rounding (or cut, so a whole step) of 2^-23 per addition, at most K + 8 of them, of sums no
    larger than sum |a b|.  The 8-bit instructions besides cut each of the eight products of a group up to 2^-12 of the
    group's largest (13 bits below its exponent, and a product's digits reach 3 1/16): at most 8 2^-12 sum |a b| for any
    grouping."""
    s = a.abs() @ b.abs().t()
    return s * ((a.shape[1] + 8) * 2.0 ** -23 + (0 if wide else 2.0 ** -9))


def whole_numbers(g, m, k, dtype, device, most=2):
    """Small whole numbers times a power of two per row and block of 128, as given by ``g``."""
    return torch.randint(-most, most + 1, (m, k), generator=g, device=device).to(dtype)
