"""Definitions in 64 bits of dense attention, of rotary positions behind a norm and of the gated residual, with the error
bounds their kernels are held to."""

import math

import torch

from norm_fp8_helpers import HALF, TINY, U32, say, within  # noqa: F401


def lens_of(n, lens, batch):
    return [n] * batch if lens is None else [min(max(int(v), 0), n) for v in lens]


def attention64(q, k, v, dy=None, scale=None, q_lens=None, k_lens=None, half=2.0 ** -8):
    """``{name: (value, bound)}`` of o, lse and, with dy, of dq, dk and dv, all float64 on the CPU.

    Bounds, before each result's own rounding.  ``half`` (h) is half a step of the type.  A score is an fp32 sum of D
    products, and its exponent's argument, the subtraction and the exponential are fp32: with g = (D + 16) 2^-23 scale |q||k|
    the largest of a row (2^-23, a whole step, per addition), a probability is off by a factor within 1 +- 4 g', g' = g +
    2^-20.  P is rounded (h) and o divided by the sum of the rounded values (another h at most), sums of N terms are off by (N
    + 16) 2^-23 of the sum of magnitudes.  D sees o's error before its rounding (h^2 with the rest of it), dS its own
    rounding (h), P's and dP's fp32 errors and D's error."""
    q, k, v = (t.detach().double().cpu() for t in (q, k, v))
    dy = None if dy is None else dy.detach().double().cpu()
    b, h, sq, d = q.shape
    kh, sk = k.shape[1:3]
    scale = d ** -0.5 if scale is None else scale
    out = {n: (torch.zeros(s, dtype=torch.float64), torch.zeros(s, dtype=torch.float64))
           for n, s in (("o", q.shape), ("dq", q.shape), ("dk", k.shape), ("dv", v.shape))}
    out["lse"] = torch.full((b, h, sq), -math.inf, dtype=torch.float64), torch.zeros(b, h, sq, dtype=torch.float64)
    step = 2.0 ** -23
    for i, (nq, nk) in enumerate(zip(lens_of(sq, q_lens, b), lens_of(sk, k_lens, b))):
        if nq == 0 or nk == 0:
            continue
        for j in range(h):
            kj = j // (h // kh)
            qq, kk, vv = q[i, j, :nq], k[i, kj, :nk], v[i, kj, :nk]
            s = scale * qq @ kk.t()
            size = scale * qq.abs() @ kk.abs().t()
            lse = torch.logsumexp(s, 1, keepdim=True)
            p = torch.exp(s - lse)
            g = 4 * ((d + 16) * step * size.amax(1, keepdim=True) + 2.0 ** -20)
            o = p @ vv
            mass = p @ vv.abs()
            eo = (2 * half + 2 * g + (nk + 16) * step) * mass
            out["o"][0][i, j, :nq], out["o"][1][i, j, :nq] = o, eo
            out["lse"][0][i, j, :nq], out["lse"][1][i, j, :nq] = lse[:, 0], (g + (nk + 16) * step)[:, 0] + 2.0 ** -21 * lse[:, 0].abs()
            if dy is None:
                continue
            do = dy[i, j, :nq]
            out["dv"][0][i, kj, :nk] += p.t() @ do
            out["dv"][1][i, kj, :nk] += (p * (half + 2 * g + ((h // kh) * nq + 16) * step)).t() @ do.abs()
            dp = do @ vv.t()
            dd = (do * o).sum(1, keepdim=True)
            edp = (d + 16) * step * do.abs() @ vv.abs().t()
            edd = (do.abs() * (eo + (half ** 2 + (d + 16) * step) * (o.abs() + eo))).sum(1, keepdim=True)
            ds = p * (dp - dd)
            eds = half * ds.abs() + (1 + half) * (2 * g * ds.abs() + p * (1 + 2 * g) * (edp + edd))
            if half < 2.0 ** -9:  # fp16 keeps dS within 2^-25 of 2^-14 of twice the largest |do| |v|
                eds = eds + 2.0 ** -38 * do.norm(dim=1).max() * vv.norm(dim=1).max()
            out["dq"][0][i, j, :nq] = scale * ds @ kk
            out["dq"][1][i, j, :nq] = scale * (eds + (nk + 16) * step * ds.abs()) @ kk.abs()
            out["dk"][0][i, kj, :nk] += scale * ds.t() @ qq
            out["dk"][1][i, kj, :nk] += scale * (eds + ((h // kh) * nq + 16) * step * ds.abs()).t() @ qq.abs()
    return out


def held(got, want, name=""):
    """A result within its bound and its own rounding, exactly 0 where the definition is without any term."""
    value, bound = want
    got = got.detach().cpu()
    print("  ", name, end="")
    assert got.shape == value.shape, (name, got.shape, value.shape)
    finite = value.isfinite()  # a log-sum-exp over no keys is -inf
    assert torch.equal(got[~finite].double(), value[~finite]), name
    got, value, bound = got[finite], value[finite], bound[finite]
    none = (value == 0) & (bound == 0)
    assert torch.equal(got[none].double(), value[none]), name
    within(got, value, bound)


def turned64(x, angle, interleaved):
    """float64 heads ``[.., D]`` with pair j turned by ``angle [.., D / 2]``."""
    d = x.shape[-1]
    cos, sin = angle.cos(), angle.sin()
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    a, b = x[..., :d // 2], x[..., d // 2:]
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)


def angles64(positions, axes, theta, d):
    """float64 angles ``[.., D / 2]`` of positions ``[.., axes]``."""
    thetas = theta if isinstance(theta, (list, tuple)) else [theta] * len(axes)
    parts = [positions[..., i, None].double() * float(t) ** (-torch.arange(0, n, 2).double() / max(n, 1))
             for i, (n, t) in enumerate(zip(axes, thetas))]
    rest = d // 2 - sum(axes) // 2
    return torch.cat(parts + [torch.zeros(*positions.shape[:-1], rest).double()], -1)


def grid_positions(grid, start, rows):
    """``[rows, axes]``: a grid's positions, 0 behind it."""
    cells = math.prod(grid)
    p = torch.cartesian_prod(*(torch.arange(s, s + n) for s, n in zip(start, grid))).view(cells, len(grid))
    return torch.cat([p, torch.zeros(rows - cells, len(grid), dtype=p.dtype)])


def rope64(x, angle, norm, weight, eps, interleaved, dy=None):
    """``{name: (value, bound)}`` of y and, with dy, of dx and dweight (float64, CPU).

    Every step is fp32 on values of the row's size: the sum of squares of C terms is off by (C + 8) 2^-24 of itself, a cosine
    by 2^-22, and each of the about eight products and sums behind them by 2^-24 of the magnitudes that enter it.  A row's mean
    of g x has (C + 8) 2^-24 of the mean of magnitudes."""
    x = x.detach().double().cpu()
    b, s, h, d = x.shape
    angle = angle[..., None, :]
    over = {"row": (2, 3), "head": (3,), "none": None}[norm]
    c = {"row": h * d, "head": d, "none": 1}[norm]
    w = torch.ones(h, d).double() if weight is None else weight.detach().double().cpu().view(-1, d)
    rel = (c + 8) * U32 + 2.0 ** -21
    rstd = 1.0
    if over:
        rstd = 1 / ((x * x).mean(over, keepdim=True) + eps).sqrt()

    def size(t):  # what a turn adds up
        return t.abs() + (torch.roll(t.unflatten(-1, (-1, 2)), 1, -1).flatten(-2) if interleaved else torch.roll(t, d // 2, -1)).abs()

    n = x * rstd * (w if over else 1.0)
    out = {"y": (turned64(n, angle, interleaved), rel * size(n))}
    if dy is not None:
        g = turned64(dy.detach().double().cpu(), -angle, interleaved)
        eg = 2.0 ** -21 * size(dy.detach().double().cpu())
        if not over:
            out["dx"] = g, eg
            return out
        u, eu = g * w, eg * w.abs()
        nh = x * rstd
        mean = (u * nh).mean(over, keepdim=True)
        emean = (eu * nh.abs()).mean(over, keepdim=True) + rel * (u * nh).abs().mean(over, keepdim=True)
        dx = rstd * (u - nh * mean)
        out["dx"] = dx, rstd * (eu + rel * u.abs() + nh.abs() * (emean + 3 * rel * (u * nh).abs().mean(over, keepdim=True)))
        dims = (0, 1) if norm == "row" else (0, 1, 2)
        terms = b * s * (1 if norm == "row" else h)
        out["dweight"] = (g * nh).sum(dims).flatten(), \
            ((eg * nh.abs()).sum(dims) + (rel + (terms + 8) * U32) * (g * nh).abs().sum(dims)).flatten()
    return out


def residual64(x, branch, gate, w, c, eps, dtype, dh=None, dy=None, shared=(False, False, False)):
    """``{name: (value, bound)}`` of h, y and, with gradients, of dx, dbranch and the three sums; w (1 + scale) and c as they
    multiply and add, gate or None; ``[B, S, C]`` float64 on the CPU, parameters broadcastable.  y is of h as it is stored.

    fp32 throughout: sums of C or of the rows' terms are off by (terms + 16) 2^-24 of the sum of magnitudes, the statistics by
    as much of the deviations, and each further step by 2^-24 of what enters."""
    cols = x.shape[-1]
    one = torch.ones(1, dtype=torch.float64)
    gt = one if gate is None else gate
    h = x + gt * branch
    eh = 2 * U32 * (x.abs() + (gt * branch).abs())
    out = {"h": (h, eh)}
    if w is None:
        if dh is not None:
            out["dx"], out["dbranch"] = (dh, 0 * dh), (dh * gt, 2 * U32 * (dh * gt).abs())
            out["dgate"] = (dh * branch).sum(1, keepdim=True), (x.shape[1] + 16) * U32 * (dh * branch).abs().sum(1, keepdim=True)
        return out
    hr = h.to(dtype).double()
    mean = hr.mean(-1, keepdim=True)
    dev = hr - mean
    rstd = 1 / ((dev * dev).mean(-1, keepdim=True) + eps).sqrt()
    n = dev * rstd
    # a stored h that is the neighbour of this one (its fp32 sum lay the other way of a midpoint) moves its n by a step; half a
    # step is HALF times the power of two at or below h
    half = (HALF[dtype] * 2.0 ** (torch.frexp(h)[1] - 1).double()).clamp(min=TINY[dtype])
    move = torch.where(eh >= ((h - hr).abs() - half).abs(), 2 * half, torch.zeros_like(h))
    stat = (cols + 16) * U32
    en = rstd * move + 2 * U32 * (n.abs() + rstd * mean.abs()) + stat * (n.abs() + rstd * hr.abs().mean(-1, keepdim=True)) + \
        (n.abs() + 1) * (rstd * move).mean(-1, keepdim=True) * (1 + n.abs().amax(-1, keepdim=True))
    out["y"] = n * w + c, en * w.abs() + 2 * U32 * ((n * w).abs() + c.abs())
    if dy is None:
        return out
    g = dy * w
    m1, m2 = g.mean(-1, keepdim=True), (g * n).mean(-1, keepdim=True)
    a1, a2 = g.abs().mean(-1, keepdim=True), (g * n).abs().mean(-1, keepdim=True)
    dt = rstd * (g - m1 - n * m2) + (0 if dh is None else dh)
    big = rstd * (g.abs() + a1 + n.abs() * a2)
    edt = stat * big + 4 * U32 * (big + (0 if dh is None else dh.abs())) + \
        rstd * (en * a2 + n.abs() * (g.abs() * en).mean(-1, keepdim=True)) + 2 * stat * big
    out["dx"] = dt, edt
    out["dbranch"] = dt * gt, edt * gt.abs() + U32 * (dt * gt).abs()

    def sums(v, e, over_all):
        dims = (0, 1) if over_all else 1
        count = v.shape[0] * v.shape[1] if over_all else v.shape[1]
        t, et = v.sum(dims, keepdim=True), (e + (count + 16) * U32 * v.abs()).sum(dims, keepdim=True)
        return t, et

    out["dgate"] = sums(dt * branch, edt * branch.abs(), shared[0])
    out["dw"] = sums(dy * n, dy.abs() * en, shared[1])
    out["dc"] = sums(dy, 0 * dy, shared[2])
    return out
