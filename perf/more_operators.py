"""The attention half of a DiT block in training and serving, as measurable cases.

``own`` false computes every operator from elementary torch operations; true calls ``svoo_amd.dense``, ``svoo_amd.rope``
and ``svoo_amd.norm``.  ``kind`` names the operator:

* ``attn``           dense attention over heads that may share keys and values, sequences padded to one length
* ``attn_grad``      the same with its backward pass: o, dq, dk, dv
* ``rope``           RMS norm (over a token's whole row or per head, or none) and rotary positions on several axes
* ``rope_grad``      the same with its backward pass: y, dx, and dweight with a norm
* ``residual``       a gated residual and the norm behind it: h = x + gate b, y = LN(h) (affine or modulated)
* ``residual_grad``  the same with its backward pass, for gradients that arrive at h and at y

Queries and keys behind a sequence's length are padding: their rows of o and of the gradients are 0.
"""

import math

import torch

own = False

_DEV = "cuda:0"
_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_EPS = 1e-6
_THETA = 10000.0


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # One new token's query against a cache of a 480p clip's keys and values (21 x 30 x 52 tokens): reading is all.
        dict(name="attn_one_query", kind="attn", batch=1, heads=12, groups=1, sq=1, sk=32760, d=128, q_pad=0, k_pad=0,
             dtype="bf16"),
        # The 14B model's cross-attention at 720p to a prompt of 512 text tokens: long queries, few keys.
        dict(name="attn_text_720p", kind="attn", batch=1, heads=40, groups=1, sq=75600, sk=512, d=128, q_pad=0, k_pad=0,
             dtype="bf16"),
        # Fine-tuning on three ragged sequences in fp16, four query heads to a key head; the last has no keys at all.
        dict(name="attn_grad_odd", kind="attn_grad", batch=3, heads=8, groups=4, sq=1037, sk=771, d=64, q_pad=100,
             k_pad=400, dtype="fp16"),
        # Training the 1.3B model's cross-attention at 480p.
        dict(name="attn_grad_text", kind="attn_grad", batch=1, heads=12, groups=1, sq=32760, sk=512, d=128, q_pad=0,
             k_pad=0, dtype="bf16"),
        # Training the 1.3B model's self-attention at 480p: the largest.
        dict(name="attn_grad_480p", kind="attn_grad", batch=1, heads=12, groups=1, sq=32760, sk=32760, d=128, q_pad=0,
             k_pad=0, dtype="bf16"),
        # One token's query row of the 1.3B model: a launch is all there is.
        dict(name="rope_one_token", kind="rope", batch=1, rows=1, heads=12, d=128, axes=3, norm="row", at="positions",
             pairs="neighbours", dtype="bf16"),
        # A query projection of the 1.3B model at 480p.
        dict(name="rope_480p", kind="rope", batch=1, rows=32760, heads=12, d=128, axes=3, norm="row", at="grid",
             pairs="neighbours", dtype="bf16"),
        # Two ragged batches of image tokens with positions far from 0, norms per head, halves of a head as pairs, in fp32.
        dict(name="rope_grad_odd", kind="rope_grad", batch=2, rows=777, heads=5, d=72, axes=2, norm="head", at="positions",
             pairs="halves", dtype="fp32"),
        # A training step of the 14B model's query rows at 720p.
        dict(name="rope_grad_720p", kind="rope_grad", batch=1, rows=75600, heads=40, d=128, axes=3, norm="row", at="grid",
             pairs="neighbours", dtype="bf16"),
        # The end of a block and the norm of the next, 1.3B at 480p: modulated, the gate in fp32.
        dict(name="residual_480p", kind="residual", batch=1, rows=32760, cols=1536, gate=True, form="modulated",
             dtype="bf16"),
        # Two short sequences of a width that is no multiple of anything, in fp16, without a gate.
        dict(name="residual_grad_odd", kind="residual_grad", batch=2, rows=513, cols=999, gate=False, form="affine",
             dtype="fp16"),
        # A training step of the 14B model's gated residual and affine norm at 720p.
        dict(name="residual_grad_720p", kind="residual_grad", batch=1, rows=75600, cols=5120, gate=True, form="affine",
             dtype="bf16"),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn_grad", "attn_grad", "rope", "rope_grad", "residual", "residual_grad"])
    if kind in ("attn", "attn_grad"):
        groups = rng.choice([1, 1, 1, 2, 4])
        heads = groups * rng.choice([1, 2, 3, 5, 8, 10])
        d = rng.choice([128, 128, 128, 64, 64, 88, 80, 40])
        batch = rng.choice([1, 1, 2, 3])
        most = min(3.0e11 / (batch * heads * d), 1.5e9 / (batch * groups))  # pairs of a query and a key
        sq = _spread(rng, 1, 40000.0)
        sk = _spread(rng, 1, min(40000.0, most / sq))
        pad = rng.random() < 0.4
        return dict(kind=kind, batch=batch, heads=heads, groups=groups, sq=sq, sk=sk, d=d,
                    q_pad=rng.randint(0, sq // 2) if pad else 0, k_pad=rng.randint(0, sk) if pad else 0,
                    dtype=rng.choice(["bf16", "bf16", "bf16", "fp16"]))
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    batch = rng.choice([1, 1, 2, 3])
    if kind in ("rope", "rope_grad"):
        d = rng.choice([128, 128, 64, 96, 72, 48, 160])
        heads = rng.choice([1, 2, 5, 12, 16, 20, 40])
        rows = _spread(rng, 1, min(75600.0, 2.0e8 / (d * heads * batch)))
        return dict(kind=kind, batch=batch, rows=rows, heads=heads, d=d, axes=rng.choice([1, 2, 3, 3]),
                    norm=rng.choice(["row", "row", "head", "none"]), at=rng.choice(["grid", "positions"]),
                    pairs=rng.choice(["neighbours", "neighbours", "halves"]), dtype=dtype)
    cols = _spread(rng, 24, 8192)
    if rng.random() < 0.5:
        cols = max(64, cols // 64 * 64)
    rows = _spread(rng, 1, min(75600.0, 2.0e8 / (cols * batch)))
    return dict(kind=kind, batch=batch, rows=rows, cols=cols, gate=rng.random() < 0.7,
                form=rng.choice(["affine", "modulated"]), dtype=dtype)


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=_DEV).manual_seed(seed)


def _noise(g, *shape, level=1.0):
    return level * torch.randn(*shape, generator=g, device=_DEV)


def _stream(g, rows, cols, level=1.0):
    """Rows of a residual stream: unit noise on channels of unequal size, a few of them far larger."""
    chan = torch.exp(0.5 * torch.randn(cols, generator=g, device=_DEV))
    far = torch.rand(cols, generator=g, device=_DEV) < 0.01
    return _noise(g, rows, cols, level=level) * torch.where(far, 8.0 * chan, chan)


def _lengths(case):
    """Valid queries and keys of each batch entry."""
    b = range(case["batch"])
    return ([max(0, case["sq"] - i * case["q_pad"]) for i in b], [max(0, case["sk"] - i * case["k_pad"]) for i in b])


def _axes(case):
    """The channels of each axis: of three, two equal ones and the rest to the first (time)."""
    d, n = case["d"], case["axes"]
    if n == 1:
        return (d,)
    if n == 2:
        return (d - 2 * (d // 4), 2 * (d // 4))
    return (d - 4 * (d // 6), 2 * (d // 6), 2 * (d // 6))


def _grid(case):
    """Whole rows of the last axes; a clip's leading frames where the rows are a 720p or 480p clip's."""
    s, n = case["rows"], case["axes"]
    if n == 1:
        return (s,)
    if n == 3:
        for h, w in ((45, 80), (30, 52)):
            if s % (h * w) == 0:
                return (s // (h * w), h, w)
    w = max(k for k in range(1, 41) if s % k == 0)
    if n == 2:
        return (s // w, w)
    h = max(k for k in range(1, 41) if s // w % k == 0)
    return (s // w // h, h, w)


def prepare(case, seed):
    g = _gen(seed)
    dtype = _DTYPES[case["dtype"]]
    kind, b = case["kind"], case["batch"]
    train = kind.endswith("_grad")
    st = {"case": case}
    if kind.startswith("attn"):
        h, kh, d = case["heads"], case["heads"] // case["groups"], case["d"]
        # queries and keys as projections leave them after a norm, [B, S, H, D] in memory; a few keys stand out
        q = _noise(g, b, case["sq"], h, d)
        k = _noise(g, b, case["sk"], kh, d) + 0.5 * _noise(g, 1, 1, kh, d)
        far = torch.rand(b, case["sk"], 1, 1, generator=g, device=_DEV) < 0.02
        k = torch.where(far, 2.5 * k, k)
        v = _noise(g, b, case["sk"], kh, d) + 0.3 * _noise(g, 1, 1, kh, d)
        st["x"] = [t.to(dtype).transpose(1, 2).requires_grad_(train) for t in (q, k, v)]
        st["lens"] = [torch.tensor(n, dtype=torch.int32, device=_DEV) if case[p] else None
                      for n, p in zip(_lengths(case), ("q_pad", "k_pad"))]
        if train:
            st["dy"] = _noise(g, b, case["sq"], h, d, level=1e-2).to(dtype).transpose(1, 2)
        return st
    s = case["rows"]
    if kind.startswith("rope"):
        h, d = case["heads"], case["d"]
        x = _stream(g, b * s, h * d).to(dtype).view(b, s, h, d)
        st["axes"] = _axes(case)
        n = {"row": h * d, "head": d, "none": 0}[case["norm"]]
        w = (1 + _noise(g, n, level=0.1)).to(dtype) if n else None
        st["x"] = [x.requires_grad_(train)] + ([w.requires_grad_(train)] if n else [])
        if case["at"] == "grid":
            st["grid"], st["positions"] = _grid(case), None
        else:  # windows of long clips and large images: positions far from 0, in no order
            st["grid"] = None
            st["positions"] = torch.randint(0, 100000, (b, s, case["axes"]), generator=g, device=_DEV, dtype=torch.int32)
        if train:
            st["dy"] = _stream(g, b * s, h * d, 1e-2).to(dtype).view(b, s, h, d)
        return st
    c = case["cols"]
    x = (_stream(g, b * s, c) + 0.3).to(dtype).view(b, s, c)
    branch = _stream(g, b * s, c, 0.5).to(dtype).view(b, s, c)
    mod = _noise(g, b, 6, c, level=0.3)  # a block's six modulation vectors, in fp32
    gate = mod[:, 2:3] if case["gate"] else None
    p = (mod[:, 4:5], mod[:, 3:4]) if case["form"] == "modulated" else \
        ((1 + _noise(g, c, level=0.1)).to(dtype), _noise(g, c, level=0.1).to(dtype))
    st["x"] = [None if t is None else t.detach().requires_grad_(train) for t in (x, branch, gate, *p)]
    if train:
        st["dh"], st["dy"] = (_stream(g, b * s, c, 1e-2).to(dtype).view(b, s, c) for _ in range(2))
    return st


# ------------------------------------------------------------------------------------------------ plain forms
def _attn_plain(st):
    case = st["case"]
    q, k, v = (t.detach() for t in st["x"])
    b, h, sq, d = q.shape
    kh, sk = k.shape[1:3]
    train = case["kind"] == "attn_grad"
    q_len, k_len = (torch.full((b,), n, device=q.device) if t is None else t for n, t in zip((sq, sk), st["lens"]))
    # query rows of the heads that share a key head, one after the other: [B, Hk, G S, D]
    heads = lambda t: t.reshape(b, kh, h // kh * sq, d).float()  # noqa: E731
    q_on = torch.arange(sq, device=q.device) < q_len[:, None]
    k_on = (torch.arange(sk, device=q.device) < k_len[:, None])[:, None, None]
    q_on = q_on.repeat(1, h // kh)[:, None, :, None]
    qs, ks, vs = heads(q), k.float(), v.float()
    ds = heads(st["dy"]) if train else None
    outs = [torch.empty_like(qs), torch.empty_like(qs), torch.empty_like(ks), torch.empty_like(vs)]
    # all key heads at once, or as many as leave room for their probabilities
    step = max(1, int(2 ** 31 // (b * qs.shape[2] * sk)))
    for i in range(0, kh, step):
        at = slice(i, i + step)
        qc, kc, vc = (t[:, at].contiguous() for t in (qs, ks, vs))
        s = (qc @ kc.transpose(2, 3).contiguous()) * d ** -0.5
        s = torch.where(k_on, s, -math.inf)
        top = s.amax(-1, keepdim=True).clamp(min=-3e38)
        p = torch.exp(s - top)
        del s
        total = p.sum(-1, keepdim=True)
        p = p / torch.where(total > 0, total, torch.ones_like(total))
        o = p @ vc
        outs[0][:, at] = torch.where(q_on, o, 0.0)
        if train:
            dy = torch.where(q_on, ds[:, at], 0.0)
            outs[3][:, at] = p.transpose(2, 3).contiguous() @ dy
            dp = dy @ vc.transpose(2, 3).contiguous()
            p = p * (dp - (dy * o).sum(-1, keepdim=True)) * d ** -0.5
            del dp
            outs[1][:, at] = p @ kc
            outs[2][:, at] = p.transpose(2, 3).contiguous() @ qc
        del p, o
    outs = [t.reshape(b, h, sq, d).to(q.dtype) for t in outs[:2]] + [t.to(q.dtype) for t in outs[2:]]
    return outs if train else outs[0]


def _rope_plain(st):
    case = st["case"]
    x, *w = (t.detach() for t in st["x"])
    b, s, h, d = x.shape
    pos = st["positions"]
    if pos is None:
        n = torch.arange(s, device=x.device)
        pos = []
        for size in reversed(st["grid"]):
            pos.insert(0, n % size)
            n = n // size
        pos = torch.stack(pos, -1)[None]
    angle = torch.cat([pos[..., a, None].double() * _THETA ** (-torch.arange(0, n, 2, device=x.device).double() / n)
                       for a, n in enumerate(st["axes"])], -1)  # far positions: in 64 bits
    cos, sin = angle.cos().float()[:, :, None], angle.sin().float()[:, :, None]
    halves = case["pairs"] == "halves"

    def turn(t, sin):
        if halves:
            u, v = t[..., :d // 2], t[..., d // 2:]
            return torch.cat([u * cos - v * sin, u * sin + v * cos], -1)
        u, v = t[..., 0::2], t[..., 1::2]
        return torch.stack([u * cos - v * sin, u * sin + v * cos], -1).flatten(-2)

    f = x.float()
    over = {"row": (2, 3), "head": 3, "none": None}[case["norm"]]
    if over:
        gain = w[0].float().view((h, d) if case["norm"] == "row" else (d,))
        rstd = torch.rsqrt((f * f).mean(over, keepdim=True) + _EPS)
        n = f * rstd
        y = turn(n * gain, sin)
    else:
        y = turn(f, sin)
    if case["kind"] == "rope":
        return y.to(x.dtype)
    dn = turn(st["dy"].float(), -sin)
    if not over:
        return y.to(x.dtype), dn.to(x.dtype)
    g = dn * gain
    dx = rstd * (g - n * (g * n).mean(over, keepdim=True))
    dw = (dn.double() * n).sum((0, 1) if case["norm"] == "row" else (0, 1, 2)).flatten()  # long sums
    return y.to(x.dtype), dx.to(x.dtype), dw.to(w[0].dtype)


def _residual_plain(st):
    case = st["case"]
    x, branch, gate, w, shift = (None if t is None else t.detach() for t in st["x"])
    dtype, affine = x.dtype, case["form"] == "affine"
    move = branch.float() if gate is None else branch.float() * gate.float()
    h = (x.float() + move).to(dtype)  # the stream is kept in its type, and normed as it is kept
    f = h.float()
    d = f - f.mean(-1, keepdim=True)
    rstd = torch.rsqrt((d * d).mean(-1, keepdim=True) + _EPS)
    n = d * rstd
    gain = w.float() if affine else 1 + w.float()
    y = n * gain + shift.float()
    if case["kind"] == "residual":
        return h, y.to(dtype)
    dy = st["dy"].float()
    g = dy * gain
    dt = st["dh"].float() + rstd * (g - g.mean(-1, keepdim=True) - n * (g * n).mean(-1, keepdim=True))
    over = (0, 1) if affine else 1
    sums = lambda t: t.sum(over, keepdim=not affine)  # noqa: E731
    out = [h, y.to(dtype), dt.to(dtype), (dt if gate is None else dt * gate.float()).to(dtype)]
    if gate is not None:
        out.append((dt.double() * branch.float()).sum(1, keepdim=True).to(gate.dtype))  # long sums
    return out + [sums(dy.double() * n).to(w.dtype), sums(dy.double()).to(shift.dtype)]


# ------------------------------------------------------------------------------------------------ the framework's
def _run_own(st):
    from svoo_amd import dense, norm, rope

    case, x = st["case"], st["x"]
    kind = case["kind"]
    if kind.startswith("attn"):
        o = dense.dense_attention(*x, q_lens=st["lens"][0], k_lens=st["lens"][1])
        return o if kind == "attn" else [o.detach(), *torch.autograd.grad(o, x, st["dy"])]
    if kind.startswith("rope"):
        y = rope.axis_rope(x[0], st["axes"], grid=st["grid"], positions=st["positions"], theta=_THETA, norm=case["norm"],
                           weight=x[1] if len(x) > 1 else None, eps=_EPS, interleaved=case["pairs"] == "neighbours")
        return y if kind == "rope" else (y.detach(), *torch.autograd.grad(y, x, st["dy"]))
    names = ("weight", "bias") if case["form"] == "affine" else ("scale", "shift")
    h, y = norm.residual_norm(*x[:3], eps=_EPS, **dict(zip(names, x[3:])))
    if kind == "residual":
        return h, y
    leaves = [t for t in x if t is not None]
    return [h.detach(), y.detach(), *torch.autograd.grad([h, y], leaves, [st["dh"], st["dy"]])]


def run(state):
    if own:
        return _run_own(state)
    case = state["case"]
    plain = {"attn": _attn_plain, "rope": _rope_plain, "residual": _residual_plain}[case["kind"].split("_")[0]]
    return plain(state)


# ------------------------------------------------------------------------------------------------ work
def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    kind, b = case["kind"], case["batch"]
    train = kind.endswith("_grad")
    if kind.startswith("attn"):
        h, kh, d = case["heads"], case["heads"] // case["groups"], case["d"]
        q, k = _lengths(case)
        pairs = h * d * sum(i * j for i, j in zip(q, k))
        rows_q, rows_k = b * case["sq"] * h * d, 2 * kh * d * sum(k)
        if not train:  # q, k and v in, o out
            return {"bytes": e * (sum(q) * h * d + rows_k + rows_q), "flops": 4 * pairs}
        return {"bytes": e * (2 * sum(q) * h * d + rows_k + 2 * rows_q + 2 * b * kh * d * case["sk"]), "flops": 14 * pairs}
    m = b * case["rows"]
    if kind.startswith("rope"):
        c = case["heads"] * case["d"]
        w = {"row": c, "head": case["d"], "none": 0}[case["norm"]] * e
        p = 4 * m * case["axes"] if case["at"] == "positions" else 0
        return {"bytes": (4 if train else 2) * m * c * e + (2 if train else 1) * w + p, "flops": (18 if train else 6) * m * c}
    c = case["cols"]
    p = (2 * c * e if case["form"] == "affine" else 8 * b * c) + (4 * b * c if case["gate"] else 0)
    # x, b in and h, y out; dh, dy in and dx, db out
    return {"bytes": (8 if train else 4) * m * c * e + (2 if train else 1) * p, "flops": (28 if train else 10) * m * c}


# ------------------------------------------------------------------------------------------------ in 64 bits
def _exact_attn(st):
    case = st["case"]
    q, k, v = (t.detach() for t in st["x"])
    train = case["kind"] == "attn_grad"
    if case["batch"] * case["heads"] > 200:
        return None
    outs = [torch.zeros(t.shape, dtype=torch.float64, device=t.device) for t in (q, q, k, v)]
    for i, (nq, nk) in enumerate(zip(*_lengths(case))):
        if nq == 0 or nk == 0:
            continue
        for j in range(case["heads"]):
            kj = j // case["groups"]
            one = [t.double().contiguous().requires_grad_(train) for t in (q[i, j, :nq], k[i, kj, :nk], v[i, kj, :nk])]
            with torch.set_grad_enabled(train):
                logits = torch.mm(one[0] / math.sqrt(case["d"]), one[1].t())
                o = torch.mm(torch.softmax(logits, 1), one[2])
                del logits
            outs[0][i, j, :nq] = o.detach()
            if train:
                got = torch.autograd.grad(o, one, st["dy"][i, j, :nq].double())
                outs[1][i, j, :nq] = got[0]
                outs[2][i, kj, :nk] += got[1]
                outs[3][i, kj, :nk] += got[2]
    return outs if train else outs[0]


def _exact_rope(st):
    case = st["case"]
    x, *w = (t.detach().double() for t in st["x"])
    train = case["kind"] == "rope_grad"
    b, s, h, d = x.shape
    if st["positions"] is not None:
        pos = st["positions"].double()
    else:
        pos = torch.cartesian_prod(*(torch.arange(n, dtype=torch.float64, device=x.device) for n in st["grid"]))
        pos = pos.view(1, s, -1)
    rates = []
    for a, n in enumerate(st["axes"]):
        j = torch.arange(n // 2, dtype=torch.float64, device=x.device)
        rates.append(pos[..., a:a + 1] * torch.exp(-2 * j / n * math.log(_THETA)))
    rates = torch.cat(rates, 2)
    turn = torch.polar(torch.ones_like(rates), rates)[:, :, None]
    leaves = [x.requires_grad_(train)] + [t.requires_grad_(train) for t in w]
    with torch.set_grad_enabled(train):
        n = x
        if case["norm"] == "row":
            n = torch.nn.functional.rms_norm(x.reshape(b, s, h * d), (h * d,), leaves[1], _EPS).view(b, s, h, d)
        elif case["norm"] == "head":
            n = torch.nn.functional.rms_norm(x, (d,), leaves[1], _EPS)
        if case["pairs"] == "halves":
            z = torch.complex(n[..., :d // 2], n[..., d // 2:]) * turn
            y = torch.cat([z.real, z.imag], -1)
        else:
            y = torch.view_as_real(torch.view_as_complex(n.unflatten(-1, (-1, 2))) * turn).flatten(-2)
    return (y.detach(), *torch.autograd.grad(y, leaves, st["dy"].double())) if train else y


def _exact_residual(st):
    case = st["case"]
    train = case["kind"] == "residual_grad"
    x, branch, gate, w, shift = (None if t is None else t.detach().double() for t in st["x"])
    dtype = st["x"][0].dtype
    h = x + branch if gate is None else torch.addcmul(x, branch, gate)
    p = [h.to(dtype).double(), w, shift]  # the norm's input is the stream in its type
    with torch.set_grad_enabled(train):
        p = [t.requires_grad_(train) for t in p]
        n = torch.nn.functional.layer_norm(p[0], p[0].shape[-1:], None, None, _EPS)
        y = n * p[1] + p[2] if case["form"] == "affine" else n + n * p[1] + p[2]
    if not train:
        return h, y
    dt, dw, db = torch.autograd.grad(y, p, st["dy"].double())
    dt = dt + st["dh"].double()
    if gate is None:
        return [h, y.detach(), dt, dt, dw, db]
    return [h, y.detach(), dt, dt * gate, (dt * branch).sum(1, keepdim=True), dw, db]


def exact(case, seed):
    st = prepare(case, seed)
    return {"attn": _exact_attn, "rope": _exact_rope, "residual": _exact_residual}[case["kind"].split("_")[0]](st)
