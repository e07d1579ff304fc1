"""The gated residual and the norm behind it against their definition in 64 bits."""

import math

import pytest
import torch

from train_ops_helpers import held, residual64, say

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def param(g, b, cols, form, dtype, device, level=0.3):
    if form is None:
        return None
    t = level * torch.randn(*{"shared": (cols,), "one": (1, 1, cols), "own": (b, 1, cols), "rows": (b, cols)}[form], generator=g)
    return t.to(dtype).to(device)


def wide(p, b, cols):
    return None if p is None else p.detach().double().cpu().view(-1, 1, cols)


def make(seed, b, s, cols, dtype, device):
    g = torch.Generator().manual_seed(seed)
    chan = torch.exp(0.5 * torch.randn(cols, generator=g))
    t = [torch.randn(b, s, cols, generator=g) * chan * f for f in (1.0, 0.5, 0.01, 0.01)]
    t[0] = t[0] + 0.3
    return g, [v.to(dtype).to(device) for v in t]


def check(x, branch, dh, dy, gate, p0, p1, modulated, eps=1e-6):
    from svoo_amd import norm

    b, s, cols = x.shape
    names = ("scale", "shift") if modulated else ("weight", "bias")
    gw, w, c = wide(gate, b, cols), wide(p0, b, cols), wide(p1, b, cols)
    w = torch.ones(1, 1, cols).double() if w is None else w
    w = 1 + w if modulated and p0 is not None else w
    c = torch.zeros(1, 1, cols).double() if c is None else c
    shared = [t is None or t.numel() == cols for t in (gate, p0, p1)]
    want = residual64(*(t.double().cpu() for t in (x, branch)), gw, w, c, eps, x.dtype, dh.double().cpu(), dy.double().cpu(), shared)
    leaves = [None if t is None else t.detach().requires_grad_() for t in (x, branch, gate, p0, p1)]
    h, y = norm.residual_norm(*leaves[:3], eps=eps, **dict(zip(names, leaves[3:])))
    some = [t for t in leaves if t is not None]
    grads = iter(torch.autograd.grad([h, y], some, [dh, dy]))
    grads = [None if t is None else next(grads) for t in leaves]
    held(h, want["h"], "h")
    held(y, want["y"], "y")
    for t, leaf, name in zip(grads, leaves, ("dx", "dbranch", "dgate", "dw", "dc")):
        if t is not None:
            assert t.shape == leaf.shape and t.dtype == leaf.dtype
            value, bound = want[name]
            held(t.view(value.shape), (value, bound), name)
    kw = dict(gate=gate, eps=eps, **dict(zip(names, (p0, p1))))
    with torch.no_grad():
        for a, e in zip(norm.residual_norm(x, branch, **kw), (h, y)):
            assert torch.equal(a, e)
    h2, y2, mean, rstd = norm.residual_norm_fwd(x, branch, **kw)
    assert torch.equal(h2, h) and torch.equal(y2, y)
    for a, e in zip(norm.residual_norm_bwd(dh, dy, h2, branch, mean, rstd, **kw), grads):
        assert (a is None) == (e is None) and (a is None or torch.equal(a, e))
    return h, y, grads


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [1, 7, 8, 64, 127, 128, 129, 512, 513, 999, 1536, 1537, 2048, 2049, 5120, 6144, 6145, 8192, 8193,
                                  16383, 16384])
def test_widths(gpu, cols, dtype):
    say("widths", cols, dtype)
    g, (x, branch, dh, dy) = make(cols, 2, 5, cols, dtype, gpu)
    f32 = torch.float32
    check(x, branch, dh, dy, param(g, 2, cols, "own", f32, gpu), param(g, 2, cols, "own", f32, gpu),
          param(g, 2, cols, "own", f32, gpu), True)
    check(x, branch, dh, dy, None, param(g, 2, cols, "shared", dtype, gpu), param(g, 2, cols, "shared", dtype, gpu), False)


@pytest.mark.parametrize("gate", [None, "shared", "one", "own", "rows"])
@pytest.mark.parametrize("p0,p1", [(None, None), ("shared", "own"), ("rows", "one"), ("own", None), (None, "shared")])
@pytest.mark.parametrize("modulated", [True, False])
def test_parameter_forms(gpu, gate, p0, p1, modulated):
    say("forms", gate, p0, p1, modulated)
    g, (x, branch, dh, dy) = make(3, 3, 40, 200, torch.bfloat16, gpu)
    ps = [param(g, 3, 200, f, t, gpu) for f, t in ((gate, torch.float32), (p0, torch.bfloat16), (p1, torch.float16))]
    check(x, branch, dh, dy, *ps, modulated)


@pytest.mark.parametrize("b,s,cols", [(1, 1, 1536), (1, 3000, 64), (1, 9001, 130), (2, 2500, 1536), (5, 700, 257), (300, 2, 40),
                                      (1, 1500, 5120)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows(gpu, b, s, cols, dtype):
    say("rows", b, s, cols, dtype)
    g, (x, branch, dh, dy) = make(4, b, s, cols, dtype, gpu)
    check(x, branch, dh, dy, param(g, b, cols, "own", torch.float32, gpu), param(g, b, cols, "shared", dtype, gpu),
          param(g, b, cols, "shared", dtype, gpu), False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("gate", [None, "shared", "own"])
@pytest.mark.parametrize("size", [(1, 1, 5), (2, 300, 96), (3, 50, 1999), (2, 7, 9000)])
def test_residual_alone(gpu, size, gate, dtype):
    from svoo_amd import norm

    say("alone", size, gate, dtype)
    g, (x, branch, dh, _) = make(5, *size, dtype, gpu)
    p = param(g, size[0], size[2], gate, torch.float32, gpu)
    want = residual64(x.double().cpu(), branch.double().cpu(), wide(p, size[0], size[2]), None, None, 0.0, dtype, dh.double().cpu())
    leaves = [t.detach().requires_grad_() for t in (x, branch, p) if t is not None]
    h = norm.gated_residual(*leaves)
    grads = torch.autograd.grad(h, leaves, dh)
    held(h, want["h"], "h")
    held(grads[0], want["dx"], "dx")
    held(grads[1], want["dbranch"], "dbranch")
    if p is not None:
        value, bound = want["dgate"]
        if gate == "shared":
            bound = (bound + size[0] * 2.0 ** -24 * value.abs()).sum(0, keepdim=True)
            value = value.sum(0, keepdim=True)
        held(grads[2].view(value.shape), (value, bound), "dgate")
    with torch.no_grad():
        assert torch.equal(norm.gated_residual(x, branch, p), h)


def test_gradients_of_expanded_parameters(gpu):
    """A parameter expanded over the batch has a gradient row for each entry."""
    from svoo_amd import norm

    g, (x, branch, dh, dy) = make(6, 3, 20, 64, torch.float32, gpu)
    ps = [param(g, 1, 64, "one", torch.float32, gpu) for _ in range(3)]
    leaves = [p.expand(3, 1, 64).detach().requires_grad_() for p in ps]
    h, y = norm.residual_norm(x, branch, leaves[0], scale=leaves[1], shift=leaves[2])
    got = torch.autograd.grad([h, y], leaves, [dh, dy])
    own = [p.expand(3, 1, 64).contiguous().requires_grad_() for p in ps]
    h2, y2 = norm.residual_norm(x, branch, own[0], scale=own[1], shift=own[2])
    assert torch.equal(h, h2) and torch.equal(y, y2)
    for a, b in zip(got, torch.autograd.grad([h2, y2], own, [dh, dy])):
        assert a.shape == (3, 1, 64) and torch.equal(a, b)


def test_one_of_two_gradients(gpu):
    """Only h or only y used afterwards: the other's gradient is 0."""
    from svoo_amd import norm

    g, (x, branch, dh, dy) = make(7, 2, 30, 96, torch.float32, gpu)
    gate, w, c = (param(g, 2, 96, f, torch.float32, gpu) for f in ("own", "shared", "shared"))
    zero = torch.zeros_like(dh)
    for i, (a, b) in enumerate(((dh, zero), (zero, dy))):
        leaves = [t.detach().requires_grad_() for t in (x, branch, gate, w, c)]
        out = norm.residual_norm(*leaves)
        got = torch.autograd.grad(out[i], leaves, (a, b)[i])
        h, y, mean, rstd = norm.residual_norm_fwd(x, branch, gate, w, c)
        for p, q in zip(got, norm.residual_norm_bwd(a, b, h, branch, mean, rstd, gate, w, c)):
            assert torch.equal(p, q)
    none = norm.residual_norm_bwd(None, dy, h, branch, mean, rstd, gate, w, c)
    for p, q in zip(none, norm.residual_norm_bwd(zero, dy, h, branch, mean, rstd, gate, w, c)):
        assert torch.equal(p, q)


def test_only_the_gradients_asked_for(gpu):
    from svoo_amd import norm

    g, (x, branch, dh, dy) = make(8, 2, 30, 96, torch.bfloat16, gpu)
    ps = [param(g, 2, 96, f, torch.float32, gpu) for f in ("own", "own", "shared")]
    names = dict(zip(("gate", "scale", "shift"), ps))
    h, y, mean, rstd = norm.residual_norm_fwd(x, branch, **names)
    want = norm.residual_norm_bwd(dh, dy, h, branch, mean, rstd, **names)
    for i in range(5):
        needs = [j == i for j in range(5)]
        got = norm.residual_norm_bwd(dh, dy, h, branch, mean, rstd, needs=needs, **names)
        assert all(t is None for j, t in enumerate(got) if j != i) and torch.equal(got[i], want[i])


def test_strides(gpu):
    from svoo_amd import norm

    g, (x, branch, dh, dy) = make(9, 2, 12, 64, torch.bfloat16, gpu)
    p = [param(g, 2, 64, "own", torch.float32, gpu) for _ in range(3)]
    table = torch.cat([t.view(2, 1, 64) for t in p], 1)  # modulation vectors as a block's table holds them
    views = dict(zip(("gate", "scale", "shift"), table.split(1, 1)))
    plain = dict(zip(("gate", "scale", "shift"), p))
    h, y, mean, rstd = norm.residual_norm_fwd(x, branch, **plain)
    grads = norm.residual_norm_bwd(dh, dy, h, branch, mean, rstd, **plain)
    for odd in (lambda t: t.transpose(0, 1).contiguous().transpose(0, 1), lambda t: torch.cat([t, t], 2)[..., 64:],
                lambda t: torch.stack([t, t], -1)[..., 0], lambda t: torch.cat([t, t], 1)[:, 12:],
                lambda t: torch.empty(t.numel() + 1, dtype=t.dtype, device=gpu)[1:].view(t.shape).copy_(t)):
        got = norm.residual_norm_fwd(odd(x), odd(branch), **views)
        assert all(torch.equal(a, b) for a, b in zip(got, (h, y, mean, rstd)))
        got = norm.residual_norm_bwd(odd(dh), odd(dy), odd(h), odd(branch), mean, rstd, **views)
        assert all(torch.equal(a, b) for a, b in zip(got, grads))


def test_empty(gpu):
    from svoo_amd import norm

    for shape in ((0, 5, 64), (2, 0, 64)):
        x, b = (torch.zeros(shape, device=gpu, requires_grad=True) for _ in range(2))
        gate = torch.ones(shape[0], 1, 64, device=gpu, requires_grad=True)
        w = torch.ones(64, device=gpu, requires_grad=True)
        h, y = norm.residual_norm(x, b, gate, w)
        grads = torch.autograd.grad((h + y).sum(), [x, b, gate, w])
        assert h.shape == y.shape == shape and all(not t.any() for t in grads)
        assert norm.gated_residual(x, b).shape == shape


def test_not_finite_rows_stay_apart(gpu):
    from svoo_amd import norm

    g, (x, branch, dh, dy) = make(10, 1, 20, 200, torch.bfloat16, gpu)
    clean = norm.residual_norm(x, branch)
    x[0, 3, 5], branch[0, 9, 150] = math.nan, math.inf
    h, y = norm.residual_norm(x, branch)
    assert y[0, 3].isnan().all() and y[0, 9].isnan().all()
    keep = [i for i in range(20) if i not in (3, 9)]
    assert torch.equal(h[0, keep], clean[0][0, keep]) and torch.equal(y[0, keep], clean[1][0, keep])


def test_the_same_norm_as_layer_norm(gpu):
    """y is the layer norm of h, to the bit where both hold a row alike."""
    from svoo_amd import norm

    for cols in (64, 500, 1536):
        g, (x, branch, _, _) = make(11, 2, 50, cols, torch.bfloat16, gpu)
        ps = [param(g, 2, cols, "own", torch.float32, gpu) for _ in range(3)]
        h, y = norm.residual_norm(x, branch, ps[0], scale=ps[1], shift=ps[2])
        assert torch.equal(h, norm.gated_residual(x, branch, ps[0]))
        assert torch.equal(y, norm.layer_norm(h, scale=ps[1], shift=ps[2]))


def test_captured_and_replayed(gpu):
    from svoo_amd import norm

    g, (x, branch, dh, dy) = make(12, 2, 400, 1536, torch.bfloat16, gpu)
    ps = [param(g, 2, 1536, f, torch.float32, gpu) for f in ("own", "shared", "shared")]

    def step():
        h, y, mean, rstd = norm.residual_norm_fwd(x, branch, *ps)
        return [h, y, *norm.residual_norm_bwd(dh, dy, h, branch, mean, rstd, *ps)]

    side = torch.cuda.Stream(gpu)
    side.wait_stream(torch.cuda.current_stream(gpu))
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream(gpu).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (13, 14, 15):
        for t, n in zip((x, branch, dh, dy), make(seed, 2, 400, 1536, torch.bfloat16, gpu)[1]):
            t.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step()):
            assert torch.equal(a, b)


def test_offsets_past_32_bits(gpu):
    from svoo_amd import norm

    g, (x, branch, dh, dy) = make(16, 3, 4, 96, torch.bfloat16, gpu)
    ps = [param(g, 3, 96, "own", torch.float32, gpu) for _ in range(3)]
    kw = dict(zip(("gate", "scale", "shift"), ps))
    h, y, mean, rstd = norm.residual_norm_fwd(x, branch, **kw)
    grads = norm.residual_norm_bwd(dh, dy, h, branch, mean, rstd, **kw)
    step = (1 << 31) + 24
    buffer = torch.empty(2 * step + 5000, dtype=torch.bfloat16, device=gpu)
    far = [buffer.as_strided(x.shape, (step, 96, 1), 1000 * i).copy_(t) for i, t in enumerate((x, branch, dh, dy))]
    got = norm.residual_norm_fwd(*far[:2], **kw)
    assert all(torch.equal(a, b) for a, b in zip(got, (h, y, mean, rstd)))
    for a, b in zip(norm.residual_norm_bwd(far[2], far[3], h, far[1], mean, rstd, **kw), grads):
        assert torch.equal(a, b)


def test_a_tensor_that_is_both_stream_and_branch(gpu):
    from svoo_amd import norm

    g, (x, _, dh, dy) = make(17, 2, 30, 64, torch.float32, gpu)
    leaf = x.detach().requires_grad_()
    h, y = norm.residual_norm(leaf, leaf)
    both = torch.autograd.grad([h, y], leaf, [dh, dy])[0]
    h2, _, mean, rstd = norm.residual_norm_fwd(x, x)
    dx, db = norm.residual_norm_bwd(dh, dy, h2, x, mean, rstd)[:2]
    assert torch.equal(h, h2) and torch.equal(both, dx + db)
    assert torch.equal(norm.gated_residual(x, x), 2 * x)


def test_streams(gpu):
    """Calls on other streams, two at a time, with workspaces of their own."""
    from svoo_amd import norm, rope

    sets = [make(i, 2, 500, 768, torch.bfloat16, gpu)[1] for i in (18, 19)]

    def step(x, branch, dh, dy):
        h, y, mean, rstd = norm.residual_norm_fwd(x, branch)
        x4 = x.view(2, 500, 6, 128)
        w = torch.ones(768, device=gpu)
        return [h, y, *norm.residual_norm_bwd(dh, dy, h, branch, mean, rstd)[:2],
                *rope.axis_rope_bwd(dy.view_as(x4), x4, (128,), grid=(500,), norm="row", weight=w)]

    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(gpu) for _ in sets]
    got = []
    for st, s in zip(streams, sets):
        st.wait_stream(torch.cuda.current_stream(gpu))
        with torch.cuda.stream(st):
            got.append(step(*s))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(a, b))
