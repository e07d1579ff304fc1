"""Layer norm and its backward pass against their formulas in 64 bits, and as parts of programs: gradients by
differences, strided and shared tensors, streams, captured graphs."""

import pytest
import torch

from norm_fp8_helpers import U32, norm64, say, within

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32

# Every width class of the kernels (forward 16, 64 and 1024 lanes a row and one to ten chunks a lane, backward also 256 lanes
# and one to three) and both sides of its borders.
WIDTHS = [1, 7, 8, 24, 127, 128, 129, 511, 512, 520, 999, 1024, 1025, 1536, 1537, 2048, 2050, 4096, 4104, 5120, 6144, 6145,
          8192, 8193, 16384]


def _inputs(seed, gpu, batch, rows, cols, dtype, form, p_dtype=None):
    g = torch.Generator(device=gpu).manual_seed(seed)
    chan = torch.exp(0.5 * torch.randn(cols, generator=g, device=gpu))
    x = (torch.randn(batch, rows, cols, generator=g, device=gpu) * chan + 0.5).to(dtype)
    dy = (0.1 * torch.randn(batch, rows, cols, generator=g, device=gpu)).to(dtype)
    p_dtype = p_dtype or dtype
    if form == "plain":
        p = {}
    elif form == "affine":
        p = dict(weight=(1 + 0.2 * torch.randn(cols, generator=g, device=gpu)).to(p_dtype),
                 bias=(0.2 * torch.randn(cols, generator=g, device=gpu)).to(p_dtype))
    else:  # strided, as a chunk of a block's modulation
        mod = (0.3 * torch.randn(batch, 6, cols, generator=g, device=gpu)).to(p_dtype)
        p = dict(scale=mod[:, 1:2], shift=mod[:, 0:1])
    return x, dy, p


def _gain(p, cols, device):
    if "scale" in p:
        return 1 + p["scale"].double(), p["shift"].double()
    one = torch.ones(cols, dtype=torch.float64, device=device)
    return (p["weight"].double() if "weight" in p else one), (p["bias"].double() if "bias" in p else 0 * one)


def _check_forward(y, x, p, eps):
    w, b = _gain(p, x.shape[-1], x.device)
    n, _, want = norm64(x.double(), w, b, eps)
    # Sums over a row: at most 24 additions in a lane, 6 across lanes and 16 across waves, so a relative 64 U of a mean of
    # magnitudes; that moves n by 64 U of 1 (the mean) and of itself (the variance, halved).  Then four roundings.
    within(y, want, 80 * U32 * (n.abs() + 1) * w.abs() + 4 * U32 * (want.abs() + b.abs()))


def _check_backward(grads, x, dy, p, eps):
    w, b = _gain(p, x.shape[-1], x.device)
    n, rstd, _ = norm64(x.double(), w, b, eps)
    g = dy.double() * w
    n1 = n.abs() + 1  # n is known to 80 U of this
    want = rstd * (g - g.mean(-1, keepdim=True) - n * (g * n).mean(-1, keepdim=True))
    mean_gn = (g.abs() * n1).mean(-1, keepdim=True)
    within(grads[0], want, 320 * U32 * rstd * (g.abs() + n1 * mean_gn))
    if not p:
        return
    each = "scale" in p and p["scale"].shape[0] > 1
    over = (1,) if each else (0, 1)
    count = x.shape[1] * (1 if each else x.shape[0])
    d = dy.double()
    # each term to 80 U of |dy| (|n| + 1), and at most one rounding per added row
    names = ("scale", "shift") if "scale" in p else ("weight", "bias")
    for got, term, size, name in ((grads[1], d * n, d.abs() * n1, names[0]), (grads[2], d, d.abs(), names[1])):
        assert got.shape == p[name].shape and got.dtype == p[name].dtype
        shape = got.shape
        within(got, term.sum(over).reshape(shape), ((80 + count) * U32 * size.sum(over)).reshape(shape))


@pytest.mark.parametrize("cols", WIDTHS)
def test_norm_and_gradients_at_every_width(gpu, cols):
    from svoo_amd import norm

    for seed, (dtype, form) in enumerate([(BF16, "modulated"), (F16, "affine"), (F32, "plain"), (F32, "modulated")]):
        batch, rows = (2, 19) if cols > 2048 else (3, 83)
        x, dy, p = _inputs(seed, gpu, batch, rows, cols, dtype, form, F32 if dtype == BF16 else None)
        say("norm", batch, rows, cols, dtype, form)
        y, mean, rstd = norm.layer_norm_fwd(x, eps=1e-6, **p)
        _check_forward(y, x, p, 1e-6)
        grads = norm.layer_norm_bwd(dy, x, mean, rstd, eps=1e-6, **p)
        _check_backward(grads, x, dy, p, 1e-6)
        again = norm.layer_norm_bwd(dy, x, mean, rstd, eps=1e-6, **p)
        assert all(a is b or torch.equal(a, b) for a, b in zip(grads, again))  # the same bits every time
        assert torch.equal(norm.layer_norm(x, eps=1e-6, **p), y)


@pytest.mark.parametrize("rows", [1, 2, 3, 5, 16, 17, 63, 64, 65, 1000, 8191, 20000])
def test_norm_row_counts(gpu, rows):
    """One row to many: one part written directly, several joined, more rows than the grid has groups."""
    from svoo_amd import norm

    for cols, form in ((40, "affine"), (256, "modulated"), (2056, "affine")):
        if rows * cols > 1 << 23:
            continue
        x, dy, p = _inputs(rows, gpu, 1, rows, cols, BF16, form, F32)
        say("norm rows", rows, cols, form)
        y, mean, rstd = norm.layer_norm_fwd(x, **p)
        _check_forward(y, x, p, 1e-6)
        _check_backward(norm.layer_norm_bwd(dy, x, mean, rstd, **p), x, dy, p, 1e-6)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_norm_through_autograd(gpu, dtype):
    """Gradients of every leaf through autograd, with an expanded incoming gradient, and none where none is asked for."""
    from svoo_amd import norm

    x, dy, p = _inputs(5, gpu, 2, 37, 264, dtype, "modulated", F32)
    xl, sc, sh = x.clone().requires_grad_(), p["scale"].clone().requires_grad_(), p["shift"].clone().requires_grad_()
    y = norm.layer_norm(xl, scale=sc, shift=sh)
    one = torch.full((1, 1, 264), 0.25, dtype=dtype, device=gpu).expand(2, 37, 264)
    got = torch.autograd.grad(y, (xl, sc, sh), one)
    _check_backward(got, x, one, p, 1e-6)
    y = norm.layer_norm(xl, scale=p["scale"], shift=sh)
    y.backward(dy)
    _check_backward((xl.grad, *_pair(norm, x, dy, p)), x, dy, p, 1e-6)
    assert torch.equal(sh.grad, _pair(norm, x, dy, p)[1])
    with pytest.raises(RuntimeError):  # once differentiable
        y = norm.layer_norm(xl, scale=sc)
        gx, = torch.autograd.grad(y, xl, dy, create_graph=True)
        gx.sum().backward()


def _pair(norm, x, dy, p):
    _, mean, rstd = norm.layer_norm_fwd(x, **p)
    return norm.layer_norm_bwd(dy, x, mean, rstd, needs=(False, True, True), **p)[1:]


def test_norm_gradient_by_differences(gpu):
    """<dx, v> against (F(x + h v) - F(x - h v)) / 2h of F = <y, dy>, all through the kernels in fp32."""
    from svoo_amd import norm

    g = torch.Generator(device=gpu).manual_seed(3)
    x, dy, p = _inputs(8, gpu, 2, 16, 96, F32, "affine")
    x = x / x.std()
    v = torch.randn(x.shape, generator=g, device=gpu)
    _, mean, rstd = norm.layer_norm_fwd(x, **p)
    dx, dw, db = norm.layer_norm_bwd(dy, x, mean, rstd, **p)
    h = 2.0 ** -7

    def f(x, p):
        return (norm.layer_norm(x, **p).double() * dy.double()).sum()

    want = (f(x + h * v, p) - f(x - h * v, p)) / (2 * h)
    # The difference is off by h^2 / 6 of the third derivative along v, whose size is that of the first by some 10
    # (each derivative of n brings a factor of |v| / sigma, of about 1, and there are six terms), and by the outputs'
    # roundings: 80 U of <|y|, |dy|> / h.
    scale = (dx.double() * v).abs().sum()
    noise = 80 * U32 * (norm.layer_norm(x, **p).double() * dy).abs().sum() / h
    assert abs((dx.double() * v).sum() - want) <= 2 * h * h * scale + noise
    u = torch.randn(96, generator=g, device=gpu)  # linear in the parameters
    for name, grad in (("weight", dw), ("bias", db)):
        up, down = dict(p), dict(p)
        up[name], down[name] = p[name] + u, p[name] - u
        want = (f(x, up) - f(x, down)) / 2
        assert abs((grad.double() * u).sum() - want) <= 200 * U32 * (norm.layer_norm(x, **p).double().abs() + 4).sum()


def test_norm_reads_strided_tensors_in_place(gpu):
    from svoo_amd import norm

    g = torch.Generator(device=gpu).manual_seed(1)
    big = torch.randn(3, 50, 2, 700, generator=g, device=gpu).to(BF16)
    w = torch.randn(1400, generator=g, device=gpu)[::2]  # strided parameters
    for x in (big[:, :, 1, 3:603], big[:, ::2, 0, 1:-2], big[1:, 7, :, :], big.transpose(0, 1)[:, :, 1],
              big[:, :, 0, :].transpose(1, 2), big[0, 0, 0], big.transpose(0, 2)):
        say("strided", tuple(x.shape), x.stride())
        p = dict(weight=w[:x.shape[-1]]) if x.shape[-1] <= 700 else {}
        y, mean, rstd = norm.layer_norm_fwd(x, **p)
        assert y.shape == x.shape and mean.shape == x.shape[:-1]
        c = x.contiguous()
        y2, mean2, rstd2 = norm.layer_norm_fwd(c, **p)
        assert torch.equal(y, y2) and torch.equal(mean, mean2)
        dy = torch.randn(x.shape, generator=g, device=gpu).to(BF16)
        wide = torch.empty(*x.shape[:-1], x.shape[-1] + 5, dtype=BF16, device=gpu)
        wide[..., 2:-3] = dy
        for a, b in zip(norm.layer_norm_bwd(wide[..., 2:-3], x, mean, rstd, **p), norm.layer_norm_bwd(dy, c, mean2, rstd2, **p)):
            assert a is b is None or torch.equal(a, b)


def test_norm_mixed_types_and_shared_parameters(gpu):
    """Parameters of other types and shapes than x's; one shared by the batch beside one that is not."""
    from svoo_amd import norm

    x, dy, _ = _inputs(4, gpu, 3, 21, 136, BF16, "plain")
    g = torch.Generator(device=gpu).manual_seed(2)
    for sc_shape, sh_shape, dt in (((136,), (3, 136), F32), ((3, 1, 136), (1, 1, 136), F16), ((1, 136), (136,), BF16),
                                   ((3, 136), None, F32), (None, (136,), F32)):
        sc = None if sc_shape is None else (0.3 * torch.randn(sc_shape, generator=g, device=gpu)).to(dt)
        sh = None if sh_shape is None else (0.3 * torch.randn(sh_shape, generator=g, device=gpu)).to(F32)
        say("shapes", sc_shape, sh_shape, dt)
        full = lambda p: torch.zeros(1, 1, 136, device=gpu, dtype=torch.float64) if p is None else \
            p.double().reshape(-1, 1, 136)  # noqa: E731
        q = dict(scale=full(sc), shift=full(sh))
        y, mean, rstd = norm.layer_norm_fwd(x, scale=sc, shift=sh, out_dtype=F32)
        assert y.dtype == F32
        _check_forward(y, x, q, 1e-6)
        dx, dsc, dsh = norm.layer_norm_bwd(dy, x, mean, rstd, scale=sc, shift=sh)
        n, _, _ = norm64(x.double(), 1, 0, 1e-6)
        for got, p, term, size in ((dsc, sc, dy.double() * n, dy.double().abs() * (n.abs() + 1)),
                                   (dsh, sh, dy.double(), dy.double().abs())):
            if p is None:
                assert got is None
                continue
            assert got.shape == p.shape and got.dtype == p.dtype
            over = (1,) if p.numel() == 3 * 136 else (0, 1)
            # the sums of up to 63 rows, and three more additions over the batch
            within(got, term.sum(over).reshape(p.shape), (150 * U32 * size.sum(over)).reshape(p.shape))


def test_norm_extreme_rows(gpu):
    """Constant rows, a mean far above the deviations, huge and tiny values, infinities and NaN in single rows."""
    from svoo_amd import norm

    g = torch.Generator(device=gpu).manual_seed(6)
    x = torch.randn(10, 640, generator=g, device=gpu)
    x[1] = 3.0
    x[2] = 0.0
    x[3] += 1000.0
    x[4] *= 1e15
    x[5] *= 1e-15
    ok = [0, 1, 2, 3, 4, 5]
    x[6, 17], x[7, 5], x[8, 100] = float("inf"), float("nan"), float("-inf")
    y, mean, rstd = norm.layer_norm_fwd(x, eps=1e-6)
    n, _, want = norm64(x[ok].double(), 1, 0, 1e-6)
    # x - mean is exact to U of itself once the mean's own rounding is taken out; row 3's deviations come from inputs as
    # they are.  Row 5 is scaled by 1 / sqrt(eps): covered by the same bound.
    within(y[ok], want, 80 * U32 * (n.abs() + 1))
    assert torch.equal(y[1], torch.zeros_like(y[1])) and torch.equal(y[2], torch.zeros_like(y[2]))
    assert y[6:9].isnan().all() and y[9].isfinite().all()
    dy = torch.randn(x.shape, generator=g, device=gpu)
    dx = norm.layer_norm_bwd(dy, x, mean, rstd)[0]
    assert dx[6:9].isnan().all() and dx[ok].isfinite().all() and dx[9].isfinite().all()


def test_norm_of_nothing(gpu):
    from svoo_amd import norm

    w = torch.ones(64, device=gpu, requires_grad=True)
    sc = torch.ones(3, 1, 64, device=gpu, requires_grad=True)
    for shape, p in (((0, 64), dict(weight=w)), ((3, 0, 64), dict(scale=sc)), ((0, 5, 64), {})):
        x = torch.empty(shape, device=gpu, dtype=BF16, requires_grad=True)
        y = norm.layer_norm(x, **p)
        assert y.shape == shape
        leaves = [x, *p.values()]
        grads = torch.autograd.grad(y, leaves, torch.empty_like(y))
        assert grads[0].shape == shape and all((t == 0).all() and t.shape == q.shape for t, q in zip(grads[1:], leaves[1:]))


@pytest.mark.parametrize("cols", [40, 128, 300, 1000, 1536, 5120, 8200])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_norm_to_fp8_equals_the_two_steps(gpu, cols, dtype):
    from svoo_amd import fp8, norm

    x, _, p = _inputs(cols, gpu, 2, 33, cols, dtype, "modulated", F32)
    for t in (torch.float8_e4m3fn, torch.float8_e5m2):
        say("norm to", t, cols, dtype)
        q, s = norm.layer_norm_fp8(x, dtype=t, **p)
        q2, s2 = fp8.fp8_quantize_rows(norm.layer_norm(x, **p), dtype=t)
        assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8)) and torch.equal(s.view(torch.uint8), s2.view(torch.uint8))


def test_norm_on_other_streams_and_in_a_graph(gpu):
    """The current stream's work, on a side stream and as a captured forward and backward pass replayed with changed
    inputs and eager work between the replays."""
    from svoo_amd import norm

    x, dy, p = _inputs(9, gpu, 2, 600, 1536, BF16, "modulated", F32)
    x2, dy2, _ = _inputs(10, gpu, 2, 600, 1536, BF16, "modulated", F32)

    def step(x, dy):
        y, mean, rstd = norm.layer_norm_fwd(x, **p)
        return (y, *norm.layer_norm_bwd(dy, x, mean, rstd, **p))

    want, want2 = step(x, dy), step(x2, dy2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(x, dy)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    xs, dys = x.clone(), dy.clone()
    with torch.cuda.stream(side):
        step(xs, dys)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(xs, dys)
    for i in range(4):
        a, b, ref = ((x, dy, want), (x2, dy2, want2))[i % 2]
        xs.copy_(a)
        dys.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(u, v) for u, v in zip(out, ref)), i
        assert all(torch.equal(u, v) for u, v in zip(step(x2, dy2), want2))


@pytest.mark.parametrize("cols", [40, 128, 500, 999, 1536, 1543, 2048, 4096, 5000, 8200, 16384])
def test_norm_gradients_of_other_types(gpu, cols):
    """An incoming gradient of another type than x's: y was asked for in that type."""
    from svoo_amd import norm

    for seed, (dtype, dy_dtype) in enumerate([(BF16, F32), (BF16, F16), (F16, BF16), (F16, F32), (F32, BF16), (F32, F16)]):
        x, dy, p = _inputs(seed, gpu, 2, 21, cols, dtype, "modulated" if seed % 2 else "affine", F32)
        dy = dy.to(dy_dtype)
        say("norm, dy of another type", cols, dtype, dy_dtype)
        y, mean, rstd = norm.layer_norm_fwd(x, out_dtype=dy_dtype, **p)
        assert y.dtype == dy_dtype
        _check_forward(y, x, p, 1e-6)
        _check_backward(norm.layer_norm_bwd(dy, x, mean, rstd, **p), x, dy, p, 1e-6)
