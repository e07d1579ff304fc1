"""Rotary positions on several axes behind an RMS norm against their definition in 64 bits."""

import math

import pytest
import torch

from train_ops_helpers import angles64, grid_positions, held, rope64, say

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def make(seed, b, s, h, d, dtype, device, norm):
    g = torch.Generator().manual_seed(seed)
    x, dy = (torch.randn(b, s, h, d, generator=g) * torch.exp(0.5 * torch.randn(h, d, generator=g)) for _ in range(2))
    n = {"row": h * d, "head": d, "none": 0}[norm]
    w = (1 + 0.1 * torch.randn(n, generator=g)).to(dtype).to(device) if n else None
    return x.to(dtype).to(device), (0.01 * dy).to(dtype).to(device), w


def check(x, dy, w, axes, *, norm="none", interleaved=True, grid=None, start=None, positions=None, theta=10000.0, eps=1e-6):
    from svoo_amd import rope

    b, s, h, d = x.shape
    pos = grid_positions(grid, start or (0,) * len(axes), s)[None] if grid else positions.cpu().view(-1, s, len(axes))
    angle = angles64(pos, axes, theta, d)
    if grid and math.prod(grid) < s:
        angle[:, math.prod(grid):] = 0
    want = rope64(x, angle, norm, w, eps, interleaved, dy)
    kw = dict(norm=norm, weight=w, eps=eps, interleaved=interleaved, grid=grid, start=start, positions=positions, theta=theta)
    leaves = [t.detach().requires_grad_() for t in (x, w) if t is not None]
    kw["weight"] = leaves[1] if w is not None else None
    y = rope.axis_rope(leaves[0], axes, **kw)
    grads = torch.autograd.grad(y, leaves, dy)
    held(y, want["y"], "y")
    held(grads[0], want["dx"], "dx")
    if w is not None:
        held(grads[1], want["dweight"], "dweight")
    kw["weight"] = w
    with torch.no_grad():
        assert torch.equal(rope.axis_rope(x, axes, **kw), y)
    dx, dw = rope.axis_rope_bwd(dy, x, axes, **kw)
    assert torch.equal(dx, grads[0]) and (w is None or torch.equal(dw, grads[1]))
    return y, grads


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("norm", ["none", "row", "head"])
@pytest.mark.parametrize("size,axes", [((1, 1, 1, 2), (2,)), ((1, 1, 12, 128), (44, 42, 42)), ((2, 30, 3, 64), (24, 20, 20)),
                                       ((1, 7, 5, 72), (36, 36)), ((3, 11, 2, 6), (2, 2, 2)), ((1, 9, 4, 20), (8, 4, 4, 4)),
                                       ((1, 5, 2, 512), (512,)), ((2, 3, 1, 36), (20, 8)), ((1, 70, 17, 48), (16, 16, 16))])
def test_forms(gpu, size, axes, norm, interleaved, dtype):
    say("forms", size, axes, norm, interleaved, dtype)
    x, dy, w = make(sum(size), *size, dtype, gpu, norm)
    g = torch.Generator().manual_seed(1)
    pos = torch.randint(-1000, 100000, (size[0], size[1], len(axes)), generator=g, dtype=torch.int32).to(gpu)
    check(x, dy, w, axes, norm=norm, interleaved=interleaved, positions=pos)


@pytest.mark.parametrize("norm,h,d", [("row", 1, 64), ("row", 3, 512), ("row", 12, 128), ("row", 13, 128), ("row", 40, 128),
                                      ("row", 41, 128), ("row", 49, 128), ("row", 128, 128), ("row", 32, 512), ("row", 100, 40),
                                      ("head", 40, 128), ("head", 17, 160), ("none", 33, 96), ("row", 31, 264), ("head", 70, 8)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_widths(gpu, norm, h, d, dtype):
    """Every class of row widths: waves a row, heads of a wave, lanes that hold nothing."""
    say("widths", norm, h, d, dtype)
    x, dy, w = make(h + d, 1, 37, h, d, dtype, gpu, norm)
    check(x, dy, w, (d // 2 // 2 * 2, d - d // 2 // 2 * 2), norm=norm, grid=(37, 1))


@pytest.mark.parametrize("norm", ["row", "head", "none"])
def test_many_rows(gpu, norm):
    """More rows than a launch has blocks."""
    x, dy, w = make(5, 2, 9001, 2, 64, torch.bfloat16, gpu, norm)
    check(x, dy, w, (24, 20, 20), norm=norm, grid=(9, 20, 50))


@pytest.mark.parametrize("grid,start,rows", [((3, 4, 5), None, 60), ((3, 4, 5), (1000000, -7, 0), 60), ((2, 2, 2), None, 30),
                                             ((60, 1, 1), (5, 5, 5), 61), ((1, 1, 1), None, 1)])
def test_grids(gpu, grid, start, rows):
    """A clip's grid, counted from anywhere; rows behind it stay as they are (a prompt's)."""
    x, dy, w = make(6, 2, rows, 3, 128, torch.float32, gpu, "none")
    y, _ = check(x, dy, w, (44, 42, 42), grid=grid, start=start)
    assert torch.equal(y[:, math.prod(grid):], x[:, math.prod(grid):])
    x, dy, w = make(7, 1, rows, 3, 128, torch.float32, gpu, "row")
    check(x, dy, w, (44, 42, 42), grid=grid, start=start, norm="row")


@pytest.mark.parametrize("kind", [torch.int32, torch.int64, torch.float32])
def test_positions(gpu, kind):
    """Far, negative and fractional positions, shared by the batch or not, and as wide as their type."""
    x, dy, w = make(8, 3, 20, 2, 64, torch.float32, gpu, "head")
    g = torch.Generator().manual_seed(2)
    p = torch.randn(3, 20, 2, generator=g) * 3e4
    p = p.to(kind) if kind != torch.float32 else p
    if kind == torch.int32:
        p[0, 0, 0], p[0, 1, 1] = 2 ** 31 - 1, -2 ** 31
    p = p.to(gpu)
    for q in (p, p[0], p[:1]):
        check(x, dy, w, (40, 24), norm="head", positions=q)
    wide = torch.stack([p, p], -1)[..., 0]
    assert not wide.is_contiguous()
    check(x, dy, w, (40, 24), norm="head", positions=wide)


def test_thetas_and_unturned_channels(gpu):
    x, dy, w = make(9, 1, 50, 2, 64, torch.float32, gpu, "row")
    y, _ = check(x, dy, None, (16, 8), grid=(5, 10), theta=(256.0, 1e6))
    assert torch.equal(y[..., 24:], x[..., 24:])
    check(x, dy, w, (0, 64), norm="row", grid=(1, 50), theta=100.0)


def test_the_tables_of_the_dit(gpu):
    """The same angles as the DiT's tables, and the same rotation as its tensor operations."""
    from svoo_amd import dit, rope

    cfg = dit.WanDiTConfig(num_attention_heads=2)
    cos, sin = dit.rope_tables(cfg, 3, 4, 5, gpu)
    x = torch.randn(1, 60, 2, 128, generator=torch.Generator().manual_seed(3)).to(gpu)
    want = dit.apply_rope(x, cos, sin)
    got = rope.axis_rope(x, (44, 42, 42), grid=(3, 4, 5))
    # the tables are rounded to fp32, and either side rounds two products and a sum
    assert ((got - want).abs() <= 2.0 ** -22 * 2 * x.abs().amax()).all()


@pytest.mark.parametrize("norm", ["none", "row", "head"])
def test_strides(gpu, norm):
    from svoo_amd import rope

    x, dy, w = make(10, 2, 33, 4, 64, torch.bfloat16, gpu, norm)
    kw = dict(norm=norm, weight=w, grid=(3, 11))
    want, wx = rope.axis_rope(x, (32, 32), **kw), rope.axis_rope_bwd(dy, x, (32, 32), **kw)
    for odd in (lambda t: t.transpose(1, 2).contiguous().transpose(1, 2), lambda t: torch.cat([t, t], 3)[..., 64:],
                lambda t: torch.empty(t.numel() + 1, dtype=t.dtype, device=gpu)[1:].view(t.shape).copy_(t),
                lambda t: torch.stack([t, t], -1)[..., 1], lambda t: torch.cat([t, t, t], 1)[:, 33:66]):
        assert torch.equal(rope.axis_rope(odd(x), (32, 32), **kw), want)
        for a, b in zip(rope.axis_rope_bwd(odd(dy), odd(x), (32, 32), **kw), wx):
            assert b is None or torch.equal(a, b)
    flat = x[:1].expand(2, -1, -1, -1)
    assert torch.equal(rope.axis_rope(flat, (32, 32), **kw), rope.axis_rope(flat.contiguous(), (32, 32), **kw))


def test_weight_of_another_type_and_of_none(gpu):
    x, dy, _ = make(11, 2, 13, 3, 64, torch.bfloat16, gpu, "none")
    for norm, n in (("row", 192), ("head", 64)):
        check(x, dy, torch.randn(n, generator=torch.Generator().manual_seed(4)).to(gpu), (32, 32), norm=norm, grid=(1, 13))
        check(x, dy, None, (32, 32), norm=norm, grid=(1, 13))


def test_rows_of_zeros_and_not_finite_rows(gpu):
    from svoo_amd import rope

    x, dy, w = make(12, 1, 20, 2, 64, torch.float32, gpu, "row")
    x[0, 3] = 0
    check(x, dy, w, (64,), norm="row", grid=(20,))
    clean = rope.axis_rope(x, (64,), norm="row", weight=w, grid=(20,))
    x[0, 7, 1, 5] = math.nan
    y = rope.axis_rope(x, (64,), norm="row", weight=w, grid=(20,))
    assert y[0, 7].isnan().all()
    y[0, 7] = clean[0, 7]
    assert torch.equal(y, clean)


def test_empty(gpu):
    from svoo_amd import rope

    for shape in ((0, 5, 2, 64), (2, 0, 2, 64)):
        x, w = torch.zeros(shape, device=gpu, requires_grad=True), torch.ones(128, device=gpu, requires_grad=True)
        pos = torch.zeros(shape[1], 1, dtype=torch.int32, device=gpu)
        y = rope.axis_rope(x, (64,), norm="row", weight=w, positions=pos)
        dx, dw = torch.autograd.grad(y.sum(), [x, w])
        assert y.shape == shape and dx.shape == shape and not dw.any()


def test_only_the_gradients_asked_for(gpu):
    from svoo_amd import rope

    x, dy, w = make(13, 1, 50, 2, 64, torch.float32, gpu, "row")
    kw = dict(norm="row", weight=w, grid=(50,))
    dx, dw = rope.axis_rope_bwd(dy, x, (64,), **kw)
    assert torch.equal(rope.axis_rope_bwd(dy, x, (64,), needs=(True, False), **kw)[0], dx)
    got = rope.axis_rope_bwd(dy, x, (64,), needs=(False, True), **kw)
    assert got[0] is None and torch.equal(got[1], dw)
    leaf = w.detach().requires_grad_()
    assert torch.equal(torch.autograd.grad(rope.axis_rope(x, (64,), norm="row", weight=leaf, grid=(50,)), leaf, dy)[0], dw)


def test_gradients_against_differences(gpu):
    from svoo_amd import rope

    x, dy, w = make(14, 1, 6, 2, 32, torch.float32, gpu, "row")
    angle = angles64(grid_positions((2, 3), (0, 0), 6)[None], (16, 16), 10000.0, 32)
    leaves = [x.detach().requires_grad_(), w.detach().requires_grad_()]
    grads = torch.autograd.grad(rope.axis_rope(leaves[0], (16, 16), norm="row", weight=leaves[1], grid=(2, 3)), leaves, dy)
    base = [t.detach().double().cpu() for t in (x, w)]
    g = torch.Generator().manual_seed(1)
    for i in range(2):
        way = torch.randn(base[i].shape, generator=g).double()

        def loss(e):
            at = list(base)
            at[i] = at[i] + e * way
            return (rope64(at[0], angle, "row", at[1], 1e-6, True)["y"][0] * dy.double().cpu()).sum()

        slope = (loss(1e-5) - loss(-1e-5)) / 2e-5
        got = (grads[i].double().cpu() * way).sum()
        assert abs(got - slope) <= 2.0 ** -18 * (grads[i].double().cpu() * way).abs().sum() + 1e-9


def test_captured_and_replayed(gpu):
    from svoo_amd import rope

    x, dy, w = make(15, 1, 500, 5, 128, torch.bfloat16, gpu, "row")
    kw = dict(norm="row", weight=w, grid=(5, 10, 10))

    def step():
        return [rope.axis_rope(x, (44, 42, 42), **kw), *rope.axis_rope_bwd(dy, x, (44, 42, 42), **kw)]

    side = torch.cuda.Stream(gpu)
    side.wait_stream(torch.cuda.current_stream(gpu))
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream(gpu).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (16, 17, 18):
        for t, n in zip((x, dy, w), make(seed, 1, 500, 5, 128, torch.bfloat16, gpu, "row")):
            t.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step()):
            assert torch.equal(a, b)


@pytest.mark.parametrize("norm", ["row", "head", "none"])
def test_offsets_past_32_bits(gpu, norm):
    from svoo_amd import rope

    x, dy, w = make(19, 3, 5, 2, 64, torch.bfloat16, gpu, norm)
    kw = dict(norm=norm, weight=w, grid=(5,))
    want, grads = rope.axis_rope(x, (64,), **kw), rope.axis_rope_bwd(dy, x, (64,), **kw)
    step = (1 << 31) + 24
    buffer = torch.empty(2 * step + 5000, dtype=torch.bfloat16, device=gpu)
    far, far_dy = (buffer.as_strided(x.shape, (step, 128, 64, 1), at).copy_(t) for at, t in ((0, x), (2000, dy)))
    assert torch.equal(rope.axis_rope(far, (64,), **kw), want)
    for a, b in zip(rope.axis_rope_bwd(far_dy, far, (64,), **kw), grads):
        assert b is None or torch.equal(a, b)
