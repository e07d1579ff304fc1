"""8-bit blocks, their product and the linear layer on them against their definitions in 64 bits."""

import pytest
import torch

from norm_fp8_helpers import (HALF, block_exponents64, fp8_values64, gelu64, product_bound, say, spread, within)

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
E4, E5 = torch.float8_e4m3fn, torch.float8_e5m2
BYTES = torch.uint8


def _wide(seed, gpu, m, k, dtype):
    """Values over many binades, zeros, ties and a block of nothing among them."""
    g = torch.Generator(device=gpu).manual_seed(seed)
    x = torch.randn(m, k, generator=g, device=gpu)
    x *= torch.exp2(torch.randint(-12, 4, (m, k), generator=g, device=gpu).float())
    x[torch.rand(m, k, generator=g, device=gpu) < 0.05] = 0
    tie = torch.rand(m, k, generator=g, device=gpu) < 0.2  # five digits: halfway between four, two steps from three
    x = torch.where(tie, torch.round(x * 8 + 0.5) / 8 + 1.0625, x)
    x[:, 128:256] *= (torch.rand(m, 1, generator=g, device=gpu) < 0.7)
    return x.to(dtype)


def _values(q, s, tall, m, k):
    """What stored values and scale bytes stand for, and the exponents, as float64."""
    e = s.view(BYTES).double() - 127
    return q.double()[:, :k] * spread(e, tall, m, k), e


def _same(got, want):
    assert torch.equal(torch.nan_to_num(got, nan=1e300), torch.nan_to_num(want, nan=1e300))


@pytest.mark.parametrize("m,k", [(1, 1), (1, 128), (3, 129), (7, 40), (128, 128), (130, 385), (257, 1000), (1000, 136)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_quantising_is_exact(gpu, m, k, dtype):
    from svoo_amd import fp8

    x = _wide(m * k, gpu, m, k, dtype)
    for t in (E4, E5):
        say("quantise", m, k, dtype, t)
        for make, tall, src in ((fp8.fp8_quantize_rows, 1, x), (fp8.fp8_quantize_blocks, 128, x)):
            q, s = make(src, dtype=t)
            want, e = fp8_values64(src.double(), tall, t)
            got, ge = _values(q, s, tall, m, k)
            assert q.dtype == t and torch.equal(ge, e)
            _same(got, want)
            assert (q.view(BYTES)[:, k:] == 0).all()
            back = fp8.fp8_dequantize(q, s, cols=k, out_dtype=F32)
            _same(back.double(), want.float().double())
            assert torch.equal(fp8.fp8_dequantize(q, s, cols=k, out_dtype=dtype), want.to(dtype))
        q, s, qt, st = fp8.fp8_quantize_both(x, dtype=t)
        q1, s1 = fp8.fp8_quantize_rows(x, dtype=t)
        q2, s2 = fp8.fp8_quantize_rows(x.t().contiguous(), dtype=t)
        for a, b in ((q, q1), (s, s1), (qt, q2), (st, s2)):
            assert torch.equal(a.view(BYTES), b.view(BYTES))
        q, s, qt, st = fp8.fp8_quantize_blocks(x, dtype=t, transposed=True)
        q1, s1 = fp8.fp8_quantize_blocks(x.t().contiguous(), dtype=t)
        assert torch.equal(qt.view(BYTES), q1.view(BYTES)) and torch.equal(st.view(BYTES), s1.view(BYTES))


def test_quantising_extreme_values(gpu):
    """The ends of fp32's range, subnormals, amax at and next to a scale's border, infinities and NaN."""
    from svoo_amd import fp8

    x = torch.zeros(12, 128, device=gpu)
    x[:, 3] = 1.0
    x[1] = 3e38
    x[2] = 1e-44
    x[3, 0], x[4, 0] = 448.0, torch.nextafter(torch.tensor(448.0), torch.tensor(500.0))
    x[5, 0], x[6, 0] = 57344.0, torch.nextafter(torch.tensor(57344.0), torch.tensor(6e4))
    x[7, 0], x[7, 1], x[7, 2] = float("inf"), float("-inf"), float("nan")
    x[8] = -0.0
    x[9] = 2.0 ** -126
    x[10, 0], x[10, 1] = 2.0 ** 127, 2.0 ** -140
    x[11, 0] = 2.0 ** -119 * 1.75  # the last scale before the clamp
    for t in (E4, E5):
        q, s = fp8.fp8_quantize_rows(x, dtype=t)
        e = block_exponents64(x.double(), 1, t)
        assert torch.equal(s.view(BYTES).double() - 127, e)
        want, _ = fp8_values64(x.double(), 1, t)
        if t == E4:
            want[7, :2] = float("nan")
        got, _ = _values(q, s, 1, 12, 128)
        _same(got, want)
        _same(fp8.fp8_dequantize(q, s, out_dtype=F32).double(), want)


def test_quantising_strided_tensors(gpu):
    from svoo_amd import fp8

    base = _wide(3, gpu, 300, 515, BF16)
    for x in (base[:, 3:], base[::3, 1:402], base.t(), base[:, ::2], base.view(3, 100, 515)[:, 1::2, 5:]):
        say("strided", tuple(x.shape), x.stride())
        c = x.contiguous()
        for a, b in zip(fp8.fp8_quantize_rows(x), fp8.fp8_quantize_rows(c)):
            assert torch.equal(a.view(BYTES), b.view(BYTES))
        if x.dim() == 2:
            for a, b in zip(fp8.fp8_quantize_both(x), fp8.fp8_quantize_both(c)):
                assert torch.equal(a.view(BYTES), b.view(BYTES))


# ------------------------------------------------------------------------------------------------ the product
def _whole(seed, gpu, m, n, k, b_tall, a_type=E4):
    """Operands of small whole numbers with a power of two per block: every product and sum is exact."""
    g = torch.Generator(device=gpu).manual_seed(seed)
    kp, kb = -(-k // 128) * 128, -(-k // 128)
    a = torch.randint(-2, 3, (m, kp), generator=g, device=gpu).float()
    b = torch.randint(-2, 3, (n, kp), generator=g, device=gpu).float()
    a[:, k:] = 0
    b[:, k:] = 0
    ea = torch.randint(-2, 2, (m, kb), generator=g, device=gpu)
    eb = torch.randint(-1, 2, (-(-n // b_tall), kb), generator=g, device=gpu)
    scales = [(e + 127).to(BYTES).view(torch.float8_e8m0fnu) for e in (ea, eb)]
    va = a.double() * spread(ea.double(), 1, m, kp)
    vb = b.double() * spread(eb.double(), b_tall, n, kp)
    return a.to(a_type), scales[0], b.to(E4), scales[1], va, vb


SHAPES = [(1, 1, 128), (1, 9216, 1536), (1, 333, 200), (2, 130, 4096), (5, 64, 384), (15, 257, 640), (16, 1000, 1280),
          (17, 96, 128), (31, 40, 2048), (33, 513, 896), (64, 64, 128), (65, 200, 300), (100, 1536, 512), (128, 128, 8960),
          (129, 129, 129), (200, 777, 256), (255, 300, 1000), (256, 256, 256), (257, 511, 384), (512, 1536, 1024),
          (513, 1025, 640), (1000, 1000, 1000), (1013, 333, 2000), (2048, 512, 128), (3000, 2000, 500), (4100, 1030, 300),
          (8200, 264, 136), (333, 1000, 33000),
          # enough tiles for the 256 x 256 kernel: edges in both directions, odd columns, one to many stages and shares
          (16300, 4224, 300), (9000, 9007, 128), (5120, 5000, 1100), (7777, 5121, 640), (1500, 1290, 20100)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product_of_whole_numbers_is_exact(gpu, m, n, k):
    """Sums of products of at most 4 2^4 over up to 33000 positions stay below 2^24 quarters of 1/2: exact in fp32, and
    in a group of eight products nothing lies 13 bits below the largest.  So the result is the rounded exact one."""
    from svoo_amd import fp8

    for tall, a_type, out in ((128, E4, F32), (128, E4, F16), (1, E5, BF16), (1, E4, F32), (128, E5, BF16)):
        qa, sa, qb, sb, va, vb = _whole(m + n + k, gpu, m, n, k, tall, a_type)
        say("whole", m, n, k, tall, a_type, out)
        c = fp8.fp8_matmul(qa, sa, qb, sb, out_dtype=out)
        want = va @ vb.t()
        assert c.shape == (m, n) and torch.equal(c, want.to(out))


@pytest.mark.parametrize("m,n,k", [(3, 77, 256), (300, 129, 200), (513, 1025, 640), (512, 1536, 4096), (9000, 9007, 128),
                                   (5120, 5000, 1100), (7777, 5121, 640), (1500, 1290, 20100)])
def test_product_with_a_bias_is_exact(gpu, m, n, k):
    """The bias, a whole number below 8, adds to the sums above without a rounding either: every column gets its own."""
    from svoo_amd import fp8

    for i, (bias_type, out) in enumerate([(BF16, BF16), (F16, F32), (F32, F16), (F32, F32)]):
        qa, sa, qb, sb, va, vb = _whole(m + n + k + i, gpu, m, n, k, (1, 128)[i % 2], E4)
        bias = torch.randint(-8, 9, (n,), device=gpu, generator=torch.Generator(device=gpu).manual_seed(i)).to(bias_type)
        say("whole, bias", m, n, k, bias_type, out)
        c = fp8.fp8_matmul(qa, sa, qb, sb, bias, out_dtype=out)
        assert torch.equal(c, (va @ vb.t() + bias.double()).to(out))


@pytest.mark.parametrize("m,n,k", [(1, 700, 1000), (40, 300, 520), (300, 500, 1000), (1000, 2000, 3000)])
@pytest.mark.parametrize("out", [BF16, F16, F32])
def test_product_of_random_matrices(gpu, m, n, k, out):
    from svoo_amd import fp8

    g = torch.Generator(device=gpu).manual_seed(m + n)
    x = torch.randn(m, k, generator=g, device=gpu) * torch.exp(torch.randn(k, generator=g, device=gpu))
    w = torch.randn(n, k, generator=g, device=gpu) / k ** 0.5
    bias = torch.randn(n, generator=g, device=gpu).to(out)
    for a_type in (E4, E5):
        qa, sa = fp8.fp8_quantize_rows(x, dtype=a_type)
        qb, sb = fp8.fp8_quantize_blocks(w)
        va, vb = fp8_values64(x.double(), 1, a_type)[0], fp8_values64(w.double(), 128, E4)[0]
        bound = product_bound(va, vb, out == F32)
        want = va @ vb.t()
        say("random", m, n, k, out, a_type)
        c = fp8.fp8_matmul(qa, sa, qb, sb, out_dtype=out)
        within(c, want, bound)
        # The cut is either way: of random sums the error's size is under 2^-13, besides the rounding
        rel = (c.double() - want).norm() / want.norm()
        assert rel <= HALF[out] + (2.0 ** -13 if out != F32 else 2.0 ** -20), rel
        want = want + bias.double()
        b1 = bound + 2.0 ** -23 * (want.abs() + bound)
        within(fp8.fp8_matmul(qa, sa, qb, sb, bias, out_dtype=out), want, b1)
        # |gelu'| <= 1.13; its own evaluation: exp and a division to a few units, the argument to 4 U of its size (< 2 y^3)
        b2 = 1.13 * b1 + 2.0 ** -22 * (4 + 2 * want.abs() ** 3).clamp(max=200) * want.abs()
        within(fp8.fp8_matmul(qa, sa, qb, sb, bias, "gelu_tanh", out), gelu64(want), b2)


def test_product_operand_views_and_leading_dimensions(gpu):
    from svoo_amd import fp8

    qa, sa, qb, sb, va, vb = _whole(1, gpu, 60, 200, 512, 1)
    want = (va @ vb.t()).float()
    wide = torch.zeros(60, 700, dtype=BYTES, device=gpu)
    for off in (16, 3):  # rows at 16-byte addresses or not (copied)
        wide[:, off:off + 512] = qa.view(BYTES)
        ws = torch.zeros(60, 9, dtype=BYTES, device=gpu)
        ws[:, 2:6] = sa.view(BYTES)
        got = fp8.fp8_matmul(wide.view(E4)[:, off:off + 512], ws.view(torch.float8_e8m0fnu)[:, 2:6], qb, sb, out_dtype=F32)
        assert torch.equal(got, want)
    got = fp8.fp8_matmul(qa.view(3, 4, 5, 512), sa.view(3, 4, 5, 4), qb, sb, out_dtype=F32)
    assert got.shape == (3, 4, 5, 200) and torch.equal(got.view(60, 200), want)
    part = fp8.fp8_matmul(qa[::2], sa[::2], qb[5:150], sb[5:150], out_dtype=F32)
    assert torch.equal(part, want[::2, 5:150])
    assert fp8.fp8_matmul(qa[:0], sa[:0], qb, sb).shape == (0, 200)
    assert fp8.fp8_matmul(qa, sa, qb[:0], sb[:0]).shape == (60, 0)


def test_product_rows_do_not_touch_each_other(gpu):
    """NaN in one row of either operand, or in a scale, stays in that row or column."""
    from svoo_amd import fp8

    for m, n in ((40, 300), (600, 700)):
        qa, sa, qb, sb, va, vb = _whole(2, gpu, m, n, 384, 1)
        for out in (F32, BF16):
            clean = fp8.fp8_matmul(qa, sa, qb, sb, out_dtype=out)
            a, b, s = qa.clone(), qb.clone(), sa.clone()
            a.view(BYTES)[7, 200] = 0x7F
            b.view(BYTES)[11, 3] = 0xFF
            s.view(BYTES)[20, 1] = 255
            c = fp8.fp8_matmul(a, s, b, sb, out_dtype=out)
            bad = torch.zeros(m, n, dtype=torch.bool, device=gpu)
            bad[7], bad[20], bad[:, 11] = True, True, True
            assert c[bad].isnan().all() and torch.equal(c[~bad], clean[~bad])


# ------------------------------------------------------------------------------------------------ the linear layer
@pytest.mark.parametrize("lead,k,n", [((1,), 64, 48), ((3, 7), 200, 136), ((130,), 128, 256), ((2, 150), 333, 1000),
                                      ((1013,), 1000, 333), ((700,), 1536, 640)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_linear_and_its_gradients(gpu, lead, k, n, dtype):
    from svoo_amd import fp8

    g = torch.Generator(device=gpu).manual_seed(k + n)
    x = torch.randn(*lead, k, generator=g, device=gpu).to(dtype)
    w = (torch.randn(n, k, generator=g, device=gpu) / k ** 0.5).to(dtype)
    b = torch.randn(n, generator=g, device=gpu).to(dtype)
    dy = (torch.randn(*lead, n, generator=g, device=gpu) * torch.exp(torch.randn(n, generator=g, device=gpu))).to(dtype)
    x2, dy2 = x.reshape(-1, k).double(), dy.reshape(-1, n).double()
    m = x2.shape[0]
    wide = dtype == F32
    for t in (E4, E5):
        say("linear", lead, k, n, dtype, t)
        leaves = [v.clone().requires_grad_() for v in (x, w, b)]
        y = fp8.fp8_linear(*leaves, grad_dtype=t)
        dx, dw, db = torch.autograd.grad(y, leaves, dy)
        vx, vw = fp8_values64(x2, 1, E4)[0], fp8_values64(w.double(), 128, E4)[0]
        bound = product_bound(vx, vw, wide)
        want = vx @ vw.t() + b.double()
        within(y.reshape(m, n), want, bound + 2.0 ** -23 * (want.abs() + bound))
        vd = fp8_values64(dy2, 1, t)[0]
        within(dx.reshape(m, k), vd @ vw, product_bound(vd, vw.t().contiguous(), wide))
        vdt, vxt = fp8_values64(dy2.t().contiguous(), 1, t)[0], fp8_values64(x2.t().contiguous(), 1, E4)[0]
        within(dw, vdt @ vxt.t(), product_bound(vdt, vxt, wide))
        within(db, dy2.sum(0), (m + 8) * 2.0 ** -24 * dy2.abs().sum(0))
        assert y.dtype == dx.dtype == dw.dtype == db.dtype == dtype and dx.shape == x.shape
        # only what is asked for, and the same bits
        y1 = fp8.fp8_linear(x, leaves[1], None, grad_dtype=t)
        dw1, = torch.autograd.grad(y1, leaves[1], dy)
        y2 = fp8.fp8_linear(leaves[0], w, b, grad_dtype=t)
        dx1, = torch.autograd.grad(y2, leaves[0], dy)
        assert torch.equal(dw1, dw) and torch.equal(dx1, dx) and torch.equal(y2, y)
        assert torch.equal(fp8.fp8_linear(x, w, b), y)


def test_linear_gradient_by_differences(gpu):
    """On whole numbers quantising changes nothing, so the layer is linear and its gradients are its differences."""
    from svoo_amd import fp8

    g = torch.Generator(device=gpu).manual_seed(9)
    ints = lambda *s: torch.randint(-2, 3, s, generator=g, device=gpu).float()  # noqa: E731
    x, w, b, dy, vx, vw, vb = ints(70, 140), ints(90, 140), ints(90), ints(70, 90), ints(70, 140), ints(90, 140), ints(90)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(fp8.fp8_linear(*leaves), leaves, dy)

    def f(x, w, b):
        return (fp8.fp8_linear(x, w, b).double() * dy.double()).sum()

    for i, v in enumerate((vx, vw, vb)):
        up, down = [x, w, b], [x, w, b]
        up[i], down[i] = up[i] + v, down[i] - v
        assert (grads[i].double() * v).sum() == (f(*up) - f(*down)) / 2


def test_linear_of_no_rows(gpu):
    from svoo_amd import fp8

    x = torch.empty(0, 3, 64, device=gpu, dtype=BF16, requires_grad=True)
    w, b = (torch.ones(s, device=gpu, dtype=BF16, requires_grad=True) for s in ((40, 64), (40,)))
    y = fp8.fp8_linear(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
    assert y.shape == (0, 3, 40) and dx.shape == x.shape and (dw == 0).all() and (db == 0).all()


def test_linear_training_step_in_a_graph(gpu):
    """Forward and backward captured with leaves made inside, replayed on changed inputs between eager steps."""
    from svoo_amd import fp8

    g = torch.Generator(device=gpu).manual_seed(4)
    data = [[torch.randn(s, generator=g, device=gpu).to(BF16) for s in ((520, 384), (300, 384), (300,), (520, 300))]
            for _ in range(2)]

    def step(x, w, b, dy):
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        y = fp8.fp8_linear(*leaves)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    want = [step(*d) for d in data]
    held = [t.clone() for t in data[0]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*held)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*held)
    for i in range(4):
        for h, t in zip(held, data[i % 2]):
            h.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want[i % 2])), i
        assert all(torch.equal(a, b) for a, b in zip(step(*data[1]), want[1]))


def test_linear_module_for_inference(gpu):
    from svoo_amd import fp8

    torch.manual_seed(0)
    lin = torch.nn.Linear(200, 333, device=gpu, dtype=BF16)
    mod = fp8.Fp8Linear.from_linear(lin)
    x = torch.randn(2, 9, 200, device=gpu, dtype=BF16)
    with torch.no_grad():
        y = mod(x)
        q, s = fp8.fp8_quantize_rows(x)
        assert torch.equal(y, mod.forward_quantized(q, s)) and torch.equal(y, fp8.fp8_linear(x, lin.weight, lin.bias))
        moved = fp8.Fp8Linear.from_linear(lin).to(torch.float16)  # the bytes stay bytes
        assert moved.weight_q.dtype == BYTES and moved.bias.dtype == F16
        assert moved(x).dtype == BF16
    again = fp8.Fp8Linear(torch.zeros(333, 200, device=gpu), torch.zeros(333, device=gpu, dtype=BF16))
    again.load_state_dict(mod.state_dict())
    with torch.no_grad():
        assert torch.equal(again(x), y)
    with pytest.raises(RuntimeError, match="no backward"):
        mod(x.requires_grad_())


def test_norm_product_gelu_product_chain(gpu):
    """The feed-forward half of a DiT block from its parts, on two streams at once, against the same in 64 bits."""
    from svoo_amd import fp8, norm

    g = torch.Generator(device=gpu).manual_seed(12)
    x = torch.randn(2, 150, 256, generator=g, device=gpu).to(BF16)
    mod = 0.3 * torch.randn(2, 6, 256, generator=g, device=gpu)
    w1 = (torch.randn(700, 256, generator=g, device=gpu) / 16).to(BF16)
    w2 = (torch.randn(256, 700, generator=g, device=gpu) / 26).to(BF16)
    b1, b2 = (0.1 * torch.randn(n, generator=g, device=gpu).to(BF16) for n in (700, 256))
    l1, l2 = fp8.Fp8Linear(w1, b1, "gelu_tanh"), fp8.Fp8Linear(w2, b2)

    def ffn():
        q, s = norm.layer_norm_fp8(x, scale=mod[:, 4:5], shift=mod[:, 3:4])
        return l2(l1.forward_quantized(q, s))

    with torch.no_grad():
        y = ffn()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            ys = [ffn() for _ in range(3)]
        yc = [ffn() for _ in range(3)]
        torch.cuda.synchronize()
    assert all(torch.equal(y, t) for t in ys + yc)
    xd = x.double()
    n = (xd - xd.mean(-1, keepdim=True)) / (xd.var(-1, correction=0, keepdim=True) + 1e-6).sqrt()
    h = (n * (1 + mod[:, 4:5].double()) + mod[:, 3:4].double()).to(BF16).double().view(300, 256)
    h = fp8_values64(h, 1, E4)[0] @ fp8_values64(w1.double(), 128, E4)[0].t() + b1.double()
    h = gelu64(h).to(BF16).double()
    want = fp8_values64(h, 1, E4)[0] @ fp8_values64(w2.double(), 128, E4)[0].t() + b2.double()
    # An intermediate that rounds the other way moves by one bf16 step, then perhaps by one e4m3 step (2^-3 of it), for
    # few of the values (one in 2^6 lies close enough to a border): relative to the result, far below 2^-3 2^-3 = 2^-6
    rel = (y.double().view(300, 256) - want).norm() / want.norm()
    assert rel <= 2.0 ** -6, rel
