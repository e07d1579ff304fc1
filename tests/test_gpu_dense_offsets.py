"""Norms and 8-bit operators on tensors past 2^31 elements or 2^32 bytes, at addresses of any alignment, and with operands of
different types."""

import pytest
import torch

from norm_fp8_helpers import fp8_values64, product_bound, say, spread, within

pytestmark = pytest.mark.gpu

E4, E5, E8 = torch.float8_e4m3fn, torch.float8_e5m2, torch.float8_e8m0fnu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
BYTES = torch.uint8


def _random(rows, cols, gpu, dtype=BF16):
    x = torch.empty(rows, cols, dtype=dtype, device=gpu)
    g = torch.Generator(device=gpu).manual_seed(rows)
    for part in x.split(1 << 15):
        part.copy_(torch.randn(part.shape, generator=g, device=gpu))
    return x


def _ends(rows):
    return slice(0, 70), slice(rows // 2, rows // 2 + 70), slice(rows - 70, rows)


def test_norm_past_2_31_elements(gpu):
    """Rows do not depend on each other: the first, middle and last ones as in a call of their own."""
    from svoo_amd import norm

    rows, cols = 270001, 8192  # 2.2e9 elements, 4.4 GB
    x = _random(rows, cols, gpu)
    w = torch.linspace(0.5, 1.5, cols, device=gpu)
    say("norm", rows, cols)
    y, mean, rstd = norm.layer_norm_fwd(x, w, w)
    q, s = norm.layer_norm_fp8(x, w, w)
    dx, dw, db = norm.layer_norm_bwd(y, x, mean, rstd, w, w)
    for at in _ends(rows):
        y1, mean1, rstd1 = norm.layer_norm_fwd(x[at], w, w)
        q1, s1 = norm.layer_norm_fp8(x[at], w, w)
        assert torch.equal(y[at], y1) and torch.equal(mean[at], mean1) and torch.equal(rstd[at], rstd1)
        assert torch.equal(q[at].view(BYTES), q1.view(BYTES)) and torch.equal(s[at].view(BYTES), s1.view(BYTES))
        assert torch.equal(dx[at], norm.layer_norm_bwd(y1, x[at], mean1, rstd1, w, w)[0])
    want = sum(part.double().sum(0) for part in y.split(4096))
    size = sum(part.double().abs().sum(0) for part in y.split(4096))
    # fp32 sums of 270001 rows: one rounding each of at most the partial sums' size
    within(db, want, rows * 2.0 ** -24 * size)


def test_quantisers_past_2_31_elements(gpu):
    from svoo_amd import fp8

    rows, cols = 270001, 8192
    x = _random(rows, cols, gpu)
    say("quantise", rows, cols)
    q, s, qt, st = fp8.fp8_quantize_both(x)
    q2, s2 = fp8.fp8_quantize_rows(x)
    for a, b in ((q, q2), (s, s2)):
        assert all(torch.equal(u.view(BYTES), v.view(BYTES)) for u, v in zip(a.split(1 << 15), b.split(1 << 15)))
    back = fp8.fp8_dequantize(q, s)
    for at in _ends(rows):
        q1, s1 = fp8.fp8_quantize_rows(x[at])
        assert torch.equal(q[at].view(BYTES), q1.view(BYTES)) and torch.equal(s[at].view(BYTES), s1.view(BYTES))
        assert torch.equal(back[at], fp8.fp8_dequantize(q1, s1))
    for c in (0, cols // 2, cols - 1):  # turned rows, each of more than 2^18 elements
        q1, s1 = fp8.fp8_quantize_rows(x[:, c].contiguous()[None])
        assert torch.equal(qt[c].view(BYTES), q1[0].view(BYTES)) and torch.equal(st[c].view(BYTES), s1[0].view(BYTES))


@pytest.mark.parametrize("m,n,k", [(600011, 4100, 128), (600011, 136, 8192), (70, 4100, 128)])
def test_product_past_2_31_elements(gpu, m, n, k):
    """More than 2^31 results, an operand of more than 2^32 bytes: whole numbers, so every row is exact."""
    from svoo_amd import fp8

    g = torch.Generator(device=gpu).manual_seed(n)
    b = torch.randint(-2, 3, (n, k), generator=g, device=gpu).float()
    a = torch.empty(m, k, dtype=E4, device=gpu)
    for part in a.split(1 << 16):
        part.copy_(torch.randint(-2, 3, part.shape, generator=g, device=gpu).float())
    ones = lambda rows: torch.full((k // 128, rows), 127, dtype=BYTES, device=gpu).view(E8).t()  # noqa: E731
    say("product", m, n, k)
    c = fp8.fp8_matmul(a, ones(m), b.to(E4), ones(n))
    for at in (*_ends(m), slice(m - 5000 if m > 5000 else 0, m)):
        assert torch.equal(c[at], (a[at].double() @ b.double().t()).to(BF16))


@pytest.mark.parametrize("m,n", [(5, 200), (300, 333), (9000, 4101)])
@pytest.mark.parametrize("out", [BF16, F32])
def test_product_at_any_address(gpu, m, n, out):
    """Scales and a bias that start at odd addresses, as slices of longer ones."""
    from svoo_amd import fp8

    g = torch.Generator(device=gpu).manual_seed(m)
    k, kb = 384, 3
    ints = lambda *s: torch.randint(-2, 3, s, generator=g, device=gpu)  # noqa: E731
    a, b = ints(m, k).float(), ints(n, k).float()
    for off in (1, 2, 3):
        ea, eb = (torch.randint(-1, 2, (rows + 7, kb), generator=g, device=gpu) for rows in (m, n))
        sa, sb = ((e + 127).to(BYTES).t().contiguous().t().view(E8)[off:][:rows] for e, rows in ((ea, m), (eb, n)))
        assert sa.stride(0) == 1 and sa.data_ptr() % 4 == off % 4
        va = a.double() * spread(ea[off:][:m].double(), 1, m, k)
        vb = b.double() * spread(eb[off:][:n].double(), 1, n, k)
        for bias_type in (BF16, F32):
            bias = ints(n + 9).to(bias_type)[off:][:n]
            say("addresses", m, n, out, off, bias_type)
            c = fp8.fp8_matmul(a.to(E4), sa, b.to(E4), sb, bias, out_dtype=out)
            assert torch.equal(c, (va @ vb.t() + bias.double()).to(out))


def test_linear_of_mixed_types(gpu):
    """x, weight, bias and the incoming gradient each in a type of their own: results in x's, the weight's and the bias's."""
    from svoo_amd import fp8

    g = torch.Generator(device=gpu).manual_seed(3)
    m, n, k = 300, 200, 264
    for tx, tw, tb in ((BF16, F32, F16), (F16, BF16, F32), (F32, F16, BF16)):
        x = torch.randn(m, k, generator=g, device=gpu).to(tx).requires_grad_()
        w = (torch.randn(n, k, generator=g, device=gpu) / 16).to(tw).requires_grad_()
        b = torch.randn(n, generator=g, device=gpu).to(tb).requires_grad_()
        dy = torch.randn(m, n, generator=g, device=gpu).to(tx)
        say("mixed", tx, tw, tb)
        y = fp8.fp8_linear(x, w, b)
        dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
        assert (y.dtype, dx.dtype, dw.dtype, db.dtype) == (tx, tx, tw, tb)
        x2, w2, d2 = x.detach().double(), w.detach().double(), dy.double()
        vx, vw = fp8_values64(x2, 1, E4)[0], fp8_values64(w2, 128, E4)[0]
        want, bound = vx @ vw.t() + b.detach().double(), product_bound(vx, vw, tx == F32)
        within(y, want, bound + 2.0 ** -23 * (want.abs() + bound))
        vd = fp8_values64(d2, 1, E4)[0]
        within(dx, vd @ vw, product_bound(vd, vw.t().contiguous(), tx == F32))
        vdt, vxt = fp8_values64(d2.t().contiguous(), 1, E4)[0], fp8_values64(x2.t().contiguous(), 1, E4)[0]
        within(dw, vdt @ vxt.t(), product_bound(vdt, vxt, tw == F32))
        within(db, d2.sum(0), (m + 8) * 2.0 ** -24 * d2.abs().sum(0))


@pytest.mark.parametrize("m,n,k", [(300, 1, 128), (65, 5, 20000), (5000, 3, 640), (70001, 1, 1100), (40000, 7, 300), (64, 2, 9000),
                                   (100000, 130, 128), (130, 100003, 128), (256, 50000, 256)])
def test_product_of_narrow_and_long_matrices(gpu, m, n, k):
    """Whole numbers with a scale per row and block, so exact: one column to many, one row of tiles or one column of them."""
    from svoo_amd import fp8

    g = torch.Generator(device=gpu).manual_seed(m + n)
    kb = -(-k // 128)
    a, b = (torch.zeros(rows, kb * 128, device=gpu) for rows in (m, n))
    for t in (a, b):
        t[:, :k] = torch.randint(-2, 3, (t.shape[0], k), generator=g, device=gpu).float()
    ea, eb = (torch.randint(-1, 2, (rows, kb), generator=g, device=gpu) for rows in (m, n))
    sa, sb = ((e + 127).to(BYTES).t().contiguous().t().view(E8) for e in (ea, eb))
    bias = torch.randint(-8, 9, (n,), generator=g, device=gpu).float()
    va, vb = a.double() * spread(ea.double(), 1, *a.shape), b.double() * spread(eb.double(), 1, *b.shape)
    want = va @ vb.t() + bias.double()
    for out in (BF16, F32):
        say("narrow", m, n, k, out)
        assert torch.equal(fp8.fp8_matmul(a.to(E4), sa, b.to(E4), sb, bias, out_dtype=out), want.to(out))


def test_operands_with_leading_dimensions_in_another_order(gpu):
    """Values and scales whose leading dimensions are transposed, so that they are copied."""
    from svoo_amd import fp8

    g = torch.Generator(device=gpu).manual_seed(2)
    x = torch.randn(6, 50, 300, generator=g, device=gpu).to(BF16)
    w = fp8.fp8_quantize_blocks(torch.randn(70, 300, generator=g, device=gpu))
    q, s = fp8.fp8_quantize_rows(x)
    want = fp8.fp8_matmul(q, s, *w).transpose(0, 1)
    assert torch.equal(fp8.fp8_matmul(q.transpose(0, 1), s.transpose(0, 1), *w), want)
    assert torch.equal(fp8.fp8_dequantize(q.transpose(0, 1), s.transpose(0, 1), cols=300),
                       fp8.fp8_dequantize(q, s, cols=300).transpose(0, 1))
    assert torch.equal(fp8.fp8_matmul(*fp8.fp8_quantize_rows(x.transpose(0, 1)), *w), want)
