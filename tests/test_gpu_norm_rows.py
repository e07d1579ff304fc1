"""Layer norm over rows that the other tests leave out, in every width class of its kernels: rows that are not finite, more
rows than the grid takes at a time, and 8-bit results of all of them."""

import pytest
import torch

from norm_fp8_helpers import U32, norm64, say, within

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32

# The forward pass's classes, (lanes a row, chunks of eight elements a lane) with their widths, whole chunks and not:
# (16, 1) to 128; (64, 1) to 512; (64, 2) to 1024 whole; (64, 3) to 1536; (64, 5) to 2560 whole; (64, 10) to 5120; (1024, 1)
# to 8192; (1024, 2) to 16384
CLASSES = [40, 57, 256, 301, 1000, 999, 1536, 1531, 2560, 2561, 5120, 5111, 8192, 8191, 16384, 16383]


@pytest.mark.parametrize("cols", CLASSES)
def test_statistics_of_rows_that_are_not_finite(gpu, cols):
    """The formula's: the mean of a row with an infinity is that infinity (NaN with both or with NaN), its variance NaN."""
    from svoo_amd import norm

    g = torch.Generator(device=gpu).manual_seed(cols)
    inf, nan = float("inf"), float("nan")
    for dtype in (BF16, F16, F32):
        x = torch.randn(12, cols, generator=g, device=gpu).to(dtype)
        last, mid = cols - 1, cols // 2
        x[1, mid], x[2, 0], x[3, last] = nan, inf, -inf
        x[4, 0], x[4, last] = inf, -inf
        x[5, 3], x[5, mid] = nan, inf
        x[6, 1], x[6, last] = inf, inf
        say("not finite", cols, dtype)
        y, mean, rstd = norm.layer_norm_fwd(x)
        want = x.double().mean(-1)
        bad = torch.zeros(12, dtype=torch.bool, device=gpu)
        bad[1:7] = True
        assert torch.equal(torch.nan_to_num(mean[bad].double(), nan=7.0), torch.nan_to_num(want[bad], nan=7.0))
        assert rstd[bad].isnan().all() and y[bad].isnan().all()
        assert mean[~bad].isfinite().all() and rstd[~bad].isfinite().all() and y[~bad].isfinite().all()
        dx, _, _ = norm.layer_norm_bwd(torch.ones_like(x), x, mean, rstd)
        assert dx[bad].isnan().all() and dx[~bad].isfinite().all()


def _resident_rows(cols):
    """Rows that one round of the forward pass's grid takes: 32 waves on each of 256 CUs, and as many lanes to a row."""
    lanes = 16 if cols <= 128 else 64 if cols <= 5120 else 1024
    threads = max(lanes, 256)
    return 256 * (2048 // threads) * (threads // lanes)


def _within_blocks(y, x, w, b, eps=1e-6):
    """Every element of y against the formula in 64 bits, some rows at a time, to the bound of the other tests: 80 U of
    |n| + 1 and four roundings."""
    for r in range(0, x.shape[0], 4096):
        n, _, want = norm64(x[r:r + 4096].double(), w, b, eps)
        within(y[r:r + 4096], want, 80 * U32 * (n.abs() + 1) * w.abs() + 4 * U32 * (want.abs() + b.abs()))


@pytest.mark.parametrize("cols", CLASSES)
def test_more_rows_than_the_grid_takes_at_a_time(gpu, cols):
    """Two and a part rounds of rows per group: the second and third row of a block (and, for rows of several waves, its
    scratch used again) against the definition, the 8-bit form against the two steps."""
    from svoo_amd import fp8, norm

    rows = 2 * _resident_rows(cols) + 37
    g = torch.Generator(device=gpu).manual_seed(cols)
    for dtype in (BF16, F16, F32):
        x = torch.randn(rows, cols, generator=g, device=gpu)
        x.mul_(torch.exp(torch.randn(rows, 1, generator=g, device=gpu))).add_(torch.randn(rows, 1, generator=g, device=gpu))
        x = x.to(dtype)
        w = 1 + 0.2 * torch.randn(cols, generator=g, device=gpu)
        b = 0.2 * torch.randn(cols, generator=g, device=gpu)
        say("many rows", rows, cols, dtype)
        y, mean, rstd = norm.layer_norm_fwd(x, w, b)
        _within_blocks(y, x, w.double(), b.double())
        want_mean = torch.cat([t.double().mean(-1) for t in x.split(4096)])
        size = torch.cat([t.double().abs().mean(-1) for t in x.split(4096)])
        within(mean, want_mean, 80 * U32 * size)
        for t in (torch.float8_e4m3fn, torch.float8_e5m2):
            q, s = norm.layer_norm_fp8(x, w, b, dtype=t)
            q2, s2 = fp8.fp8_quantize_rows(y, dtype=t)
            assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8))
            assert torch.equal(s.view(torch.uint8), s2.view(torch.uint8))


@pytest.mark.parametrize("cols", [40, 57, 256, 301, 1000, 999, 1536, 1531, 2560, 2561, 5120, 5111, 8192, 8191, 16384, 16383])
def test_many_rows_of_each_batch_entry(gpu, cols):
    """The same with parameters per batch entry: a block's rows are one entry's, and it takes several of them."""
    from svoo_amd import norm

    batch = 3
    rows = 2 * (_resident_rows(cols) // batch) + 11
    g = torch.Generator(device=gpu).manual_seed(cols + 1)
    x = torch.randn(batch, rows, cols, generator=g, device=gpu).to(BF16)
    sc, sh = (0.3 * torch.randn(batch, 1, cols, generator=g, device=gpu) for _ in range(2))
    say("many rows of a batch entry", batch, rows, cols)
    y = norm.layer_norm(x, scale=sc, shift=sh)
    for i in range(batch):
        _within_blocks(y[i], x[i], 1 + sc[i].double(), sh[i].double())


@pytest.mark.parametrize("cols", sorted({1, 7, 8, 24, 40, 127, 128, 129, 130, 300, 511, 512, 513, 520, 999, 1000, 1024, 1025, 1032,
                                         1535, 1536, 1537, 2048, 2050, 2560, 2561, 4096, 4104, 5111, 5120, 5121, 6145, 8191, 8192,
                                         8193, 8200, 16383, 16384}))
def test_8_bit_results_in_every_class(gpu, cols):
    """Bit for bit the two steps, whatever ends a row's last block of 128; also where a block's maximum is infinite (an
    infinity in y from fp16's range, from x, or from a shift) or NaN."""
    from svoo_amd import fp8, norm

    g = torch.Generator(device=gpu).manual_seed(cols)
    inf, nan = float("inf"), float("nan")
    for dtype in (BF16, F16, F32):
        x = torch.randn(2, 23, cols, generator=g, device=gpu).to(dtype)
        x[0, 1, cols // 2], x[0, 2, cols - 1], x[1, 3, 0] = nan, inf, -inf
        sc, sh = (0.3 * torch.randn(2, 1, cols, generator=g, device=gpu) for _ in range(2))
        big, top = sc.clone(), sh.clone()
        big[0, 0, ::5] = 60000.0  # beyond fp16 where |n| passes 1.1; finite in the others
        top[0, 0, cols // 3], top[1, 0, cols - 1], top[1, 0, 0] = inf, -inf, nan
        say("to 8 bits", cols, dtype)
        for scale, shift in ((sc, sh), (big, sh), (sc, top), (None, None)):
            y = norm.layer_norm(x, scale=scale, shift=shift)
            if scale is big and dtype == F16 and cols > 40:
                assert y.isinf().any()
            for t in (torch.float8_e4m3fn, torch.float8_e5m2):
                q, s = norm.layer_norm_fp8(x, scale=scale, shift=shift, dtype=t)
                q2, s2 = fp8.fp8_quantize_rows(y, dtype=t)
                assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8))
                assert torch.equal(s.view(torch.uint8), s2.view(torch.uint8))
