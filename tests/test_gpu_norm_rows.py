"""Layer norm over rows that the other tests leave out, in every width class of its kernels: rows that are not finite, more
rows than the grid takes at a time, and 8-bit results of all of them."""

import pytest
import torch

from norm_fp8_helpers import say

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
