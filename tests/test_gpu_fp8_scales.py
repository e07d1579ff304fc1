"""Products over the whole range of scales, against 64 bits."""

import pytest
import torch

from norm_fp8_helpers import say

pytestmark = pytest.mark.gpu

E4, E5, E8 = torch.float8_e4m3fn, torch.float8_e5m2, torch.float8_e8m0fnu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _operand(rows, values, byte, dtype, gpu):
    """Rows with ``values`` in turn at one contracted position of 128 and zeros beside it, one scale byte for all."""
    v = torch.zeros(rows, 128, device=gpu)
    v[:, 5] = torch.tensor(values, device=gpu).repeat(-(-rows // len(values)))[:rows]
    q = v.to(dtype)
    assert torch.equal(q.float(), v)
    return q, torch.full((rows, 1), byte, dtype=torch.uint8, device=gpu).view(E8), v.double()


@pytest.mark.parametrize("m", [7, 64, 65, 300, 5000])  # few rows, shares, both tiles
@pytest.mark.parametrize("a_type", [E4, E5])
def test_product_at_every_scale(gpu, m, a_type):
    """Every scale byte of a with one of b that brings the products near 1, and with b's own of 1: one product per result,
    so the exact value rounded once.  With fp32 results an operand's values are those that bf16 has: in steps of 2^-133
    below 2^-126, infinite from 2^128 on."""
    from svoo_amd import fp8

    n = 1200 if m == 5000 else 160
    a_values = [1.0, 2.0 ** -9, 1.125, 448.0, -2.0 ** -6, 0.0, 7.0] if a_type == E4 else \
        [1.0, 2.0 ** -16, 1.25, 57344.0, -2.0 ** -14, 0.0, 7.0]
    b_values = [1.0, 256.0, -2.0 ** -6, 3.5, 0.0]
    for byte in [*range(0, 12), 60, 127, 200, *range(240, 255)]:
        for other in sorted({127, min(254 - byte, 254)}):
            qa, sa, va = _operand(m, a_values, byte, a_type, gpu)
            qb, sb, vb = _operand(n, b_values, other, E4, gpu)
            say("scales", m, a_type, byte, other)
            xa, xb = va * 2.0 ** (byte - 127), vb * 2.0 ** (other - 127)
            for out in (BF16, F16, F32):
                a, b = (xa, xb) if out != F32 else (xa.to(BF16).double(), xb.to(BF16).double())
                want = (a[:, 5:6] * b[:, 5]).to(out) + 0.0  # 0 for both zeros
                got = fp8.fp8_matmul(qa, sa, qb, sb, out_dtype=out) + 0.0
                assert torch.equal(torch.nan_to_num(got, nan=1.5), torch.nan_to_num(want, nan=1.5)), (byte, other, out)
