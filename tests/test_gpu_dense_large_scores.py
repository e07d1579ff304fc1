"""Dense attention where scores are so large that a step of fp32 is more than the range of fp16's probabilities."""

import math

import pytest
import torch

from test_gpu_dense import BF, FP, make
from train_ops_helpers import say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("d,sk", [(64, 65), (128, 500), (64, 4099)])
@pytest.mark.parametrize("power", [0, 4, 10, 14, 15, 16, 17, 18])
def test_one_key_each_at_large_scores(gpu, power, d, sk, dtype):
    """Each query picks one key, whose score is 50 to 650 times 2^power and at least 100 times 2^power above every other: o is that
    key's value, bit for bit, whatever one step of such a score is (16 at the last: the highest P lies within 2^-8 .. 2^8)."""
    from svoo_amd import dense

    say("large", power, d, sk, dtype)
    g = torch.Generator().manual_seed(sk)
    n = 300
    pick = torch.randint(0, sk, (n,), generator=g)
    pick[0], pick[-1] = 0, sk - 1
    bits = ((torch.arange(sk)[:, None] >> torch.arange(13)) & 1) * 2.0 - 1
    keys = torch.zeros(sk, d)
    keys[:, :13] = bits
    for sign in (1.0, -1.0):  # and the same with all scores below 0
        shift = torch.zeros(sk, d)
        shift[:, 13] = -16.0 if sign < 0 else 0.0
        q = 50 * keys[pick]
        q[:, 13] = 50.0
        q, k = q.expand(1, 2, n, d).to(dtype).to(gpu), (keys + shift).expand(1, 1, sk, d).to(dtype).to(gpu)
        v = torch.randn(1, 1, sk, d, generator=g).to(dtype).to(gpu)
        o = dense.dense_attention(q, k, v, scale=2.0 ** power)
        assert torch.equal(o, v[:, :, pick].expand(1, 2, n, d))


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("sq,sk", [(80, 90), (3, 5000)])
def test_a_query_that_is_not_finite(gpu, sq, sk, dtype, value):
    """Its row is NaN (its scores are infinities of both signs), and the others keep their bits."""
    from svoo_amd import dense

    say("not finite", value, sq, sk, dtype)
    q, k, v, _ = make(61, 1, 2, 2, sq, sk, 64, dtype, gpu)
    clean = dense.dense_attention_fwd(q, k, v)
    q2 = q.clone()
    q2[0, 1, sq // 2, 3] = value
    o, _, lse = dense.dense_attention_fwd(q2, k, v)
    bad = torch.zeros(1, 2, sq, dtype=torch.bool, device=gpu)
    bad[0, 1, sq // 2] = True
    assert o[bad].isnan().all() and torch.equal(o[~bad], clean[0][~bad])
    assert not lse[bad].isfinite().any() and torch.equal(lse[~bad], clean[2][~bad])
