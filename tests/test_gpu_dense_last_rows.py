"""Dense attention whose last rows hold infinities, where a tile goes on behind them."""

import math

import pytest
import torch

from test_gpu_dense import BF, FP, lens, make
from train_ops_helpers import say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("d", [64, 128, 40])
@pytest.mark.parametrize("sq,sk,k_len", [(80, 90, None), (80, 1, None), (300, 129, None), (80, 200, 70), (3, 5001, None),
                                         (3, 9000, 4100), (80, 128, None)])
def test_an_infinite_value_of_the_last_key(gpu, sq, sk, k_len, d, dtype):
    """Its column of o is infinite, not NaN, and the others keep their bits."""
    from svoo_amd import dense

    say("last value", sq, sk, k_len, d, dtype)
    q, k, v, _ = make(41, 1, 2, 2, sq, sk, d, dtype, gpu)
    kw = dict(k_lens=lens(None if k_len is None else [k_len], gpu))
    clean = dense.dense_attention(q, k, v, **kw)
    for value in (math.inf, -math.inf):
        v2 = v.clone()
        v2[0, 1, (k_len or sk) - 1, 9] = value
        o = dense.dense_attention(q, k, v2, **kw)
        assert (o[0, 1, :, 9] == value).all()
        o[0, 1, :, 9] = clean[0, 1, :, 9]
        assert torch.equal(o, clean)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("d", [64, 128, 40])
@pytest.mark.parametrize("heads,sq,q_len,sk", [(2, 90, None, 80), (2, 1, None, 80), (4, 129, None, 300), (2, 200, 70, 80),
                                               (2, 5001, None, 30), (2, 128, None, 80)])
def test_an_infinite_gradient_of_the_last_query(gpu, heads, sq, q_len, sk, d, dtype):
    """Its column of dv is infinite, not NaN; dv's other columns, and the other queries' dq, are as they were."""
    from svoo_amd import dense

    say("last gradient", heads, sq, q_len, sk, d, dtype)
    q, k, v, dy = make(42, 1, heads, 2, sq, sk, d, dtype, gpu)
    kw = dict(q_lens=lens(None if q_len is None else [q_len], gpu))
    fwd = dense.dense_attention_fwd(q, k, v, **kw)
    clean = dense.dense_attention_bwd(dy, q, k, v, *fwd, **kw)
    last = (q_len or sq) - 1
    dy2 = dy.clone()
    dy2[0, -1, last, 9] = -math.inf
    dq, dk, dv = dense.dense_attention_bwd(dy2, q, k, v, *fwd, **kw)
    assert (dv[0, 1, :, 9] == -math.inf).all()
    dv[0, 1, :, 9] = clean[2][0, 1, :, 9]
    assert torch.equal(dv, clean[2])
    if dtype is BF:  # fp16's dS is scaled by the largest incoming gradient of the heads
        rows = torch.arange(sq, device=gpu) != last
        assert torch.equal(dq[0, -1, rows], clean[0][0, -1, rows])
        assert torch.equal(dq[0, :-1], clean[0][0, :-1])
        assert torch.equal(dk[:, 0], clean[1][:, 0])
