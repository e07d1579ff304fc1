"""Dense attention where scores are -inf: keys that a channel masks, and products that overflow."""

import math

import pytest
import torch

from test_gpu_dense import BF, FP, make
from train_ops_helpers import HALF, attention64, held, say

pytestmark = pytest.mark.gpu

# queries, keys, the keys whose score is -inf: whole tiles of 64 before, between and behind the others
STRETCHES = [
    (70, 300, [(0, 64)]), (70, 300, [(0, 200)]), (70, 300, [(0, 299)]), (70, 300, [(1, 300)]), (70, 300, [(64, 128), (256, 300)]),
    (300, 130, [(0, 65)]), (5, 9000, [(0, 8999)]), (5, 9000, [(0, 100), (3000, 6200)]), (5, 9000, [(1, 9000)]),
    (1, 64, [(0, 63)]),
]


def kept(sk, stretches):
    on = torch.ones(sk, dtype=torch.bool)
    for a, b in stretches:
        on[a:b] = False
    return on


@pytest.mark.parametrize("d", [64, 128, 40])
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("sq,sk,stretches", STRETCHES)
def test_keys_that_a_channel_masks(gpu, sq, sk, stretches, dtype, d):
    """A channel is 1 in every query and -inf in the masked keys: the others' results are those without these keys.  dq has no
    value in that channel, where dS = 0 is multiplied by -inf."""
    from svoo_amd import dense

    say("channel", sq, sk, stretches, dtype, d)
    q, k, v, dy = make(31, 1, 4, 2, sq, sk, d, dtype, gpu)
    on = kept(sk, stretches)
    q[..., 0] = 1.0
    k[..., 0] = torch.where(on, 0.0, -math.inf).to(gpu)
    want = attention64(q, k[:, :, on], v[:, :, on], dy, half=HALF[dtype])
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = dense.dense_attention(*leaves)
    dq, dk, dv = torch.autograd.grad(o, leaves, dy)
    held(o, want["o"], "o")
    held(dense.dense_attention_fwd(q, k, v)[2], want["lse"], "lse")
    assert not dv[:, :, ~on].any() and not dk[:, :, ~on].any()
    held(dv[:, :, on], want["dv"], "dv")
    held(dk[:, :, on], want["dk"], "dk")
    assert dq[..., 0].isnan().all()
    held(dq[..., 1:], tuple(t[..., 1:] for t in want["dq"]), "dq")


@pytest.mark.parametrize("sq,sk,stretches", STRETCHES)
def test_products_that_overflow(gpu, sq, sk, stretches):
    """2^100 in a channel of every third query and -2^100 in that of the masked keys: their scores are past fp32's range, and the
    queries between see all keys."""
    from svoo_amd import dense

    say("overflow", sq, sk, stretches)
    q, k, v, dy = make(32, 1, 2, 2, sq, sk, 128, BF, gpu)
    on = kept(sk, stretches)
    flag = torch.arange(sq) % 3 == 0
    q[..., 5] = torch.where(flag, 2.0 ** 100, 0.0).to(gpu)
    k[..., 5] = torch.where(on, 0.0, -2.0 ** 100).to(gpu)
    few = attention64(q[:, :, flag], k[:, :, on], v[:, :, on], dy[:, :, flag])
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = dense.dense_attention(*leaves)
    grads = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(o, leaves, dy)))
    grads["o"], grads["lse"] = o.detach(), dense.dense_attention_fwd(q, k, v)[2]
    for name in ("o", "lse", "dq"):
        held(grads[name][:, :, flag], few[name], name)
    if (~flag).any():
        all_keys = attention64(q[:, :, ~flag], k, v, dy[:, :, ~flag])
        for name in ("o", "lse", "dq"):
            held(grads[name][:, :, ~flag], all_keys[name], name)
        for name in ("dk", "dv"):  # the sums of both kinds of queries
            for part in range(2):
                all_keys[name][part][:, :, on] += few[name][part]
            held(grads[name], all_keys[name], name)
    else:
        for name in ("dk", "dv"):
            held(grads[name][:, :, on], few[name], name)
            assert not grads[name][:, :, ~on].any()


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("sq,sk", [(70, 300), (3, 9000), (200, 64), (1, 1)])
def test_queries_whose_every_score_is_minus_infinity(gpu, sq, sk, dtype):
    """They have no probabilities: o and the log-sum-exp are NaN, and so are their gradients.  Other heads keep their bits."""
    from svoo_amd import dense

    say("none", sq, sk, dtype)
    q, k, v, dy = make(33, 1, 2, 2, sq, sk, 64, dtype, gpu)
    q[..., 0] = 1.0
    clean = dense.dense_attention_fwd(q, k, v)
    clean_grads = dense.dense_attention_bwd(dy, q, k, v, *clean)
    k2 = k.clone()
    k2[:, 1, :, 0] = -math.inf
    o, rest, lse = dense.dense_attention_fwd(q, k2, v)
    assert o[:, 1].isnan().all() and lse[:, 1].isnan().all()
    assert torch.equal(o[:, 0], clean[0][:, 0]) and torch.equal(lse[:, 0], clean[2][:, 0])
    for t, c in zip(dense.dense_attention_bwd(dy, q, k2, v, o, rest, lse), clean_grads):
        assert t[:, 1].isnan().all() and torch.equal(t[:, 0], c[:, 0])
