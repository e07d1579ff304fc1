"""Dense attention in fp16 where nearly all of the probability lies on one key whose value is 0."""

import math

import pytest
import torch

from test_gpu_dense import FP, lens, make
from train_ops_helpers import HALF, attention64, held, say

pytestmark = pytest.mark.gpu


def with_sink(seed, b, h, sq, sk, d, far, at, device):
    """Queries and keys whose scores lie within about 0.5 of 0, but for the key ``at``, ``far`` above, with a value of 0."""
    q, k, v, dy = make(seed, b, h, 1, sq, sk, d, FP, device, level=0.1)
    q[..., 0] = 8.0
    k[..., 0] = 0.0
    k[:, :, at] = 0.0
    k[:, :, at, 0] = far * math.sqrt(d) / 8.0
    v = v + 0.5
    v[:, :, at] = 0.0
    return q, k, v, dy


def probabilities(q, k):
    q, k = q.double().cpu(), k.double().cpu().repeat_interleave(q.shape[1] // k.shape[1], 1)
    return torch.softmax(q @ k.transpose(2, 3).contiguous() * q.shape[3] ** -0.5, -1)


def check(q, k, v, dy):
    """Within the bounds of other scores, and D within what is left of o in fp16: its smallest half step, 2^-25, times |do|."""
    from svoo_amd import dense

    want = attention64(q, k, v, dy, half=HALF[FP])
    p, scale = probabilities(q, k), q.shape[3] ** -0.5
    more = scale * 2.0 ** -25 * dy.double().cpu().abs().sum(-1, keepdim=True) * p
    heads, kk = q.shape[1] // k.shape[1], k.double().cpu().abs()
    want["dq"] = want["dq"][0], want["dq"][1] + more @ kk.repeat_interleave(heads, 1)
    sums = more.transpose(2, 3).contiguous() @ q.double().cpu().abs()
    want["dk"] = want["dk"][0], want["dk"][1] + sums.unflatten(1, (-1, heads)).sum(2)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = dense.dense_attention(*leaves)
    held(o, want["o"], "o")
    held(dense.dense_attention_fwd(q, k, v)[2], want["lse"], "lse")
    for t, name in zip(torch.autograd.grad(o, leaves, dy), ("dq", "dk", "dv")):
        held(t, want[name], name)


# 256 blocks of queries walk over all keys in one piece, fewer in shares
@pytest.mark.parametrize("b,h,sq,sk,d,far,at", [
    (16, 16, 3, 4000, 64, 12.0, 0), (16, 16, 3, 4000, 128, 14.02, 100), (16, 16, 3, 8192, 64, 14.02, 0),
    (16, 16, 3, 8192, 64, 17.0, 5000), (16, 16, 3, 8192, 40, 17.0, -1), (16, 16, 2, 20001, 64, 16.02, 0),
    (1, 2, 40, 8192, 64, 14.02, 0), (1, 2, 300, 3000, 128, 16.0, 10), (1, 1, 700, 200, 64, 9.0, 70),
])
def test_keys_far_below_a_key_without_a_value(gpu, b, h, sq, sk, d, far, at):
    """What the far keys add is all of o, and D's part of the sink's gradient.  P has all its bits down to 2^-26 of a row's
    largest, 18 below it."""
    say("sink", b, h, sq, sk, d, far, at)
    check(*with_sink(51, b, h, sq, sk, d, far, at, gpu))


@pytest.mark.parametrize("far", [19.0, 21.0, 23.0])
def test_keys_still_further_below(gpu, far):
    """Down to 2^-36 of the row's largest P has a step of its own: 2^-24 where the largest is 2^12, so each is off by 2^-37 of
    the largest at most, in the products and in what they are divided by."""
    from svoo_amd import dense

    say("further", far)
    q, k, v, _ = with_sink(52, 16, 16, 2, 8192, 64, far, 0, gpu)
    v = v * 64  # so that o is far from fp16's own smallest step
    value, bound = attention64(q, k, v, half=HALF[FP])["o"]
    top = probabilities(q, k).amax(-1, keepdim=True)
    more = 2.0 ** -37 * top * (v.double().cpu().abs().sum(2, keepdim=True) + 8192 * value.abs())
    held(dense.dense_attention(q, k, v), (value, bound + more), "o")
    held(dense.dense_attention(q, k, v, k_lens=lens([8192] * 16, gpu)), (value, bound + more), "o")


@pytest.mark.parametrize("b,h,sq", [(1, 2, 90), (16, 16, 3)])
@pytest.mark.parametrize("sk,rise", [(1500, 2.0), (1500, 3.0), (600, 8.0), (600, 0.5)])
def test_scores_that_rise_from_tile_to_tile(gpu, b, h, sq, sk, rise):
    """A row's maximum grows with every tile of 64 keys, past every earlier one."""
    say("rise", b, h, sq, sk, rise)
    q, k, v, dy = make(53, b, h, 1, sq, sk, 64, FP, gpu, level=0.3)
    q[..., 0] = 8.0
    k[..., 0] = (torch.arange(sk, device=gpu) // 64 * rise).to(FP)
    check(q, k, v, dy)
