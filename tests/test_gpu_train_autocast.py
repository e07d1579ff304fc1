"""The training attention in an fp32 transformer under autocast."""

import copy

import pytest
import torch

from train_ops_helpers import HALF, say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_an_fp32_attention_under_autocast(gpu, dtype):
    """Output and gradients against the formulas in 64 bits.  Fewer than 12 tensors are rounded to the type on the way to the
    output (x, four weights, q, k and v, their turned forms, P, o, the result), fewer than 24 to a gradient; each is half a step
    at most and passes maps that do not enlarge a random error against its signal by more than 2."""
    from svoo_amd import dit
    from svoo_amd.inference import replace_wan_attention_trainable

    cfg = dit.WanDiTConfig(num_attention_heads=2, ffn_dim=64, num_layers=1, text_dim=32)
    pipe = dit.make_pipe(cfg, device=gpu, dtype=torch.float32, seed=4)
    attn = pipe.transformer.blocks[0].attn1
    exact = copy.deepcopy(attn).double().cpu()
    replace_wan_attention_trainable(pipe, 64, 96, 9)
    g = torch.Generator().manual_seed(2)
    x, dy = (torch.randn(2, 72, cfg.dim, generator=g) for _ in range(2))
    rope = dit.rope_tables(cfg, 3, 4, 6, gpu)
    leaf = x.to(gpu).requires_grad_()
    with torch.autocast("cuda", dtype):
        out = attn(leaf, rotary_emb=rope)
    assert out.dtype == dtype
    names, params = zip(*attn.named_parameters())
    got = torch.autograd.grad(out, [leaf, *params], dy.to(gpu, dtype))
    cos, sin = (t.double().cpu()[..., 0::2] for t in rope)
    xd = x.double().requires_grad_()

    def turned(t):
        t = t.unflatten(2, (2, -1))
        a, b = t[..., 0::2], t[..., 1::2]
        return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2).transpose(1, 2)

    q, k = turned(exact.norm_q(exact.to_q(xd))), turned(exact.norm_k(exact.to_k(xd)))
    v = exact.to_v(xd).unflatten(2, (2, -1)).transpose(1, 2)
    o = torch.softmax(q @ k.transpose(2, 3) / 128 ** 0.5, -1) @ v
    want_out = exact.to_out[0](o.transpose(1, 2).flatten(2))
    want = torch.autograd.grad(want_out, [xd, *dict(exact.named_parameters()).values()], dy.double())

    def rel(a, b):
        return ((a.detach().double().cpu() - b).norm() / b.norm()).item()

    say("autocast", dtype, rel(out, want_out.detach()))
    assert rel(out, want_out.detach()) <= 24 * HALF[dtype]
    for name, a, b in zip(("x", *names), got, want):
        assert a.dtype == torch.float32 and a.isfinite().all()
        if name != "to_k.bias":  # a shift of all keys moves no probability
            say(name, rel(a, b))
            assert rel(a, b) <= 48 * HALF[dtype], name
