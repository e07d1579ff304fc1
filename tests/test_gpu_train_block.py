"""A Wan block's training step on dense attention, rotary positions, norms and gated residuals together."""

import copy

import pytest
import torch

from train_ops_helpers import HALF, say

pytestmark = pytest.mark.gpu


def _model(gpu, dtype, layers=1):
    from svoo_amd import dit

    cfg = dit.WanDiTConfig(num_attention_heads=2, ffn_dim=256, num_layers=layers, text_dim=64)
    pipe = dit.make_pipe(cfg, device=gpu, dtype=dtype, seed=3)
    g = torch.Generator().manual_seed(1)
    for m in pipe.transformer.modules():
        if isinstance(m, (torch.nn.RMSNorm, torch.nn.LayerNorm)) and m.weight is not None:
            m.weight.data.add_(0.1 * torch.randn(m.weight.shape, generator=g).to(m.weight))
    return pipe, cfg, g


def _rel(a, b):
    return ((a.double().cpu() - b).norm() / b.norm()).item()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_blocks_gradients(gpu, dtype):
    """A block's output and every gradient against the same block in float64 on the CPU.

    Between the block's weights and a gradient lie fewer than 40 tensors that are rounded to the type (projections, norms,
    attention, residuals, and each one's gradient), and P and dS.  Each rounding is half a step at most, relative 2-norm
    included, and passes a linear map or norm that does not enlarge a random error against its signal by more than 2 here:
    80 half-steps bound them all, and a wrong term is of order 1."""
    from svoo_amd import dit
    from svoo_amd.inference import replace_wan_attention_trainable

    pipe, cfg, g = _model(gpu, dtype)
    block = pipe.transformer.blocks[0]
    exact = copy.deepcopy(block).double().cpu()
    replace_wan_attention_trainable(pipe, 64, 96, 9)
    pipe.transformer.fuse_norms(residuals=True)
    x, ctx, temb, dy = (torch.randn(2, n, cfg.dim, generator=g).to(dtype) for n in (72, 11, 6, 72))
    rope = dit.rope_tables(cfg, 3, 4, 6, gpu)
    args = [t.to(gpu).requires_grad_() for t in (x, ctx, temb)]
    names, params = zip(*block.named_parameters())
    out = block(*args, rope)
    got = torch.autograd.grad(out, [*args, *params], dy.to(gpu))

    def reference(x, ctx, temb):  # the block's formulas in 64 bits
        ln = torch.nn.functional.layer_norm
        mod = (exact.scale_shift_table + temb).chunk(6, dim=1)
        cos, sin = (t.double().cpu() for t in rope)

        def attend(attn, x, c, turn):
            q, k, v = attn.norm_q(attn.to_q(x)), attn.norm_k(attn.to_k(c)), attn.to_v(c)
            q, k, v = (t.unflatten(2, (attn.heads, -1)) for t in (q, k, v))
            if turn:
                q, k = (torch.stack((t[..., 0::2] * cos[..., 0::2] - t[..., 1::2] * sin[..., 0::2],
                                     t[..., 0::2] * sin[..., 0::2] + t[..., 1::2] * cos[..., 0::2]), -1).flatten(-2) for t in (q, k))
            p = torch.softmax(torch.einsum("bqhd,bkhd->bhqk", q, k) / 128 ** 0.5, -1)
            return attn.to_out[0](torch.einsum("bhqk,bkhd->bqhd", p, v).flatten(2))

        n = ln(x, (cfg.dim,), eps=1e-6) * (1 + mod[1]) + mod[0]
        x = x + mod[2] * attend(exact.attn1, n, n, True)
        n = ln(x, (cfg.dim,), exact.norm2.weight, exact.norm2.bias, 1e-6)
        x = x + attend(exact.attn2, n, ctx, False)
        return x + mod[5] * exact.ffn(ln(x, (cfg.dim,), eps=1e-6) * (1 + mod[4]) + mod[3])

    leaves = [t.double().requires_grad_() for t in (x, ctx, temb)]
    want_out = reference(*leaves)
    want = torch.autograd.grad(want_out, [*leaves, *exact.parameters()], dy.double())
    assert _rel(out.detach(), want_out.detach()) <= 80 * HALF[dtype]
    for name, a, b in zip(("x", "ctx", "temb", *names), got, want):
        say(name, dtype, "%.2g" % _rel(a, b) if b.norm() > 0 else "")
        if "to_k.bias" in name:  # a shift of all keys moves no probability: 0 but for roundings
            scale = dict(zip(names, want[3:]))[name.replace("to_k.bias", "to_q.bias")].norm()
            assert (a.double().cpu() - b).norm() <= 80 * HALF[dtype] * max(scale, b.norm())
        else:
            assert _rel(a, b) <= 80 * HALF[dtype], name


@pytest.mark.parametrize("linear", [False, True])
def test_a_models_step_runs_and_every_parameter_has_its_gradient(gpu, linear):
    from svoo_amd import dit
    from svoo_amd.inference import replace_wan_attention_trainable, replace_wan_linear

    pipe, cfg, g = _model(gpu, torch.bfloat16, layers=2)
    replace_wan_attention_trainable(pipe, 128, 128, 5)
    if linear:
        replace_wan_linear(pipe, trainable=True)
    model = pipe.transformer.fuse_norms(residuals=True).requires_grad_(True)
    lat = torch.randn(dit.latent_shape(cfg, 128, 128, 5), generator=g).to(gpu, torch.bfloat16)
    txt = torch.randn(1, 9, 64, generator=g).to(gpu, torch.bfloat16)
    model(lat, torch.tensor([500.0], device=gpu), txt).float().square().mean().backward()
    for n, p in model.named_parameters():
        assert p.grad is not None and p.grad.isfinite().all(), n
        assert p.grad.any() or n.endswith("to_k.bias"), n


def test_inference_with_8_bit_layers_and_fused_residuals(gpu):
    """The 8-bit FFN takes its rows from the norm, behind a residual of its own, and the model's output stays within the
    8-bit layers' roundings of itself without the fusion."""
    from svoo_amd import dit
    from svoo_amd.inference import replace_wan_attention_trainable, replace_wan_linear

    pipe, cfg, g = _model(gpu, torch.bfloat16, layers=2)
    replace_wan_attention_trainable(pipe, 128, 128, 5)
    replace_wan_linear(pipe)
    lat = torch.randn(dit.latent_shape(cfg, 128, 128, 5), generator=g).to(gpu, torch.bfloat16)
    txt = torch.randn(1, 9, 64, generator=g).to(gpu, torch.bfloat16)
    t = torch.tensor([500.0], device=gpu)
    with torch.no_grad():
        want = pipe.transformer.fuse_norms()(lat, t, txt)
        got = pipe.transformer.fuse_norms(residuals=True)(lat, t, txt)
    # six residuals a model of two blocks, each rounded once instead of twice: 12 half-steps of bf16, which move 8-bit values
    # (half a step 2^-4) of eight layers where they lie next to a midpoint
    assert _rel(got, want.double().cpu()) <= 12 * 2.0 ** -8 + 8 * 2.0 ** -4


def test_other_blocks_keep_their_results(gpu):
    """Without the new switches a model's results are those of its tensor operations and fused norms, bit for bit."""
    from svoo_amd import dit

    pipe, cfg, g = _model(gpu, torch.bfloat16, layers=2)
    lat = torch.randn(dit.latent_shape(cfg, 128, 128, 5), generator=g).to(gpu, torch.bfloat16)
    txt = torch.randn(1, 9, 64, generator=g).to(gpu, torch.bfloat16)
    t = torch.tensor([500.0], device=gpu)
    with torch.no_grad():
        want = pipe.transformer.fuse_norms()(lat, t, txt)
        pipe.transformer.fuse_norms(residuals=True)(lat, t, txt)
        assert torch.equal(pipe.transformer.fuse_norms()(lat, t, txt), want)
