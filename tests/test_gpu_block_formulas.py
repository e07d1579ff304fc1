"""A Wan block with and without fused norms, fused residuals and an 8-bit FFN, against its formulas."""

import copy

import pytest
import torch

from train_ops_helpers import say

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def make_block(device, seed=5):
    """A block with random norms, an FFN whose results are as large as the stream, and inputs of order 1 (so gates too)."""
    from svoo_amd import dit

    cfg = dit.WanDiTConfig(num_attention_heads=2, ffn_dim=384, num_layers=1, text_dim=64)
    pipe = dit.make_pipe(cfg, device=device, dtype=BF, seed=seed)
    g = torch.Generator().manual_seed(seed)
    block = pipe.transformer.blocks[0].requires_grad_(False)
    for m in block.modules():
        if isinstance(m, (torch.nn.RMSNorm, torch.nn.LayerNorm)) and m.weight is not None:
            m.weight.data.add_(0.1 * torch.randn(m.weight.shape, generator=g).to(m.weight))
        if isinstance(m, torch.nn.Linear):
            m.weight.data.mul_(3.0)
    x, ctx, temb = (torch.randn(2, n, cfg.dim, generator=g).to(BF) for n in (72, 11, 6))
    return pipe, block, [x, ctx, temb, dit.rope_tables(cfg, 3, 4, 6, device)]


def eight_bit_ffn(block):
    from svoo_amd import Fp8Linear

    block.ffn = torch.nn.Sequential(Fp8Linear.from_linear(block.ffn[0], "gelu_tanh"), torch.nn.Identity(),
                                    Fp8Linear.from_linear(block.ffn[2]))


def composed(block, x, ctx, temb, rope, norms, residuals, eight):
    """The block as calls of its parts."""
    from svoo_amd import norm

    shift, scale, gate, c_shift, c_scale, c_gate = (block.scale_shift_table.float() + temb.float()).unbind(1)
    shift, scale, gate, c_shift, c_scale, c_gate = (t[:, None] for t in (shift, scale, gate, c_shift, c_scale, c_gate))

    def modulated(t, by, to):
        if norms:
            return norm.layer_norm(t, scale=by, shift=to, eps=1e-6)
        return (torch.nn.functional.layer_norm(t.float(), t.shape[-1:], None, None, 1e-6) * (1 + by) + to).to(BF)

    a = block.attn1(modulated(x, scale, shift), rotary_emb=rope)
    w, b = block.norm2.weight, block.norm2.bias
    if residuals:
        x, n = norm.residual_norm(x, a, gate, w, b, eps=1e-6)
    else:
        x = (x.float() + a.float() * gate).to(BF)
        n = norm.layer_norm(x, w, b, eps=1e-6) if norms else \
            torch.nn.functional.layer_norm(x.float(), x.shape[-1:], w.float(), b.float(), 1e-6).to(BF)
    a = block.attn2(n, ctx)
    x = norm.gated_residual(x, a) if residuals else x + a
    if eight and norms:
        f = block.ffn[2](block.ffn[0].forward_quantized(*norm.layer_norm_fp8(x, scale=c_scale, shift=c_shift, eps=1e-6)))
    else:
        f = block.ffn(modulated(x, c_scale, c_shift))
    return norm.gated_residual(x, f, c_gate) if residuals else (x.float() + f.float() * c_gate).to(BF)


@pytest.mark.parametrize("train", [False, True])
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("norms,residuals", [(False, False), (True, False), (True, True)])
def test_a_block_is_its_parts_bit_for_bit(gpu, norms, residuals, eight, train):
    from svoo_amd.inference import replace_wan_attention_trainable

    say("block", norms, residuals, eight, train)
    pipe, block, (*args, rope) = make_block(gpu)
    if train:
        replace_wan_attention_trainable(pipe, 64, 96, 9)
    if eight:
        eight_bit_ffn(block)
    args = [t.to(gpu) for t in args]
    pipe.transformer.fuse_norms(residuals=True)  # switches that do not stay
    pipe.transformer.fuse_norms(norms, residuals=residuals)
    with torch.no_grad():
        assert torch.equal(block(*args, rope), composed(block, *args, rope, norms, residuals, eight))


CHANGES = ("gate negated", "gate one", "c_gate negated", "c_gate one", "c_scale and c_shift exchanged", "no c_scale", "no c_shift",
           "no cross-attention", "no ffn", "scale and shift exchanged")


def formulas(block, weights, x, ctx, temb, rope, change=None):
    """``(out, norms of the three branches and the stream)`` in 64 bits on the CPU, ``weights`` of the two FFN layers; with a
    change, of another block."""
    shift, scale, gate, c_shift, c_scale, c_gate = (t[:, None] for t in (block.scale_shift_table + temb).unbind(1))
    one, none = torch.ones_like(gate), torch.zeros_like(gate)
    gate = {"gate negated": -gate, "gate one": one}.get(change, gate)
    c_gate = {"c_gate negated": -c_gate, "c_gate one": one}.get(change, c_gate)
    if change == "c_scale and c_shift exchanged":
        c_scale, c_shift = c_shift, c_scale
    if change == "scale and shift exchanged":
        scale, shift = shift, scale
    c_scale = none if change == "no c_scale" else c_scale
    c_shift = none if change == "no c_shift" else c_shift
    cos, sin = (t.double().cpu()[..., 0::2] for t in rope)

    def ln(t, w=None, b=None):
        return torch.nn.functional.layer_norm(t, t.shape[-1:], w, b, 1e-6)

    def attend(attn, x, c, turn):
        q, k, v = attn.norm_q(attn.to_q(x)), attn.norm_k(attn.to_k(c)), attn.to_v(c)
        q, k, v = (t.unflatten(2, (attn.heads, -1)) for t in (q, k, v))
        if turn:
            q, k = (torch.stack((t[..., 0::2] * cos - t[..., 1::2] * sin, t[..., 0::2] * sin + t[..., 1::2] * cos), -1).flatten(-2)
                    for t in (q, k))
        q, k, v = (t.transpose(1, 2) for t in (q, k, v))
        o = torch.softmax(q @ k.transpose(2, 3) / 128 ** 0.5, -1) @ v
        return attn.to_out[0](o.transpose(1, 2).flatten(2))

    n = ln(x) * (1 + scale) + shift
    a1 = gate * attend(block.attn1, n, n, True)
    h = x + a1
    a2 = attend(block.attn2, ln(h, block.norm2.weight, block.norm2.bias), ctx, False)
    a2 = 0 * a2 if change == "no cross-attention" else a2
    h = h + a2
    (w0, b0), (w2, b2) = weights
    f = torch.nn.functional.gelu((ln(h) * (1 + c_scale) + c_shift) @ w0.t() + b0, approximate="tanh") @ w2.t() + b2
    f = 0 * f if change == "no ffn" else c_gate * f
    return h + f, [t.norm().item() for t in (a1, a2, f, h)]


def bound_of(sizes):
    """In 2-norm, in which errors of roundings apart add as their squares.  16-bit roundings: fewer than 20 in each branch, which
    pass maps that do not enlarge a random error against its signal by more than 2, half a step 2^-8 each: 2 sqrt(20) 2^-8 < 9
    2^-8.  The stream is rounded three times.  8-bit rows (weights are taken as they are held): both FFN inputs, 2^-4 each, the
    first through the GELU, which enlarges an error against its signal by 1.13 / 0.58 at most for values about 0:
    sqrt(1.95^2 + 1) 2^-4 < 0.14."""
    a1, a2, f, h = sizes
    return 9 * 2.0 ** -8 * (a1 + a2 + f) + 3 ** 0.5 * 2.0 ** -8 * h + 0.14 * f


@pytest.mark.parametrize("train", [False, True])
def test_an_8_bit_ffn_behind_fused_residuals(gpu, train):
    """Against the formulas, at inputs and gates where a wrong gate, shift, scale or branch is further off than the bound."""
    from svoo_amd import fp8_dequantize
    from svoo_amd.inference import replace_wan_attention_trainable

    pipe, block, (*args, rope) = make_block(gpu)
    exact = copy.deepcopy(block).double().cpu()
    if train:
        replace_wan_attention_trainable(pipe, 64, 96, 9)
    eight_bit_ffn(block)
    weights = [(fp8_dequantize(m.weight_q.view(torch.float8_e4m3fn), m.weight_scale.view(torch.float8_e8m0fnu),
                               out_dtype=torch.float32).double().cpu(), m.bias.double().cpu())
               for m in (block.ffn[0], block.ffn[2])]
    doubles = [t.double() for t in args]
    with torch.no_grad():
        want, sizes = formulas(exact, weights, *doubles, rope)
        for change in CHANGES:
            off = (formulas(exact, weights, *doubles, rope, change)[0] - want).norm().item()
            assert off > 1.5 * bound_of(sizes), (change, off, bound_of(sizes))
        for residuals in (False, True):
            pipe.transformer.fuse_norms(residuals=residuals)
            off = (block(*(t.to(gpu) for t in args), rope).double().cpu() - want).norm().item()
            say("8 bits", residuals, "%.3g of %.3g" % (off, bound_of(sizes)))
            assert off <= bound_of(sizes)
