"""GPU tests of the 8-bit linear layers and the fused norms inside Wan-shaped blocks.

The operators have their own tests against 64 bits; here a block has to call them as it should, so it is compared bit for
bit with the same operators written out one after the other."""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def say(*a):
    print("[case]", *a, flush=True)


def _pipe(gpu, layers=2, heads=2, ffn=512, second=False):
    from svoo_amd import dit

    cfg = dit.WanDiTConfig(num_attention_heads=heads, ffn_dim=ffn, num_layers=layers, text_dim=64)
    pipe = dit.make_pipe(cfg, device=gpu, dtype=BF16, seed=5)
    g = torch.Generator(device=gpu).manual_seed(8)
    with torch.no_grad():
        for name, p in pipe.transformer.named_parameters():
            if name.endswith("bias"):  # zero otherwise
                p.copy_(torch.randn(p.shape, generator=g, device=gpu) * 0.1)
    if second:
        pipe.transformer_2 = dit.make_pipe(cfg, device=gpu, dtype=BF16, seed=6).transformer
    return pipe


def _inputs(cfg, gpu, batch, rows, seed=3):
    g = torch.Generator(device=gpu).manual_seed(seed)

    def draw(*shape, dtype=BF16):
        return torch.randn(shape, generator=g, device=gpu).to(dtype)

    return draw(batch, rows, cfg.dim), draw(batch, 7, cfg.dim), draw(batch, 6, cfg.dim, dtype=torch.float32) * 0.3


class Mix:
    """A processor of elementwise operations alone, whose gradients do not depend on the schedule."""

    def __call__(self, attn, hidden_states, encoder_hidden_states=None, attention_mask=None, rotary_emb=None,
                 timestep=None):
        if getattr(attn, "fused_projections", False):
            q, k, v = attn.to_qkv(hidden_states).chunk(3, dim=-1)
        else:
            ctx = hidden_states if encoder_hidden_states is None else encoder_hidden_states
            q, k, v = attn.to_q(hidden_states), attn.to_k(ctx), attn.to_v(ctx)
        return attn.to_out[1](attn.to_out[0](q * 0.5 + k[:, :1] - v[:, -1:]))


def _written_out(weights, x, ctx, temb, eps, linear, fused=False):
    """A block with :class:`Mix` from the operators: ``linear(x, w, b)`` (one for attn1's three projections if ``fused``),
    the norms of :mod:`svoo_amd.norm`."""
    from svoo_amd import norm

    w = weights
    shift, scale, gate, c_shift, c_scale, c_gate = (w["scale_shift_table"].float() + temb).chunk(6, dim=1)

    def lin(name, t):
        return linear(t, w[name + ".weight"], w[name + ".bias"])

    def attention(name, t, c):
        if fused and t is c:
            w3, b3 = (torch.cat([w[f"{name}.to_{n}.{p}"] for n in "qkv"]) for p in ("weight", "bias"))
            q, k, v = linear(t, w3, b3).chunk(3, dim=-1)
        else:
            q, k, v = (lin(f"{name}.to_{n}", s) for n, s in (("q", t), ("k", c), ("v", c)))
        return lin(name + ".to_out.0", q * 0.5 + k[:, :1] - v[:, -1:])

    n = norm.layer_norm(x, scale=scale, shift=shift, eps=eps)
    x = (x.float() + attention("attn1", n, n).float() * gate).to(x.dtype)
    n = norm.layer_norm(x, w["norm2.weight"], w["norm2.bias"], eps=eps)
    x = x + attention("attn2", n, ctx)
    n = norm.layer_norm(x, scale=c_scale, shift=c_shift, eps=eps)
    h = torch.nn.functional.gelu(lin("ffn.0", n), approximate="tanh")
    return x, n, h, lambda h: (x.float() + lin("ffn.2", h).float() * c_gate).to(x.dtype)


@pytest.mark.parametrize("batch,rows,heads,ffn", [(1, 1, 1, 512), (1, 300, 2, 520), (2, 33, 3, 1000)])
def test_block_for_inference(gpu, batch, rows, heads, ffn):
    from svoo_amd import fp8
    from svoo_amd.inference import replace_wan_linear

    say("block, 8-bit inference", batch, rows, heads, ffn)
    pipe = _pipe(gpu, 1, heads, ffn)
    block, cfg = pipe.transformer.blocks[0], pipe.transformer.config
    weights = {n: p.detach().clone() for n, p in block.named_parameters()}
    layers = replace_wan_linear(pipe)
    pipe.transformer.fuse_norms()
    assert len(layers) == 1 + 1 + 4 + 2 and all(isinstance(m, fp8.Fp8Linear) for m in layers)
    assert not any(type(m) is torch.nn.Linear for m in block.modules())
    assert block.attn1.fused_projections and not hasattr(block.attn1, "to_q")
    for a in (block.attn1, block.attn2):
        a.set_processor(Mix())
    x, ctx, temb = _inputs(cfg, gpu, batch, rows)

    def linear(t, w, b, act="none"):
        return fp8.fp8_matmul(*fp8.fp8_quantize_rows(t), *fp8.fp8_quantize_blocks(w), bias=b, activation=act,
                              out_dtype=t.dtype)

    with torch.no_grad():
        got = block(x, ctx, temb, None)
        _, n, _, end = _written_out(weights, x, ctx, temb, cfg.eps, linear, fused=True)
        want = end(linear(n, weights["ffn.0.weight"], weights["ffn.0.bias"], "gelu_tanh"))
        assert torch.equal(got, want)
        # without the fused norms the layers take 16-bit rows
        pipe.transformer.fuse_norms(False)
        assert block(x, ctx, temb, None).isfinite().all()
    with pytest.raises(RuntimeError, match="no backward pass"):
        pipe.transformer.fuse_norms()
        block(x, ctx, temb, None)


@pytest.mark.parametrize("batch,rows,grad_dtype", [(1, 300, torch.float8_e4m3fn), (2, 33, torch.float8_e5m2)])
def test_block_for_training(gpu, batch, rows, grad_dtype):
    from svoo_amd import fp8
    from svoo_amd.inference import replace_wan_linear

    say("block, 8-bit training", batch, rows, grad_dtype)
    pipe = _pipe(gpu, 1, 2, 520)
    model = pipe.transformer.train()
    block, cfg = model.blocks[0], model.config
    before = dict(block.named_parameters())
    layers = replace_wan_linear(pipe, trainable=True, grad_dtype=grad_dtype)
    assert len(layers) == 10 and all(type(m) is fp8.Fp8TrainLinear and m.training for m in layers)
    after = dict(block.named_parameters())
    assert before.keys() == after.keys() and all(after[n] is p for n, p in before.items())
    model.fuse_norms()
    for a in (block.attn1, block.attn2):
        a.set_processor(Mix())
    x, ctx, temb = _inputs(cfg, gpu, batch, rows)
    dy = torch.randn(x.shape, generator=torch.Generator(device=gpu).manual_seed(4), device=gpu).to(BF16)

    def run(f):
        leaves = [t.clone().requires_grad_() for t in (x, ctx, temb)]
        out = f(*leaves)
        used = [p for n, p in before.items() if "norm_" not in n]
        return (out, *torch.autograd.grad(out, [*leaves, *used], dy))

    def by_hand(a, c, t):
        _, _, h, end = _written_out(before, a, c, t, cfg.eps, lambda v, w, b: fp8.fp8_linear(v, w, b, grad_dtype))
        return end(h)

    got, want = run(lambda a, c, t: block(a, c, t, None)), run(by_hand)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(g.isfinite().all() and g.any() for g in got)


def test_training_steps_move_the_shared_parameters(gpu):
    """A few steps of an optimiser through the whole model: layers read their parameters anew at every call."""
    from svoo_amd import fp8
    from svoo_amd.inference import replace_wan_linear

    pipe = _pipe(gpu, 2, 1, 256)
    model = pipe.transformer.train().fuse_norms()
    replace_wan_linear(pipe, trainable=True)
    from svoo_amd import dit

    g = torch.Generator(device=gpu).manual_seed(1)
    lat = torch.randn(dit.latent_shape(model.config, 64, 64, 5), generator=g, device=gpu).to(BF16)
    txt = torch.randn(1, 9, 64, generator=g, device=gpu).to(BF16)
    t = torch.tensor([500.0], device=gpu)
    opt = torch.optim.SGD(model.parameters(), lr=1e-2)
    weight = model.blocks[0].ffn[0].weight
    outs = []
    for _ in range(3):
        before = weight.detach().clone()
        out = model(lat, t, txt)
        out.float().square().mean().backward()
        outs.append(out.detach())
        assert all(p.grad is not None and p.grad.isfinite().all() for p in model.parameters())
        opt.step()
        opt.zero_grad()
        assert not torch.equal(before, weight)
    assert not torch.equal(outs[0], outs[1]) and not torch.equal(outs[1], outs[2])
    x = torch.randn(3, weight.shape[1], generator=g, device=gpu).to(BF16)
    with torch.no_grad():
        layer = model.blocks[0].ffn[0]
        assert torch.equal(layer(x), fp8.fp8_linear(x, weight, layer.bias))


def test_pipeline_with_svoo_attention(gpu):
    """The sparse processors on the fused projections, both transformers, one graph of a whole block."""
    from svoo_amd import dit
    from svoo_amd.inference import replace_wan_attention, replace_wan_linear
    from svoo_amd.processor import WanAttn_SAPAttn_Processor

    pipe = _pipe(gpu, second=True)
    cls = type("P", (WanAttn_SAPAttn_Processor,), {})
    procs = replace_wan_attention(pipe, 256, 256, 9, first_layers_fp=0, first_times_fp=1e9, num_q_centroids=4,
                                  num_k_centroids=8, top_p_kmeans=0.9, min_kc_ratio=0.1, kmeans_iter_init=2,
                                  kmeans_iter_step=2, processor_cls=cls)
    assert len(replace_wan_linear(pipe)) == 2 * 2 * 8
    g = torch.Generator().manual_seed(0)
    lat = torch.randn(dit.latent_shape(pipe.transformer.config, 256, 256, 9), generator=g).to(gpu, BF16)
    txt = torch.randn(1, 16, 64, generator=g).to(gpu, BF16)
    with torch.no_grad():
        for model in (pipe.transformer, pipe.transformer_2):
            out = model.fuse_norms()(lat, torch.tensor([500.0], device=gpu), txt)
            assert out.shape == lat.shape and out.isfinite().all()
    assert all(p._last_call is not None for p in procs)  # the sparse path ran
    # a block with dense attention, captured: replays follow their inputs
    block = pipe.transformer.blocks[0]
    for a in (block.attn1, block.attn2):
        a.set_processor(Mix())
    x, ctx, temb = _inputs(pipe.transformer.config, gpu, 1, 200)
    with torch.no_grad():
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            for _ in range(2):
                block(x, ctx, temb, None)
        torch.cuda.current_stream().wait_stream(stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = block(x, ctx, temb, None)
        for seed in range(4):
            for t, new in zip((x, ctx, temb), _inputs(pipe.transformer.config, gpu, 1, 200, seed)):
                t.copy_(new)
            graph.replay()
            got = y.clone()
            assert torch.equal(got, block(x, ctx, temb, None))
            torch.cuda.synchronize()


def test_what_is_replaced(gpu):
    """Hooked and wrapped layers stay, a diffusers-like GELU projection is fused, another activation is not."""
    from types import SimpleNamespace

    from svoo_amd import fp8
    from svoo_amd.inference import replace_wan_linear

    nn = torch.nn

    class GELU(nn.Module):  # as diffusers names it
        def __init__(self, approximate):
            super().__init__()
            self.proj, self.approximate = nn.Linear(128, 256), approximate

        def forward(self, x):
            return nn.functional.gelu(self.proj(x), approximate=self.approximate)

    class Wrapped(nn.Linear):
        pass

    class Block(nn.Module):
        def __init__(self, net):
            super().__init__()
            self.attn1 = None
            self.ffn = nn.ModuleList(net)

    blocks = nn.ModuleList([Block([GELU("tanh"), nn.Linear(256, 128)]), Block([GELU("none"), Wrapped(256, 128)])])
    hooked = nn.Linear(256, 128)
    hooked.register_forward_hook(lambda *a: None)
    watched = GELU("tanh")  # its own call is waited for: only the layer inside may change
    watched.register_forward_pre_hook(lambda *a: None)
    blocks.append(Block([nn.Sequential(nn.Linear(128, 256), nn.GELU()), hooked, watched]))
    blocks.to(gpu, BF16)
    x = torch.randn(5, 128, generator=torch.Generator(device=gpu).manual_seed(2), device=gpu).to(BF16)
    first = blocks[0].ffn[0].proj
    layers = replace_wan_linear(SimpleNamespace(transformer=SimpleNamespace(blocks=blocks)))
    a, b, c = (block.ffn for block in blocks)
    assert isinstance(a[0], fp8.Fp8Linear) and a[0].activation == "gelu_tanh" and isinstance(a[1], fp8.Fp8Linear)
    assert type(b[0]) is GELU and isinstance(b[0].proj, fp8.Fp8Linear) and b[0].proj.activation == "none"
    assert type(b[1]) is Wrapped and c[1] is hooked
    assert isinstance(c[0][0], fp8.Fp8Linear) and c[0][0].activation == "none" and type(c[0][1]) is nn.GELU
    assert c[2] is watched and watched.proj.activation == "none"
    assert layers == [a[0], a[1], b[0].proj, c[0][0], watched.proj]
    assert replace_wan_linear(SimpleNamespace(transformer=SimpleNamespace(blocks=blocks))) == []  # nothing is left to do
    with torch.no_grad():
        want = fp8.fp8_matmul(*fp8.fp8_quantize_rows(x), *fp8.fp8_quantize_blocks(first.weight), bias=first.bias,
                              activation="gelu_tanh")
        assert torch.equal(a[0](x), want)


def test_hooks_on_the_ffn_are_called(gpu):
    """A hook on the FFN or on its first layer gets its call; the values are those of the layers one after the other."""
    from svoo_amd.inference import replace_wan_linear

    pipe = _pipe(gpu, 1, 1)
    replace_wan_linear(pipe)
    block = pipe.transformer.fuse_norms().blocks[0]
    for a in (block.attn1, block.attn2):
        a.set_processor(Mix())
    x, ctx, temb = _inputs(pipe.transformer.config, gpu, 1, 50)
    with torch.no_grad():
        want = block(x, ctx, temb, None)
        for module in (block.ffn, block.ffn[0]):
            seen = []
            handle = module.register_forward_hook(lambda m, args, out: seen.append(args[0].dtype))
            assert torch.equal(block(x, ctx, temb, None), want)  # quantised in the norm or behind it: the same values
            handle.remove()
            assert seen == [BF16]
