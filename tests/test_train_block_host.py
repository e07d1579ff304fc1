"""The training attention processor and the fused residuals in a Wan block, without a GPU."""

import pytest
import torch


@pytest.fixture
def launches(monkeypatch):
    from svoo_amd import _lib

    seen = []
    monkeypatch.setattr(_lib, "launch", lambda device, name, *args: seen.append((name, args)))
    monkeypatch.setattr(_lib, "require_gpu_tensor", lambda t, name: None)
    return seen


def _pipe(dtype=torch.bfloat16, heads=2, layers=2):
    from svoo_amd import dit

    cfg = dit.WanDiTConfig(num_attention_heads=heads, ffn_dim=64, num_layers=layers, text_dim=32)
    return dit.make_pipe(cfg, dtype=dtype), cfg


def test_installed_in_both_attentions_with_the_clips_grid():
    from svoo_amd.inference import replace_wan_attention_trainable
    from svoo_amd.processor import WanAttn_TrainAttn_Processor

    pipe, _ = _pipe()
    got = replace_wan_attention_trainable(pipe, 64, 96, 9)
    assert len(got) == 4 and all(type(p) is WanAttn_TrainAttn_Processor for p in got)
    assert all(p.grid == (3, 4, 6) and p.axes == (44, 42, 42) and p.theta == 10000.0 for p in got)
    assert [b.attn1.processor for b in pipe.transformer.blocks] == got[::2]
    assert [b.attn2.processor for b in pipe.transformer.blocks] == got[1::2]


def test_an_image_branch_and_wide_heads_are_refused_before_the_first_change():
    from svoo_amd.inference import replace_wan_attention_trainable

    pipe, cfg = _pipe()
    pipe.transformer.blocks[1].attn2.add_k_proj = torch.nn.Linear(4, 4)
    before = [a.processor for b in pipe.transformer.blocks for a in (b.attn1, b.attn2)]
    with pytest.raises(ValueError, match="image branch"):
        replace_wan_attention_trainable(pipe, 64, 96, 9)
    pipe.transformer.blocks[1].attn2.add_k_proj = None
    cfg.attention_head_dim = 256
    with pytest.raises(ValueError, match="head dim 256"):
        replace_wan_attention_trainable(pipe, 64, 96, 9)
    assert [a.processor for b in pipe.transformer.blocks for a in (b.attn1, b.attn2)] == before


def test_launches_of_a_block(launches):
    """One launch a norm with its rotation, one an attention, one a residual with its norm."""
    from svoo_amd import dit
    from svoo_amd.inference import replace_wan_attention_trainable

    pipe, cfg = _pipe(layers=1)
    replace_wan_attention_trainable(pipe, 64, 96, 9)
    pipe.transformer.fuse_norms(residuals=True)
    block = pipe.transformer.blocks[0]
    x, ctx, temb = (torch.randn(1, n, cfg.dim).bfloat16() for n in (72, 5, 6))
    with torch.no_grad():
        block(x, ctx, temb, dit.rope_tables(cfg, 3, 4, 6, "cpu"))
    assert [n for n, _ in launches] == [
        "svoo_layer_norm_fwd", "svoo_axis_rope_fwd", "svoo_axis_rope_fwd", "svoo_dense_attention_fwd", "svoo_residual_norm_fwd",
        "svoo_axis_rope_fwd", "svoo_axis_rope_fwd", "svoo_dense_attention_fwd", "svoo_residual_norm_fwd", "svoo_residual_norm_fwd"]
    launches.clear()
    pipe.transformer.fuse_norms()
    with torch.no_grad():
        block(x, ctx, temb, dit.rope_tables(cfg, 3, 4, 6, "cpu"))
    assert "svoo_residual_norm_fwd" not in [n for n, _ in launches]
    assert not pipe.transformer.fuse_norms(False, residuals=True).blocks[0].fused_residuals


def test_tokens_of_another_clip_masks_and_image_branches_are_refused(launches):
    from svoo_amd import dit
    from svoo_amd.inference import replace_wan_attention_trainable

    pipe, cfg = _pipe(layers=1)
    replace_wan_attention_trainable(pipe, 64, 96, 9)
    attn = pipe.transformer.blocks[0].attn1
    x = torch.zeros(1, 71, cfg.dim).bfloat16()
    with pytest.raises(ValueError, match="71 tokens for a grid"):
        attn(x, rotary_emb=dit.rope_tables(cfg, 1, 71, 1, "cpu"))
    with pytest.raises(ValueError, match="no attention mask"):
        attn(x, attention_mask=torch.ones(1, 1, 71, 71, dtype=torch.bool))
    attn.add_k_proj = torch.nn.Linear(4, 4)
    with pytest.raises(ValueError, match="image branch"):
        attn(x)
    assert not launches


def test_norms_that_something_watches_are_called(launches):
    from svoo_amd import dit
    from svoo_amd.inference import replace_wan_attention_trainable

    pipe, cfg = _pipe(layers=1)
    replace_wan_attention_trainable(pipe, 64, 96, 9)
    attn = pipe.transformer.blocks[0].attn1
    x, seen = torch.randn(1, 72, cfg.dim).bfloat16(), []
    rope = dit.rope_tables(cfg, 3, 4, 6, "cpu")

    def norms():
        launches.clear()
        with torch.no_grad():
            attn(x, rotary_emb=rope)
        return [args[9] for n, args in launches if n == "svoo_axis_rope_fwd"]

    assert norms() == [1, 1]
    handle = attn.norm_q.register_forward_hook(lambda *a: seen.append("hook"))
    assert norms() == [0, 1] and seen == ["hook"]
    handle.remove()
    forward = attn.norm_k.forward
    attn.norm_k.forward = lambda t: (seen.append("forward"), forward(t))[1]
    assert norms() == [1, 0] and seen[-1] == "forward"
    del attn.norm_k.forward
    handle = torch.nn.modules.module.register_module_forward_hook(lambda m, a, o: seen.append(m))
    try:
        assert norms() == [0, 0] and attn.norm_q in seen
    finally:
        handle.remove()
    attn.norm_q = None
    assert norms() == [0, 1]


def test_traced_and_with_tangents_as_tensor_operations(launches):
    """Tracing and forward-mode AD see tensor operations that give what the dense processor gives."""
    import torch.autograd.forward_ad as fwd

    from svoo_amd import dit
    from svoo_amd.inference import replace_wan_attention_trainable

    pipe, cfg = _pipe(torch.float32, layers=1)
    block = pipe.transformer.blocks[0].requires_grad_(False)
    rope = dit.rope_tables(cfg, 3, 4, 6, "cpu")
    x, ctx, temb = (torch.randn(1, n, cfg.dim) for n in (72, 5, 6))

    def run(x):
        return block(x, ctx, temb, rope)

    with torch.no_grad():
        want = run(x)
        replace_wan_attention_trainable(pipe, 64, 96, 9)
        pipe.transformer.fuse_norms(residuals=True)
        assert torch.allclose(torch.jit.trace(run, (x,), check_trace=False)(x), want, rtol=0, atol=2e-5)
        with fwd.dual_level():
            out = fwd.unpack_dual(run(fwd.make_dual(x, torch.ones_like(x))))
            assert torch.allclose(out.primal, want, rtol=0, atol=2e-5) and out.tangent is not None
    assert not launches
