"""What installing the training attention refuses in two transformers, without a GPU."""

import pytest
import torch


def _pipe(heads=2, dim=128, patch=(1, 2, 2)):
    from svoo_amd import dit

    cfg = dit.WanDiTConfig(num_attention_heads=heads, attention_head_dim=dim, patch_size=patch, ffn_dim=64, num_layers=2,
                           text_dim=32)
    return dit.make_pipe(cfg, dtype=torch.bfloat16)


def _attentions(pipe):
    return [a for t in (pipe.transformer, pipe.transformer_2) for b in t.blocks for a in (b.attn1, b.attn2)]


def _two(**second):
    pipe = _pipe()
    pipe.transformer_2 = _pipe(**second).transformer
    return pipe


@pytest.mark.parametrize("second,match", [(dict(dim=256, heads=1), "head dim 256"), (dict(patch=(1, 4, 4)), "patches of")])
def test_a_second_transformer_is_looked_at_before_the_first_change(second, match):
    from svoo_amd.inference import replace_wan_attention_trainable

    pipe = _two(**second)
    before = [a.processor for a in _attentions(pipe)]
    with pytest.raises(ValueError, match=match):
        replace_wan_attention_trainable(pipe, 64, 96, 9)
    assert [a.processor for a in _attentions(pipe)] == before


def test_an_attention_that_takes_no_processor_is_refused_before_the_first_change():
    from svoo_amd.inference import replace_wan_attention_trainable

    class Plain(torch.nn.Module):
        pass

    pipe = _two()
    pipe.transformer_2.blocks[1].attn2 = Plain()
    others = _attentions(pipe)[:-1]
    before = [a.processor for a in others]
    with pytest.raises(ValueError, match="set_processor"):
        replace_wan_attention_trainable(pipe, 64, 96, 9)
    assert [a.processor for a in others] == before


def test_each_transformer_has_the_axes_of_its_heads():
    from svoo_amd.inference import replace_wan_attention_trainable

    pipe = _two(dim=64)
    got = replace_wan_attention_trainable(pipe, 64, 96, 9)
    assert [p.axes for p in got] == [(44, 42, 42)] * 4 + [(24, 20, 20)] * 4 and all(p.grid == (3, 4, 6) for p in got)


def test_fp32_projections_are_refused_at_the_call(monkeypatch):
    from svoo_amd import _lib, dit
    from svoo_amd.inference import replace_wan_attention_trainable

    monkeypatch.setattr(_lib, "launch", lambda *a: None)
    monkeypatch.setattr(_lib, "require_gpu_tensor", lambda t, name: None)
    cfg = dit.WanDiTConfig(num_attention_heads=2, ffn_dim=64, num_layers=1, text_dim=32)
    pipe = dit.make_pipe(cfg, dtype=torch.float32)
    replace_wan_attention_trainable(pipe, 64, 96, 9)
    x = torch.zeros(1, 72, cfg.dim)
    attn = pipe.transformer.blocks[0].attn1
    with torch.no_grad(), pytest.raises(TypeError, match="bfloat16 or float16"):
        attn(x, rotary_emb=dit.rope_tables(cfg, 3, 4, 6, "cpu"))
    with torch.no_grad(), torch.autocast("cpu", torch.bfloat16):
        assert attn(x, rotary_emb=dit.rope_tables(cfg, 3, 4, 6, "cpu")).dtype == torch.bfloat16


def test_the_rotary_base_is_the_configurations():
    from types import SimpleNamespace

    from svoo_amd import dit
    from svoo_amd.inference import replace_wan_attention_trainable

    cfg = dit.WanDiTConfig(num_attention_heads=2, ffn_dim=64, num_layers=1, text_dim=32, rope_theta=500.0)
    pipe = dit.make_pipe(cfg, dtype=torch.bfloat16)
    pipe.transformer_2 = _pipe().transformer
    assert [p.theta for p in replace_wan_attention_trainable(pipe, 64, 96, 9)] == [500.0] * 2 + [10000.0] * 4
    assert {p.theta for p in replace_wan_attention_trainable(pipe, 64, 96, 9, theta=7.0)} == {7.0}
    pipe.transformer_2 = None
    # a configuration that names no base
    pipe.transformer.config = SimpleNamespace(patch_size=cfg.patch_size, attention_head_dim=cfg.attention_head_dim)
    assert {p.theta for p in replace_wan_attention_trainable(pipe, 64, 96, 9)} == {10000.0}
