"""Training a Wan-shaped model on 8-bit linear layers beside the attention processors."""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _model(gpu, first_layers_fp=0):
    from svoo_amd import dit
    from svoo_amd.inference import replace_wan_attention, replace_wan_linear
    from svoo_amd.processor import WanAttn_SAPAttn_Processor

    cfg = dit.WanDiTConfig(num_attention_heads=1, ffn_dim=256, num_layers=2, text_dim=64)
    pipe = dit.make_pipe(cfg, device=gpu, dtype=BF16, seed=5)
    replace_wan_attention(pipe, 128, 128, 5, first_layers_fp=first_layers_fp, first_times_fp=1e9, num_q_centroids=2,
                          num_k_centroids=4, top_p_kmeans=0.9, min_kc_ratio=0.1, kmeans_iter_init=2, kmeans_iter_step=2,
                          processor_cls=type("P", (WanAttn_SAPAttn_Processor,), {}))
    replace_wan_linear(pipe, trainable=True)
    model = pipe.transformer.fuse_norms()
    g = torch.Generator().manual_seed(0)
    lat = torch.randn(dit.latent_shape(cfg, 128, 128, 5), generator=g).to(gpu, BF16)
    txt = torch.randn(1, 9, 64, generator=g).to(gpu, BF16)
    return lambda: model(lat, torch.tensor([500.0], device=gpu), txt), model


def test_sparse_attention_refuses_to_train(gpu):
    """Its kernels have no backward pass: the projections before it would get no gradient.  Evaluation runs."""
    step, _ = _model(gpu)
    with torch.no_grad():
        assert step().isfinite().all()
    with pytest.raises(RuntimeError, match="sparse attention has no backward pass"):
        step()


def test_dense_layers_of_the_sparse_processors_train(gpu):
    """Where the processors run dense attention, every parameter has its gradient."""
    step, model = _model(gpu, first_layers_fp=2)
    step().float().square().mean().backward()
    assert all(p.grad is not None and p.grad.isfinite().all() for p in model.parameters())
    assert all(getattr(b.attn1, n).weight.grad.any() for b in model.blocks for n in ("to_q", "to_k", "to_v"))
