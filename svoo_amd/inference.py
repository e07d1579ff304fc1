"""Install the SVOO attention processors into a Wan or HunyuanVideo pipeline (the reference's configuration surface).

``replace_wan_attention`` follows ``svoo/models/wan/inference.py:23-440`` (the SAP, EAR and dense
patterns): it derives the token geometry from the pipeline, writes the configuration as class
attributes of the pattern's processor class (shared by every layer, as in the reference) and
registers one processor instance per transformer block (``transformer_2`` too, for Wan2.2).  The pipeline is
duck-typed: ``pipe.transformer.blocks[i].attn1.set_processor``, ``pipe.transformer.config``
(``patch_size``, ``num_attention_heads``, ``attention_head_dim``) and ``pipe.vae_scale_factor_*``.
No kernel warm-up is needed: the HIP kernels are compiled ahead of time.

``replace_hunyuan_attention`` (also under the reference's name ``replace_hunyuan10_attention``) does
the same for HunyuanVideo 1.0 (``svoo/models/hunyuan10/inference.py:31-231``): one
:class:`Hunyuan_SAPAttn_Processor` per double-stream block (layers ``0 .. D-1``), then per
single-stream block (layers ``D ..``), the numbering the per-layer profile CSV is indexed by.

``replace_wan_linear`` puts 8-bit linear layers into the blocks of a Wan pipeline; it has no counterpart in the reference.
"""

from __future__ import annotations

import os

import torch

from . import _lib
from .fp8 import Fp8Linear, Fp8TrainLinear
from .processor import (Hunyuan_SAPAttn_Processor, WanAttn_DenseAttn_Processor, WanAttn_EARAttn_Processor,
                        WanAttn_SAPAttn_Processor)
from .sparsity import SparsityLookup
from .sparsity.exact import resume_requested


def wan_token_geometry(pipe, height: int, width: int, num_frames: int):
    """``(num_frame_patches, frame_patches_one_frame)`` of a Wan pipeline (``inference.py:81-83``)."""
    patch = pipe.transformer.config.patch_size
    num_frame_patches = 1 + num_frames // (pipe.vae_scale_factor_temporal * patch[0])
    mod_value = pipe.vae_scale_factor_spatial * patch[1]
    frame_patches_one_frame = int(height // mod_value) * int(width // mod_value)
    return num_frame_patches, frame_patches_one_frame


def replace_wan_attention(
    pipe,
    height,
    width,
    num_frames,
    first_layers_fp,
    first_times_fp,
    num_inference_steps=None,
    attention_backend="flexattn",
    pattern="SAP",
    num_q_centroids=None,
    num_k_centroids=None,
    top_p_kmeans=None,
    min_kc_ratio=0,
    max_kc_ratio=0,
    ear_gamma=1.0,
    kmeans_iter_init=0,
    kmeans_iter_step=0,
    zero_step_kmeans_init=False,
    use_global_constraints=False,
    use_routing_transformer_strategy=False,
    use_svoo=True,
    start_reuse_step=None,
    reuse_interval=1,
    use_dynamic_min_kc_ratio=False,
    sparsity_csv_path=None,
    dynamic_min_kc_ratio_min=None,
    dynamic_min_kc_ratio_max=None,
    measure_attention_sparsity=False,
    sparsity_output_file="attention_sparsity.txt",
    sparsity_batch_size=0,
    sparsity_query_samples=0,
    sparsity_threshold=0.95,
    sparsity_start_step=1,
    processor_cls=None,
    **unused,
):
    """Configure SVOO attention and install one processor per Wan DiT block.

    Arguments keep the reference's names and meaning (``svoo/models/wan/inference.py:23-74``);
    ``first_layers_fp`` is a layer count and ``first_times_fp`` a timestep threshold, as the CLI
    passes them.  ``max_kc_ratio`` is forwarded to the SAP mask (EAR has no cap).  Patterns:
    ``"SAP"`` (:class:`WanAttn_SAPAttn_Processor`), ``"EAR"`` (:class:`WanAttn_EARAttn_Processor`, with
    ``ear_gamma``) and the ``"dense"`` diagnostic (:class:`WanAttn_DenseAttn_Processor`: dense attention,
    used to record sparsity profiles); anything else, or ``use_svoo=False``, raises ``ValueError`` as the
    reference does (``:77-78``), and the global-constraint / routing variants raise
    ``NotImplementedError``.  ``processor_cls`` overrides the pattern's class (a subclass keeps the
    configuration local to it).  A missing or unreadable profile CSV disables the dynamic ratios
    (``:308-320``).  With ``measure_attention_sparsity`` every processor also appends the exact per-head
    sparsity of each (layer, step) to ``sparsity_output_file`` (the offline profile producer).  Returns the
    processors.
    """
    if pattern not in ("SAP", "EAR", "dense") or not use_svoo:
        raise ValueError("Only SVOO, EAR and dense diagnostic patterns are supported in this release.")
    if use_global_constraints or use_routing_transformer_strategy:
        raise NotImplementedError("global-constraint and routing-transformer variants are not built here")
    num_frame_patches, frame_patches_one_frame = wan_token_geometry(pipe, height, width, num_frames)
    blocks = pipe.transformer.blocks
    num_layers = len(blocks)

    cls = processor_cls or {"SAP": WanAttn_SAPAttn_Processor, "EAR": WanAttn_EARAttn_Processor,
                            "dense": WanAttn_DenseAttn_Processor}[pattern]
    if pattern != "dense":
        cls.use_ear = pattern == "EAR"  # inference.py:282
        cls.ear_gamma = ear_gamma
    cls.first_layers_fp = first_layers_fp
    cls.first_times_fp = first_times_fp
    cls.context_length = 0
    cls.num_frame = num_frame_patches
    cls.frame_size = frame_patches_one_frame
    cls.num_q_centroids = num_q_centroids
    cls.num_k_centroids = num_k_centroids
    cls.top_p_kmeans = top_p_kmeans
    cls.min_kc_ratio = min_kc_ratio
    cls.max_kc_ratio = max_kc_ratio
    cls.num_layers = num_layers
    cls.kmeans_iter_init = kmeans_iter_init
    cls.kmeans_iter_step = kmeans_iter_step
    cls.zero_step_kmeans_init = zero_step_kmeans_init
    cls.use_svoo = True
    cls.start_reuse_step = start_reuse_step
    cls.reuse_interval = reuse_interval
    cls.use_dynamic_min_kc_ratio = False
    cls.sparsity_lookup = None
    # a fresh step counter for this pipeline (the class-level state the processors share)
    cls._current_internal_timestep = None
    cls._inference_step_counter = 0
    cls._seen_timesteps = set()
    if use_dynamic_min_kc_ratio and sparsity_csv_path:
        try:
            cls.sparsity_lookup = SparsityLookup(sparsity_csv_path)
            cls.use_dynamic_min_kc_ratio = True
            cls.dynamic_min_kc_ratio_min = dynamic_min_kc_ratio_min
            cls.dynamic_min_kc_ratio_max = dynamic_min_kc_ratio_max
        except Exception:  # the reference silently falls back to the scalar ratio
            cls.use_dynamic_min_kc_ratio = False
            cls.sparsity_lookup = None

    # offline profiling (inference.py:322-341): a fresh raw log unless SVOO_SPARSITY_RESUME keeps it
    cls.measure_attention_sparsity = measure_attention_sparsity
    cls.sparsity_output_file = sparsity_output_file
    cls.sparsity_batch_size = sparsity_batch_size
    cls.sparsity_query_samples = sparsity_query_samples
    cls.sparsity_threshold = sparsity_threshold
    cls.sparsity_start_step = sparsity_start_step
    if measure_attention_sparsity and sparsity_output_file:
        d = os.path.dirname(sparsity_output_file)
        if d:
            os.makedirs(d, exist_ok=True)
        if not resume_requested():
            open(sparsity_output_file, "w", encoding="utf-8").close()

    processors = []
    for transformer in (pipe.transformer, getattr(pipe, "transformer_2", None)):
        if transformer is None:
            continue
        for layer_idx, block in enumerate(transformer.blocks):
            if hasattr(block.attn1, "set_processor"):
                proc = cls(layer_idx=layer_idx)
                proc.num_layers = num_layers
                block.attn1.set_processor(proc)
                processors.append(proc)
    return processors


def _unwatched(m) -> bool:
    """No hook waits for a call of the module, and its ``forward`` is its class's."""
    return not (m._forward_hooks or m._forward_pre_hooks or m._backward_hooks or m._backward_pre_hooks
                or "forward" in m.__dict__)


def _plain_linear(m) -> bool:
    """A ``torch.nn.Linear`` that nothing wraps or watches."""
    return type(m) is torch.nn.Linear and _unwatched(m)


def _tanh_gelu(m) -> bool:
    return type(m) is torch.nn.GELU and m.approximate == "tanh" and _unwatched(m)


def replace_wan_linear(pipe, trainable: bool = False, grad_dtype=torch.float8_e4m3fn):
    """Put 8-bit linear layers into every block of a Wan pipeline's transformers (``transformer_2`` too).

    Every plain ``torch.nn.Linear`` of a block's ``attn1``, ``attn2`` and ``ffn`` is replaced; embedders, modulation and
    the head stay as they are, as do layers that something else wraps or hooks.  For inference
    (:class:`svoo_amd.fp8.Fp8Linear`) the weight is laid out in 8 bits once and its original released, the query, key and
    value projections of ``attn1`` become one ``to_qkv`` (``fused_projections``, which the processors here and in
    diffusers know), and a tanh GELU behind the first ``ffn`` layer enters that layer's product.  With ``trainable``
    (:class:`svoo_amd.fp8.Fp8TrainLinear`) layers share the parameters of those they replace and have gradients, the
    incoming ones in ``grad_dtype``.  Weights have to be on the GPU.  Returns the new layers."""
    transformers = [t for t in (pipe.transformer, getattr(pipe, "transformer_2", None)) if t is not None]
    parts = [part for t in transformers for block in t.blocks
             for part in (getattr(block, n, None) for n in ("attn1", "attn2", "ffn")) if part is not None]
    for part in parts:  # before the first layer changes
        for m in part.modules():
            if _plain_linear(m):
                _lib.elem_type(m.weight, "weight")
                if m.bias is not None:
                    _lib.elem_type(m.bias, "bias")
                if 0 in m.weight.shape:
                    raise ValueError(f"replace_wan_linear: a layer of shape {tuple(m.weight.shape)}")
    layers = []

    def convert(linear, activation="none"):
        new = Fp8TrainLinear.from_linear(linear, grad_dtype) if trainable else Fp8Linear.from_linear(linear, activation)
        layers.append(new)
        return new

    def walk(parent):
        kids = list(parent.named_children())
        for i, (name, m) in enumerate(kids):
            if _plain_linear(m):
                fuse = not trainable and isinstance(parent, torch.nn.Sequential) and i + 1 < len(kids) and \
                    _tanh_gelu(kids[i + 1][1])
                setattr(parent, name, convert(m, "gelu_tanh" if fuse else "none"))
                if fuse:
                    setattr(parent, kids[i + 1][0], torch.nn.Identity())
            elif type(m).__name__ == "GELU" and getattr(m, "approximate", None) == "tanh" and not trainable and \
                    _unwatched(m) and _plain_linear(getattr(m, "proj", None)):  # diffusers' projection with its GELU
                setattr(parent, name, convert(m.proj, "gelu_tanh"))
            else:
                walk(m)

    with torch.no_grad():
        for t in transformers:
            for block in t.blocks:
                attn = getattr(block, "attn1", None)
                qkv = [getattr(attn, n, None) for n in ("to_q", "to_k", "to_v")]
                if not trainable and all(_plain_linear(m) for m in qkv) and not getattr(attn, "fused_projections", False) \
                        and len({(m.in_features, m.weight.dtype, m.bias is None) for m in qkv}) == 1:
                    bias = None if qkv[0].bias is None else torch.cat([m.bias for m in qkv])
                    attn.to_qkv = Fp8Linear(torch.cat([m.weight for m in qkv]), bias)
                    attn.fused_projections = True
                    layers.append(attn.to_qkv)
                    del attn.to_q, attn.to_k, attn.to_v
        for part in parts:
            walk(part)
    return layers


def _configure_profile(cls, use_dynamic_min_kc_ratio, sparsity_csv_path, dynamic_min_kc_ratio_min,
                       dynamic_min_kc_ratio_max) -> None:
    """Per-head ratios from a profile CSV; a missing or unreadable CSV leaves the scalar ratio in force."""
    cls.use_dynamic_min_kc_ratio = False
    cls.sparsity_lookup = None
    cls.dynamic_min_kc_ratio_min = None
    cls.dynamic_min_kc_ratio_max = None
    if use_dynamic_min_kc_ratio and sparsity_csv_path:
        try:
            cls.sparsity_lookup = SparsityLookup(sparsity_csv_path)
        except Exception:
            return
        cls.use_dynamic_min_kc_ratio = True
        cls.dynamic_min_kc_ratio_min = dynamic_min_kc_ratio_min
        cls.dynamic_min_kc_ratio_max = dynamic_min_kc_ratio_max


def replace_hunyuan_attention(
    pipe,
    height,
    width,
    num_frames,
    prompt_length,
    first_layers_fp,
    first_times_fp,
    pattern="SAP",
    num_q_centroids=None,
    num_k_centroids=None,
    top_p_kmeans=None,
    min_kc_ratio=0,
    max_kc_ratio=0,
    kmeans_iter_init=0,
    kmeans_iter_step=0,
    zero_step_kmeans_init=False,
    context_length=256,
    use_svoo=True,
    start_reuse_step=None,
    reuse_interval=1,
    use_dynamic_min_kc_ratio=False,
    sparsity_csv_path=None,
    dynamic_min_kc_ratio_min=None,
    dynamic_min_kc_ratio_max=None,
    measure_attention_sparsity=False,
    sparsity_output_file="attention_sparsity.txt",
    sparsity_batch_size=0,
    sparsity_query_samples=0,
    sparsity_threshold=0.95,
    sparsity_start_step=1,
    processor_cls=None,
    **unused,
):
    """Configure SVOO attention and install one processor per HunyuanVideo 1.0 transformer block.

    Arguments keep the names and meaning of ``replace_hunyuan10_attention``
    (``svoo/models/hunyuan10/inference.py:31-65``).  The token geometry is HunyuanVideo's: ``1 +
    num_frames // 4`` latent frames of ``height * width // 256`` patches, and 256 text tokens (the
    reference fixes the text length at 256 whatever ``context_length`` says, ``:68-70``; so does this
    function).  Only the SAP pattern with ``use_svoo`` exists for HunyuanVideo (``:66-67``); anything
    else raises ``ValueError``.  ``prompt_length`` (the valid text tokens) must lie in ``[0, 256]``.

    Processors go to ``block.attn.processor`` of every ``pipe.transformer.transformer_blocks`` entry
    (double stream, layers ``0 .. D-1``) and then of every ``single_transformer_blocks`` entry (layers
    ``D + i``, ``:207-231``).  The blocks must pass ``timestep`` to their attention, as the reference's
    patched block forwards do (``custom_models.py:383-390``; the pipeline side is not part of this
    package).  ``processor_cls`` overrides the class (a subclass keeps the configuration local).
    Returns the processors in layer order.
    """
    if pattern != "SAP" or not use_svoo:
        raise ValueError("Only SVOO (pattern='SAP') is supported for HunyuanVideo in this release.")
    context_length = 256
    if not 0 <= int(prompt_length) <= context_length:
        raise ValueError(f"prompt_length={prompt_length} must lie in [0, {context_length}]")
    tr = pipe.transformer
    double = list(tr.transformer_blocks)
    single = list(getattr(tr, "single_transformer_blocks", []))

    cls = processor_cls or Hunyuan_SAPAttn_Processor
    cls.first_layers_fp = first_layers_fp
    cls.first_times_fp = first_times_fp
    cls.prompt_length = int(prompt_length)
    cls.context_length = context_length
    cls.num_frame = 1 + num_frames // 4
    cls.frame_size = height * width // 256
    cls.num_layers = len(double) + len(single)
    cls.num_q_centroids = num_q_centroids
    cls.num_k_centroids = num_k_centroids
    cls.top_p_kmeans = top_p_kmeans
    cls.min_kc_ratio = min_kc_ratio
    cls.max_kc_ratio = max_kc_ratio
    cls.kmeans_iter_init = kmeans_iter_init
    cls.kmeans_iter_step = kmeans_iter_step
    cls.zero_step_kmeans_init = zero_step_kmeans_init
    cls.use_svoo = True
    cls.start_reuse_step = start_reuse_step
    cls.reuse_interval = 1 if reuse_interval is None else max(1, int(reuse_interval))
    _configure_profile(cls, use_dynamic_min_kc_ratio, sparsity_csv_path, dynamic_min_kc_ratio_min,
                       dynamic_min_kc_ratio_max)
    cls.measure_attention_sparsity = measure_attention_sparsity
    cls.sparsity_output_file = sparsity_output_file
    cls.sparsity_batch_size = sparsity_batch_size
    cls.sparsity_query_samples = sparsity_query_samples
    cls.sparsity_threshold = sparsity_threshold
    cls.sparsity_start_step = sparsity_start_step

    processors = []
    for layer_idx, block in enumerate(double + single):
        proc = cls(layer_idx=layer_idx)
        proc.num_layers = cls.num_layers
        block.attn.processor = proc
        processors.append(proc)
    return processors


replace_hunyuan10_attention = replace_hunyuan_attention
