"""What the layer norm and the 8-bit operators hand to their C entries: the arguments and buffers of each launch, recorded
on the CPU in place of the launch itself."""

import pytest
import torch


@pytest.fixture
def launches(monkeypatch):
    from svoo_amd import _lib

    seen = []
    monkeypatch.setattr(_lib, "launch", lambda device, name, *args: seen.append((name, args)))
    monkeypatch.setattr(_lib, "require_gpu_tensor", lambda t, name: None)
    return seen


# dict(zip(..)) of svoo_layer_norm_bwd's arguments
BWD = ("x", "x_type", "x_batch", "x_row", "dy", "dy_type", "dy_batch", "dy_row", "w", "w_type", "w_batch", "modulated", "mean",
       "rstd", "batch", "rows", "cols", "dx", "dw", "dw_type", "db", "db_type", "ws", "ws_bytes")
ELEM_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def _params(batch, cols, kind, dtype=torch.float32):
    """A parameter of a layer norm of x ``[batch, .., cols]``."""
    if kind is None:
        return None
    p = torch.randn(cols).to(dtype)
    return {"shared": p, "expanded": p.expand(batch, 1, cols), "expanded2": p.expand(batch, cols),
            "own": torch.randn(batch, 1, cols).to(dtype), "rows": torch.randn(batch, cols).to(dtype)}[kind]


@pytest.mark.parametrize("kinds", [("expanded", "expanded"), ("expanded2", "expanded2"), ("expanded", None), (None, "expanded"),
                                   ("expanded", "shared"), ("expanded2", "own"), ("own", "expanded"), ("shared", "expanded2"),
                                   ("own", "rows"), ("shared", "shared"), ("shared", "own")])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradients_of_every_parameter_form_are_written_whole(launches, kinds, dtype):
    """A parameter with a row per batch entry has its gradient written for each entry, also where the entries share memory:
    the launch covers as many entries as the buffer holds, and the gradient has the parameter's shape and type."""
    from svoo_amd import norm

    batch, rows, cols = 3, 5, 16
    x = torch.randn(batch, rows, cols)
    st = torch.zeros(batch, rows)
    names = ("scale", "shift")
    p = dict(zip(names, (_params(batch, cols, k, dtype) for k in kinds)))
    dx, *grads = norm.layer_norm_bwd(x, x, st, st, **p)
    name, args = launches[0]
    a = dict(zip(BWD, args))
    assert name == "svoo_layer_norm_bwd" and a["batch"] * a["rows"] == batch * rows and a["cols"] == cols
    per_entry = [k is not None and k != "shared" for k in kinds]
    assert a["batch"] == (batch if any(per_entry) else 1)
    assert a["x_batch"] == a["rows"] * cols and a["x_row"] == cols
    assert a["w_batch"] == (0 if kinds[0] in (None, "shared", "expanded", "expanded2") else cols)
    for i, key in enumerate(("dw", "db")):
        param, grad = p[names[i]], grads[i]
        if param is None:
            assert grad is None and a[key] is None
            continue
        assert grad.shape == param.shape and grad.dtype == param.dtype
        if per_entry[i] or a["batch"] == 1:  # written by the launch itself: as many elements as there are
            assert a[key] == grad.data_ptr() and a["batch"] * cols == grad.numel()
            assert a[key + "_type"] == ELEM_TYPES[dtype]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sums_over_the_batch_are_launches_too(launches, dtype):
    """The gradient of a parameter shared by the entries, beside one that is not: a second launch adds the entries' sums, in
    the parameter's type, and no tensor operation (whose scratch a captured graph would clear by a memset)."""
    from torch.utils._python_dispatch import TorchDispatchMode

    from svoo_amd import norm

    class Ops(TorchDispatchMode):
        seen = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.seen.append(func.overloadpacket.__name__)
            return func(*args, **(kwargs or {}))

    x, st = torch.randn(6, 5, 16), torch.zeros(6, 5)
    sc, sh = _params(6, 16, "own"), _params(6, 16, "shared", dtype)
    with Ops() as ops:
        _, dsc, dsh = norm.layer_norm_bwd(x, x, st, st, scale=sc, shift=sh)
    first, second = (dict(zip(BWD, args)) for _, args in launches)
    assert first["batch"] == 6 and first["dw"] == dsc.data_ptr() and first["db_type"] == 2
    assert second["dy"] == first["db"] and (second["batch"], second["rows"], second["cols"]) == (1, 6, 16)
    assert (second["dy_type"], second["dy_row"]) == (2, 16) and second["dx"] is None and second["dw"] is None
    assert second["db"] == dsh.data_ptr() and second["db_type"] == ELEM_TYPES[dtype]
    assert dsh.shape == (16,) and dsh.dtype == dtype and dsc.shape == (6, 1, 16)
    assert "sum" not in ops.seen


def test_forward_reads_expanded_parameters_as_shared_ones(launches):
    """No split by batch entries where none is needed: one batch of all rows."""
    from svoo_amd import norm

    x = torch.randn(4, 7, 16)
    norm.layer_norm(x, scale=_params(4, 16, "expanded"), shift=_params(4, 16, "expanded2"))
    norm.layer_norm_bwd(x, x, torch.zeros(4, 7), torch.zeros(4, 7), scale=_params(4, 16, "expanded"),
                        needs=(True, False, False))
    (_, fwd), (_, bwd) = launches
    assert fwd[12:15] == (1, 28, 16)
    assert dict(zip(BWD, bwd))["batch"] == 1


# ------------------------------------------------------------------------------------------------ records and tangents
def _operators():
    """Every operator as a function of one matrix, by name."""
    from svoo_amd import fp8, norm

    w, st = torch.randn(128, 128), torch.zeros(4)
    a, b = fp8.fp8_quantize_rows(w), fp8.fp8_quantize_blocks(w)
    train = fp8.Fp8TrainLinear(128, 128)
    return {
        "layer_norm": lambda x: norm.layer_norm(x), "layer_norm of a scale": lambda x: norm.layer_norm(w[:4], scale=x),
        "layer_norm_fwd": lambda x: norm.layer_norm_fwd(x)[0], "layer_norm_fp8": lambda x: norm.layer_norm_fp8(x)[0],
        "layer_norm_bwd": lambda x: norm.layer_norm_bwd(x, w[:4], st, st)[0],
        "layer_norm_bwd of x": lambda x: norm.layer_norm_bwd(w[:4], x, st, st)[0],
        "fp8_quantize_rows": lambda x: fp8.fp8_quantize_rows(x)[0],
        "fp8_quantize_blocks": lambda x: fp8.fp8_quantize_blocks(x)[0],
        "fp8_quantize_both": lambda x: fp8.fp8_quantize_both(x)[0],
        "fp8_linear": lambda x: fp8.fp8_linear(x, w), "fp8_linear of a weight": lambda x: fp8.fp8_linear(w, x),
        "Fp8TrainLinear": train, "Fp8Linear": fp8.Fp8Linear(w),
        "fp8_matmul of a bias": lambda x: fp8.fp8_matmul(*a, *b, x[0]),
    }


NAMES = ["layer_norm", "layer_norm of a scale", "layer_norm_fwd", "layer_norm_fp8", "layer_norm_bwd", "layer_norm_bwd of x",
         "fp8_quantize_rows", "fp8_quantize_blocks", "fp8_quantize_both", "fp8_linear", "fp8_linear of a weight",
         "Fp8TrainLinear", "Fp8Linear", "fp8_matmul of a bias"]


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("grad", [False, True])
def test_tangents_are_refused(launches, name, grad):
    """A tensor with a tangent would come out without one; in the same level, tensors without tangents are taken."""
    import torch.autograd.forward_ad as fwd

    with torch.set_grad_enabled(grad):
        f = _operators()[name]
        x = torch.randn(4, 128)
        launches.clear()
        with fwd.dual_level():
            with pytest.raises(RuntimeError, match="forward-mode"):
                f(fwd.make_dual(x, torch.ones_like(x)))
            assert not launches
            if name != "Fp8TrainLinear" or not grad:
                f(x)
                assert launches


@pytest.mark.parametrize("name", NAMES)
def test_tracing_is_refused(launches, name):
    """A trace would hold the allocation of the result and no launch: refused by name, before one."""
    from torch.fx.experimental.proxy_tensor import make_fx

    f = _operators()[name]
    x = torch.randn(4, 128)
    launches.clear()
    with torch.no_grad():
        with pytest.raises(RuntimeError, match="cannot be recorded"):
            torch.jit.trace(f, (x,), check_trace=False)
        for pre_dispatch in (False, True):
            with pytest.raises(RuntimeError, match="cannot be recorded"):
                make_fx(f, pre_dispatch=pre_dispatch)(x)
        assert not launches
        with torch.device("cpu"):  # a function mode that records nothing
            f(x)
        assert launches


class _Mix:
    def __call__(self, attn, hidden_states, encoder_hidden_states=None, attention_mask=None, rotary_emb=None, timestep=None):
        return attn.to_out[0](attn.to_q(hidden_states))


def _block():
    from svoo_amd import dit

    torch.manual_seed(0)
    cfg = dit.WanDiTConfig(num_attention_heads=1, ffn_dim=64, num_layers=1, text_dim=32)
    block = dit.make_pipe(cfg, dtype=torch.float32).transformer.blocks[0].requires_grad_(False)
    for attn in (block.attn1, block.attn2):
        attn.set_processor(_Mix())
    return block, torch.randn(1, 5, cfg.dim), torch.randn(1, 3, cfg.dim), torch.randn(1, 6, cfg.dim)


def test_fused_norms_step_back_for_records_and_tangents(launches):
    """A block with fused norms traces and takes tangents as one without."""
    import torch.autograd.forward_ad as fwd

    block, x, ctx, temb = _block()

    def run(x):
        return block(x, ctx, temb, None)

    def tangent():
        with fwd.dual_level():
            return fwd.unpack_dual(run(fwd.make_dual(x, torch.ones_like(x)))).tangent

    with torch.no_grad():
        want, want_traced = tangent(), torch.jit.trace(run, (x,), check_trace=False)(2 * x)
        block.fused_norms = True
        assert torch.equal(tangent(), want)
        assert torch.equal(torch.func.jvp(run, (x,), (torch.ones_like(x),))[1], want)
        assert torch.equal(torch.jit.trace(run, (x,), check_trace=False)(2 * x), want_traced)
        assert not launches
        run(x)
        assert [name for name, _ in launches] == ["svoo_layer_norm_fwd"] * 3


# ------------------------------------------------------------------------------------------------ no work for a backward pass
@pytest.mark.parametrize("how", ["no_grad", "inference_mode", "nothing requires a gradient", "x alone", "weight alone", "both"])
def test_linear_lays_out_what_its_backward_pass_reads_and_no_more(launches, how):
    """Transposed copies of the weight (for dx) and of x (for dw) where that gradient may be asked for; none in evaluation."""
    import contextlib

    from svoo_amd import fp8

    off = {"no_grad": torch.no_grad, "inference_mode": torch.inference_mode}.get(how)
    x = torch.randn(3, 5, 64, requires_grad=off is not None or how in ("x alone", "both"))
    w = torch.randn(32, 64, requires_grad=off is not None or how in ("weight alone", "both"))
    with off() if off is not None else contextlib.nullcontext():
        y = fp8.fp8_linear(x, w, torch.randn(32, requires_grad=off is not None))
    need_x, need_w = how in ("x alone", "both"), how in ("weight alone", "both")
    assert y.shape == (3, 5, 32) and y.requires_grad == (need_x or need_w)
    names, args = zip(*launches)
    assert names == ("svoo_fp8_quantize_tiles", "svoo_fp8_quantize_tiles" if need_w else "svoo_fp8_quantize_rows",
                     "svoo_fp8_matmul")
    assert (args[0][9] is not None) == need_x  # the weight's transposed values
    if need_w:
        assert args[1][9] is not None


# ------------------------------------------------------------------------------------------------ training beside attention
@pytest.mark.parametrize("lost", [False, True])
@pytest.mark.parametrize("trainable", [False, True])
def test_attention_without_a_backward_pass_refuses_trainable_8_bit_projections(launches, lost, trainable):
    """A result without a graph from projections with one is refused for the layers that exist to train, and only there."""
    from types import SimpleNamespace

    from svoo_amd import fp8
    from svoo_amd.processor import WanAttn_SAPAttn_Processor

    class Processor(WanAttn_SAPAttn_Processor):
        def attention_core_logic(self, query, key, value, timestep):
            out = (query + key + value).transpose(1, 2).flatten(2, 3)
            return out.detach() if lost else out

    make = fp8.Fp8TrainLinear if trainable else torch.nn.Linear
    attn = SimpleNamespace(heads=1, to_q=make(64, 64), to_k=make(64, 64), to_v=make(64, 64), to_out=[lambda t: t] * 2)
    proc, x, t = Processor(0), torch.randn(1, 6, 64), torch.tensor([3.0])
    launches.clear()
    if trainable and lost:
        with pytest.raises(RuntimeError, match="sparse attention has no backward pass"):
            proc(attn, x, timestep=t)
    else:
        assert proc(attn, x, timestep=t).requires_grad == (not lost)
    with torch.no_grad():
        assert proc(attn, x, timestep=t).shape == x.shape


@pytest.mark.parametrize("lost", [False, True])
def test_hunyuan_attention_refuses_trainable_8_bit_projections_too(launches, lost):
    from types import SimpleNamespace

    from svoo_amd import fp8
    from svoo_amd.processor import Hunyuan_SAPAttn_Processor

    class Processor(Hunyuan_SAPAttn_Processor):
        def attention_core_logic(self, query, key, value, timestep, layer_idx=None, cu_max_seqlens=None):
            out = query + key + value
            return out.detach() if lost else out

    attn = SimpleNamespace(heads=1, norm_q=None, norm_k=None, to_out=[lambda t: t] * 2,
                           **{n: fp8.Fp8TrainLinear(64, 64) for n in ("to_q", "to_k", "to_v")})
    proc, x, t = Processor(0), torch.randn(1, 6, 64), torch.tensor([3.0])
    if lost:
        with pytest.raises(RuntimeError, match="sparse attention has no backward pass"):
            proc(attn, x, timestep=t)
    else:
        proc(attn, x, timestep=t)
    with torch.no_grad():
        proc(attn, x, timestep=t)


# ------------------------------------------------------------------------------------------------ what no launch can hold
def test_more_batch_entries_than_a_launch_has_blocks_are_refused():
    from svoo_amd import _lib

    lib = _lib.lib()
    for batch, cols in ((1 << 24, 8), (1 << 30, 8), (1 << 24, 5120), (1 << 22, 6145), (1 << 22, 16384)):
        assert lib.svoo_layer_norm_fwd(16, 0, cols, cols, 16, 2, cols, None, 2, 0, 1, 1e-6, batch, 1, cols, 16, 0, None, None,
                                       0, None, None, None) == -2
        assert f"{batch} batch entries of {cols} columns" in _lib.last_error()
        assert lib.svoo_layer_norm_bwd(16, 0, cols, cols, 16, 0, cols, cols, None, 2, 0, 1, 16, 16, batch, 1, cols, 16, 16, 2,
                                       16, 2, None, 0, None) == -2
        assert f"{batch} batch entries of {cols} columns" in _lib.last_error()


# ------------------------------------------------------------------------------------------------ an FFN that is someone else's
def test_an_ffn_with_a_forward_of_its_own_is_called(launches):
    """The block hands 8-bit rows to the FFN's first layer past its call only where nothing has replaced a call: a forward
    set on an instance (as offloading does), a subclass's, and hooks on every module get theirs."""
    from svoo_amd import fp8

    class Own(fp8.Fp8Linear):
        def forward(self, x):
            seen.append("subclass")
            return super().forward(x)

    class OwnSequential(torch.nn.Sequential):
        def forward(self, x):
            seen.append("container")
            return super().forward(x)

    seen = []
    block, x, ctx, temb = _block()
    block.fused_norms = True
    plain = torch.nn.Sequential(fp8.Fp8Linear.from_linear(block.ffn[0], "gelu_tanh"), torch.nn.Identity(),
                                fp8.Fp8Linear.from_linear(block.ffn[2]))

    def run(ffn):
        block.ffn = ffn
        seen.clear()
        launches.clear()
        with torch.no_grad():
            block(x, ctx, temb, None)
        return [name for name, _ in launches].count("svoo_fp8_quantize_rows")

    assert run(plain) == 1 and seen == []  # the second layer's rows; the first's come from the norm
    assert run(torch.nn.Sequential(Own.from_linear(torch.nn.Linear(128, 64)), *plain[1:])) == 2 and seen == ["subclass"]
    assert run(OwnSequential(*plain)) == 2 and seen == ["container"]
    forward = plain[0].forward
    plain[0].forward = lambda t: (seen.append("instance"), forward(t))[1]
    assert run(plain) == 2 and seen == ["instance"]
    del plain[0].forward
    handle = torch.nn.modules.module.register_module_forward_hook(lambda m, args, out: seen.append(m))
    try:
        assert run(plain) == 2 and plain in seen and plain[0] in seen
    finally:
        handle.remove()
    assert run(plain) == 1


@pytest.mark.parametrize("trainable", [False, True])
@pytest.mark.parametrize("spoil", ["a bias in fp64", "a weight in fp64", "a weight of nothing", "a type of gradients"])
def test_a_pipeline_with_one_layer_that_no_call_could_take_is_left_as_it_was(launches, trainable, spoil):
    from svoo_amd import dit
    from svoo_amd.inference import replace_wan_linear

    cfg = dit.WanDiTConfig(num_attention_heads=1, ffn_dim=64, num_layers=2, text_dim=32)
    pipe = dit.make_pipe(cfg, dtype=torch.float32)
    ffn = pipe.transformer.blocks[1].ffn
    kw = {}
    if spoil == "a bias in fp64":
        ffn[2].bias = torch.nn.Parameter(ffn[2].bias.detach().double())
    elif spoil == "a weight in fp64":
        ffn[2].double()
    elif spoil == "a weight of nothing":
        ffn[2] = torch.nn.Linear(64, 0)
    elif trainable:
        kw = dict(grad_dtype=torch.bfloat16)
    else:
        return
    before = {n: id(m) for n, m in pipe.transformer.named_modules()}
    with pytest.raises((TypeError, ValueError)):
        replace_wan_linear(pipe, trainable=trainable, **kw)
    assert {n: id(m) for n, m in pipe.transformer.named_modules()} == before
