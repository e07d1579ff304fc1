"""What the layer norm and the 8-bit operators refuse, before any launch and without a GPU."""

import pytest
import torch


def _call(name, args, change, order):
    from svoo_amd import _lib

    assert set(change) <= set(args)
    a = {**args, **change}
    rc = getattr(_lib.lib(), name)(*[a[k] for k in order], None)
    return rc, _lib.last_error()


FWD = dict(x=16, x_type=0, xb=640, xr=64, w=None, w_type=2, wb=0, b=None, b_type=2, bb=0, modulated=0, eps=1e-6, batch=2,
           rows=10, cols=64, y=16, y_type=0, q=None, s=None, fp8=0, mean=None, rstd=None)


@pytest.mark.parametrize("change,code,message", [
    (dict(x_type=3), -1, "element type 3"), (dict(y_type=-1), -1, "element types"), (dict(w_type=9), -1, "element types"),
    (dict(cols=0), -1, "cols=0"), (dict(cols=16385), -2, "16385 columns"), (dict(batch=-1), -1, "batch=-1"),
    (dict(rows=1 << 31), -2, "2^31 rows"), (dict(batch=1 << 16, rows=1 << 15), -2, "2^31 rows"),
    (dict(x=None), -1, "null pointer"), (dict(y=None), -1, "one of y"), (dict(q=16, s=16), -1, "one of y"),
    (dict(y=None, q=16), -1, "one of y"), (dict(y=None, q=12, s=16), -1, "8-byte"), (dict(fp8=2), -1, "8-bit type 2"),
])
def test_norm_entry_refusals(change, code, message):
    rc, text = _call("svoo_layer_norm_fwd", FWD, change, list(FWD))
    assert rc == code and message in text, text


BWD = dict(x=16, x_type=0, xb=640, xr=64, dy=16, dy_type=0, db_=640, dr=64, w=None, w_type=2, wb=0, modulated=0, mean=16,
           rstd=16, batch=1, rows=1000, cols=64, dx=16, dw=16, dw_type=2, db=16, db_type=2, ws=None, ws_bytes=0)


@pytest.mark.parametrize("change,code,message", [
    (dict(), -3, "workspace of 0 bytes"), (dict(ws=16, ws_bytes=100), -3, "workspace of 100"),
    (dict(dy_type=5), -1, "element types"), (dict(mean=None), -1, "null pointer"), (dict(dy=None), -1, "null pointer"),
    (dict(rows=0), -1, "parameter gradients of no rows"), (dict(cols=20000), -2, "20000 columns"),
])
def test_norm_backward_entry_refusals(change, code, message):
    rc, text = _call("svoo_layer_norm_bwd", BWD, change, list(BWD))
    assert rc == code and message in text, text


def test_entries_with_nothing_to_do_launch_nothing():
    from svoo_amd import _lib

    lib = _lib.lib()
    assert _call("svoo_layer_norm_fwd", FWD, dict(rows=0, x=None), list(FWD))[0] == 0
    assert _call("svoo_layer_norm_bwd", BWD, dict(rows=0, dw=None, db=None), list(BWD))[0] == 0
    assert _call("svoo_layer_norm_bwd", BWD, dict(dx=None, dw=None, db=None), list(BWD))[0] == 0
    assert lib.svoo_fp8_quantize_rows(None, 0, 64, 0, 64, 0, None, None, None) == 0
    assert lib.svoo_fp8_dequantize(None, 128, None, 1, 1, 1, 0, 64, 0, None, 0, None) == 0
    assert lib.svoo_fp8_matmul(None, 128, None, 1, 1, 0, None, 128, None, 1, 1, 1, None, 0, 0, 0, 5, 128, None, 0, None, 0, None) == 0
    assert lib.svoo_layer_norm_bwd_workspace_size(0, 5, 5) == 0
    assert lib.svoo_layer_norm_bwd_workspace_size(1, 1, 64) == 0  # one part writes its gradients itself
    assert lib.svoo_layer_norm_bwd_workspace_size(1, 32760, 1536) <= 1 << 24
    assert lib.svoo_fp8_quantize_tiles_workspace_size(129, 100) == 800


MM = dict(a=16, ar=128, sa=16, sar=1, sac=4, a_type=0, b=16, br=128, sb=16, sbr=1, sbc=1, tall=128, bias=None, bias_type=0, act=0, m=4, n=4,
          k=128, c=16, c_type=0, ws=None, ws_bytes=0)


@pytest.mark.parametrize("change,code,message", [
    (dict(a_type=2), -1, "8-bit type 2"), (dict(c_type=3), -1, "element types"), (dict(tall=64), -1, "64 rows a scale"),
    (dict(act=2), -1, "activation 2"), (dict(k=100), -1, "k=100"), (dict(k=0), -1, "k=0"), (dict(m=-1), -1, "m=-1"),
    (dict(m=1 << 30), -2, "m=1073741824"), (dict(a=None), -1, "null"), (dict(sb=None), -1, "null"), (dict(c=None), -1, "null"),
    (dict(a=8), -1, "16-byte"), (dict(br=136), -1, "16-byte"),
])
def test_product_entry_refusals(change, code, message):
    rc, text = _call("svoo_fp8_matmul", MM, change, list(MM))
    assert rc == code and message in text, text


QT = dict(x=16, type=0, xr=64, rows=4, cols=64, fp8=0, square=0, q=16, s=16, qt=16, st=16, sums=None, sums_type=2, ws=None,
          ws_bytes=0)


@pytest.mark.parametrize("change,code,message", [
    (dict(type=3), -1, "element type 3"), (dict(fp8=-1), -1, "8-bit type"), (dict(s=None), -1, "without scales"),
    (dict(st=None), -1, "without scales"), (dict(q=4), -1, "8 and 16-byte"), (dict(qt=8), -1, "8 and 16-byte"),
    (dict(sums=16), -3, "workspace of 0"), (dict(sums=16, square=1), -1, "square"), (dict(cols=0), -1, "4 x 0"),
    (dict(rows=0, sums=16), -1, "no rows"), (dict(q=None, s=None, qt=None, st=None), -1, "null"), (dict(x=None), -1, "null"),
    (dict(rows=1 << 40), -2, "2^24"), (dict(rows=9000000), -2, "9000000 rows"),
])
def test_tile_quantiser_entry_refusals(change, code, message):
    rc, text = _call("svoo_fp8_quantize_tiles", QT, change, list(QT))
    assert rc == code and message in text, text


def test_row_quantiser_and_dequantiser_entry_refusals():
    from svoo_amd import _lib

    lib = _lib.lib()
    for args, message in (((16, 7, 64, 4, 64, 0, 16, 16, None), "element type 7"), ((16, 0, 64, 4, 64, 0, 4, 16, None), "8-byte"),
                          ((16, 0, 64, 4, 64, 0, None, 16, None), "null"), ((16, 0, 64, -4, 64, 0, 16, 16, None), "-4 x 64")):
        assert lib.svoo_fp8_quantize_rows(*args) == -1 and message in _lib.last_error()
    for args, message in (((16, 128, 16, 1, 1, 7, 4, 64, 0, 16, 0, None), "7 rows a scale"),
                          ((16, 12, 16, 1, 1, 1, 4, 64, 0, 16, 0, None), "8-byte"), ((16, 128, None, 1, 1, 1, 4, 64, 0, 16, 0, None), "null")):
        assert lib.svoo_fp8_dequantize(*args) == -1 and message in _lib.last_error()


def test_norm_refuses_in_python():
    from svoo_amd import norm

    x = torch.zeros(2, 3, 8)
    for t in (torch.zeros(2, 3, 8, dtype=torch.float64), torch.zeros(2, 8, dtype=torch.int32), [1.0]):
        with pytest.raises((TypeError, AttributeError)):
            norm.layer_norm(t)
    with pytest.raises(AssertionError, match="GPU"):
        norm.layer_norm(x)
    with pytest.raises(ValueError, match="not both"):
        norm.layer_norm(x, weight=torch.zeros(8), shift=torch.zeros(8))
    with pytest.raises(ValueError, match="not both"):
        norm.layer_norm(x, weight=torch.zeros(8, requires_grad=True), shift=torch.zeros(8))
    with pytest.raises(ValueError, match="eps"):
        norm.layer_norm(x, eps=-1.0)
    with pytest.raises(ValueError, match="eps"):
        norm.layer_norm(x, eps=float("nan"))
    with pytest.raises(RuntimeError, match="no backward"):
        norm.layer_norm_fp8(x.requires_grad_())
    with pytest.raises(TypeError, match="float8"):
        norm.layer_norm_fp8(torch.zeros(2, 8), dtype=torch.bfloat16)


def test_fp8_refuses_in_python():
    from svoo_amd import fp8

    x = torch.zeros(4, 128)
    q, s = x.to(torch.float8_e4m3fn), torch.zeros(4, 1, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    with pytest.raises(AssertionError, match="GPU"):
        fp8.fp8_quantize_rows(x)
    with pytest.raises(TypeError, match="float8"):
        fp8.fp8_quantize_rows(x, dtype=torch.int8)
    with pytest.raises(TypeError, match="bfloat16, float16 or float32"):
        fp8.fp8_quantize_rows(x.double())
    with pytest.raises(RuntimeError, match="no backward"):
        fp8.fp8_quantize_rows(x.clone().requires_grad_())
    with pytest.raises(ValueError, match="a matrix"):
        fp8.fp8_quantize_blocks(torch.zeros(2, 3, 4))
    with pytest.raises(ValueError, match="a matrix"):
        fp8.fp8_quantize_both(torch.zeros(4))
    with pytest.raises(ValueError, match="activation"):
        fp8.fp8_matmul(q, s, q, s, activation="relu")
    with pytest.raises(TypeError, match="float8_e8m0fnu"):
        fp8.fp8_matmul(q, x, q, s)
    with pytest.raises(TypeError, match="e4m3"):
        fp8.fp8_matmul(x, s, q, s)
    with pytest.raises(AssertionError, match="GPU"):
        fp8.fp8_matmul(q, s, q, s)
    with pytest.raises(RuntimeError, match="no backward"):
        fp8.fp8_matmul(q, s, q, s, bias=torch.zeros(4, requires_grad=True))
    with pytest.raises(ValueError, match="activation"):
        fp8.Fp8Linear(x, activation="tanh")
    with pytest.raises((TypeError, AssertionError)):
        fp8.fp8_linear(x, x)
    with pytest.raises(TypeError, match="float8"):
        fp8.fp8_linear(x, x, grad_dtype=torch.float16)
    with pytest.raises(TypeError, match="float8"):
        fp8.Fp8TrainLinear.from_linear(torch.nn.Linear(8, 8), grad_dtype=torch.bfloat16)


@pytest.mark.parametrize("trainable", [False, True])
def test_replace_wan_linear_leaves_a_pipeline_that_it_refuses(trainable):
    from svoo_amd import dit
    from svoo_amd.inference import replace_wan_linear

    cfg = dit.WanDiTConfig(num_attention_heads=1, ffn_dim=64, num_layers=2, text_dim=32)
    pipe = dit.make_pipe(cfg, dtype=torch.float32)
    before = {n: id(m) for n, m in pipe.transformer.named_modules()}
    with pytest.raises(AssertionError, match="GPU"):
        replace_wan_linear(pipe, trainable=trainable)
    assert {n: id(m) for n, m in pipe.transformer.named_modules()} == before
    assert not pipe.transformer.fused_norms and not any(b.fused_norms for b in pipe.transformer.blocks)


def test_train_linear_shares_parameters():
    from svoo_amd import fp8

    for bias in (True, False):
        old = torch.nn.Linear(8, 16, bias=bias).eval()
        new = fp8.Fp8TrainLinear.from_linear(old, torch.float8_e5m2)
        assert new.weight is old.weight and new.bias is old.bias and new.grad_dtype == torch.float8_e5m2
        assert (new.in_features, new.out_features, new.training) == (8, 16, False)
        assert new.state_dict().keys() == old.state_dict().keys()
