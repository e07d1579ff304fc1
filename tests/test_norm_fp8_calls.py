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
