"""What dense attention, rotary positions and gated residuals refuse, before any launch and without a GPU, and the arguments
that they hand to their C entries, recorded on the CPU in place of the launches."""

import math

import pytest
import torch


@pytest.fixture
def launches(monkeypatch):
    from svoo_amd import _lib

    seen = []
    monkeypatch.setattr(_lib, "launch", lambda device, name, *args: seen.append((name, args)))
    monkeypatch.setattr(_lib, "require_gpu_tensor", lambda t, name: None)
    return seen


def _call(name, args, change):
    from svoo_amd import _lib

    assert set(change) <= set(args)
    rc = getattr(_lib.lib(), name)(*{**args, **change}.values(), None)
    return rc, _lib.last_error()


def _rows(*names):
    return {f"{n}{s}": v for n in names for s, v in (("", 16), ("_b", 1024), ("_h", 64), ("_r", 128))}


SIZES = dict(type=0, batch=1, heads=2, kv_heads=2, sq=8, sk=8, d=64, scale=0.1, q_lens=None, k_lens=None)
FWD = {**_rows("q", "k", "v"), **SIZES, **dict(o=16, rest=None, lse=16, ws=None, ws_bytes=0)}
BWD = {**_rows("dy", "q", "k", "v", "o"), **dict(rest=None, lse=16), **SIZES,
       **dict(dq=16, dk=16, dv=16, ws=256, ws_bytes=1 << 20)}
SHARED = [
    (dict(type=2), -1, "element type 2"), (dict(batch=-1), -1, "batch=-1"), (dict(d=0), -1, "d=0"), (dict(d=136), -2, "d=136"),
    (dict(d=60), -2, "d=60"), (dict(heads=3), -1, "3 heads share 2"), (dict(kv_heads=0), -1, "share 0"),
    (dict(sq=(1 << 30) + 1), -2, "up to 2^30"), (dict(sk=1 << 30, batch=2), -2, "tiles of 256"), (dict(scale=0.0), -1, "scale=0"),
    (dict(scale=-1.0), -1, "scale=-1"), (dict(scale=math.inf), -1, "scale=inf"), (dict(scale=math.nan), -1, "scale=nan"),
    (dict(q=None), -1, "null pointer"), (dict(k=None), -1, "null pointer"), (dict(lse=None), -1, "null pointer"),
    (dict(q=8), -1, "16-byte"), (dict(k_r=130), -1, "16-byte"), (dict(v_h=4), -1, "16-byte"), (dict(q_r=1 << 23), -1, "16-byte"),
    (dict(q_r=-128), -1, "16-byte"),
]


@pytest.mark.parametrize("change,code,message", SHARED + [(dict(o=None), -1, "null pointer"), (dict(o=8), -1, "16-byte"),
                                                          (dict(rest=8), -1, "16-byte"),
                                                          (dict(sk=5000), -3, "workspace of 0 bytes")])
def test_attention_entry_refusals(change, code, message):
    rc, text = _call("svoo_dense_attention_fwd", FWD, change)
    assert rc == code and message in text, text


@pytest.mark.parametrize("change,code,message", SHARED + [(dict(dy=None), -1, "null pointer"), (dict(dk=8), -1, "16-byte"),
                                                          (dict(ws_bytes=16), -3, "workspace of 16"), (dict(sk=0), -1, "sk=0"),
                                                          (dict(ws=None), -3, "workspace"), (dict(ws=8), -3, "workspace")])
def test_attention_backward_entry_refusals(change, code, message):
    rc, text = _call("svoo_dense_attention_bwd", BWD, change)
    assert rc == code and message in text, text


ROPE = dict(x=16, type=0, xb=640, xr=128, xh=64, batch=1, rows=10, heads=2, d=64, norm=1, w=16, w_type=0, eps=1e-6, axes=1,
            channels=None, theta=None, grid=None, start=None, pos=16, pos_type=1, pos_b=0, halves=0, y=16)


def _rope_args(change):
    import ctypes

    a = dict(ROPE)
    n = change.get("axes", 1)
    a["channels"] = (ctypes.c_int * max(n, 1))(*change.pop("each", (64,) * max(n, 1)))
    a["theta"] = (ctypes.c_double * max(n, 1))(*change.pop("thetas", (1e4,) * max(n, 1)))
    if change.get("pos_type") == 0:
        a["grid"] = (ctypes.c_int * n)(*change.pop("cells"))
    return a, change


@pytest.mark.parametrize("change,code,message", [
    (dict(type=3), -1, "element types"), (dict(w_type=-1), -1, "element types"), (dict(d=63), -1, "d=63"), (dict(d=0), -1, "d=0"),
    (dict(d=514), -2, "d=514"), (dict(heads=0), -1, "heads=0"), (dict(norm=3), -1, "norm 3"), (dict(heads=257), -2, "257 heads"),
    (dict(rows=1 << 31), -2, "tokens"), (dict(batch=1 << 16, rows=1 << 15), -2, "tokens"), (dict(axes=0), -1, "0 axes"),
    (dict(axes=5, each=(8,) * 5), -1, "5 axes"), (dict(each=(63,)), -1, "63 channels"), (dict(each=(-2,)), -1, "-2 channels"),
    (dict(each=(66,)), -1, "more than 64"), (dict(axes=2, each=(40, 40)), -1, "more than 64"), (dict(thetas=(0.0,)), -1, "theta 0"),
    (dict(thetas=(math.nan,)), -1, "theta nan"), (dict(pos_type=4), -1, "position type 4"), (dict(pos=None), -1, "null pointer"),
    (dict(pos_type=0, cells=(0,)), -1, "grid of 0"), (dict(x=None), -1, "null pointer"), (dict(y=None), -1, "null pointer"),
])
def test_rope_entry_refusals(change, code, message):
    rc, text = _call("svoo_axis_rope_fwd", *_rope_args(dict(change)))
    assert rc == code and message in text, text


RES = dict(x=16, type=0, xb=640, xr=64, b=16, bb=640, br=64, gate=None, gate_type=2, gate_b=0, w=None, w_type=2, w_b=0, c=None,
           c_type=2, c_b=0, modulated=0, eps=1e-6, batch=1, rows=10, cols=64, h=16, y=16, mean=None, rstd=None)
RES_BWD = dict(dh=16, dhb=640, dhr=64, dy=16, dyb=640, dyr=64, type=0, h=16, b=16, bb=640, br=64, gate=16, gate_type=2, gate_b=0,
               w=16, w_type=2, w_b=0, modulated=0, mean=16, rstd=16, batch=1, rows=10, cols=64, dx=16, db=16, dgate=16,
               dgate_type=2, dgate_each=0, dw=16, dw_type=2, dw_each=0, dc=16, dc_type=2, dc_each=0, ws=16, ws_bytes=1 << 20)
RES_SHARED = [(dict(type=3), -1, "element type 3"), (dict(gate_type=7), -1, "element types"), (dict(cols=0), -1, "cols=0"),
              (dict(cols=16385), -2, "16385 columns"), (dict(rows=1 << 31), -2, "2^31 rows"), (dict(batch=-1), -1, "batch=-1"),
              (dict(batch=65536), -2, "65536 batch entries"), (dict(h=None), -1, "null pointer")]


@pytest.mark.parametrize("change,code,message", RES_SHARED + [(dict(b=None), -1, "null pointer"), (dict(x=None), -1, "null")])
def test_residual_entry_refusals(change, code, message):
    rc, text = _call("svoo_residual_norm_fwd", RES, change)
    assert rc == code and message in text, text


@pytest.mark.parametrize("change,code,message", RES_SHARED + [
    (dict(dh=None, dy=None), -1, "no incoming gradient"), (dict(mean=None), -1, "null pointer"), (dict(dy=None), -1, "without dy"),
    (dict(b=None), -1, "without the branch"), (dict(ws=None), -3, "workspace"), (dict(ws_bytes=100), -3, "workspace of 100"),
    (dict(rows=0), -1, "no rows"), (dict(dw_type=5), -1, "element types")])
def test_residual_backward_entry_refusals(change, code, message):
    rc, text = _call("svoo_residual_norm_bwd", RES_BWD, change)
    assert rc == code and message in text, text


def test_entries_with_nothing_to_do_launch_nothing():
    from svoo_amd import _lib

    lib = _lib.lib()
    assert _call("svoo_dense_attention_fwd", FWD, dict(sq=0, q=None))[0] == 0
    assert _call("svoo_dense_attention_bwd", BWD, dict(dq=None, dk=None, dv=None))[0] == 0
    assert _call("svoo_residual_norm_fwd", RES, dict(rows=0, x=None))[0] == 0
    assert _call("svoo_residual_norm_bwd", RES_BWD, dict(dx=None, db=None, dgate=None, dw=None, dc=None))[0] == 0
    assert _call("svoo_axis_rope_fwd", *_rope_args(dict(rows=0, x=None)))[0] == 0
    assert lib.svoo_dense_attention_fwd_workspace_size(1, 12, 32760, 32760, 128) == 0  # blocks enough for whole rows
    assert lib.svoo_dense_attention_bwd_workspace_size(0, 0, 1, 1, 5, 5, 64, 1, 1) == 0
    assert lib.svoo_axis_rope_bwd_workspace_size(1, 5, 2, 64, 0) == 0
    assert lib.svoo_residual_norm_bwd_workspace_size(0, 5, 64) == 0


# ------------------------------------------------------------------------------------------------ in Python
def test_attention_refuses_in_python(launches):
    from svoo_amd import dense

    q = torch.zeros(2, 4, 5, 64, dtype=torch.bfloat16)
    k = torch.zeros(2, 2, 7, 64, dtype=torch.bfloat16)
    for bad in (q.float(), q.double(), q.to(torch.int32), [1.0]):
        with pytest.raises((TypeError, AttributeError), match="bfloat16 or float16|requires_grad"):
            dense.dense_attention(bad, k, k)
    with pytest.raises(ValueError, match="k: torch.float16"):
        dense.dense_attention(q, k.half(), k)
    for args in ((q[0], k[0], k[0]), (q, k, k[:, :, :5]), (q[:1], k, k), (q, k[..., :32], k[..., :32])):
        with pytest.raises(ValueError, match="expected"):
            dense.dense_attention(*args)
    with pytest.raises(ValueError, match="3 query heads over 2"):
        dense.dense_attention(q[:, :3], k, k)
    for d in (0, 129):
        with pytest.raises(ValueError, match="head dim"):
            dense.dense_attention(*(torch.zeros(1, 1, 2, d, dtype=torch.bfloat16) for _ in range(3)))
    for scale in (0.0, -1.0, math.nan, math.inf):
        with pytest.raises(ValueError, match="scale"):
            dense.dense_attention(q, k, k, scale=scale)
    for lens in ([5, 5], torch.tensor([5, 5]), torch.tensor([5], dtype=torch.int32), torch.tensor([[5, 5]], dtype=torch.int32)):
        with pytest.raises(ValueError, match="q_lens: int32"):
            dense.dense_attention(q, k, k, q_lens=lens)
        with pytest.raises(ValueError, match="k_lens: int32"):
            dense.dense_attention(q, k, k, k_lens=lens)
    with pytest.raises(RuntimeError, match="no backward"):
        dense.dense_attention_fwd(q.requires_grad_(), k, k)
    q = q.detach()
    lse = torch.zeros(2, 4, 5)
    for dy, o, l, what in ((q[:, :2], q, lse, "dy"), (q, q.half(), lse, "o"), (q, q, lse.double(), "lse"), (q, q, lse[:1], "lse")):
        with pytest.raises(ValueError, match=f"{what}: "):
            dense.dense_attention_bwd(dy, q, k, k, o, None, l)
    assert not launches


def test_rope_refuses_in_python(launches):
    from svoo_amd import rope

    x = torch.zeros(2, 6, 3, 64)
    pos = torch.zeros(6, 1, dtype=torch.int32)
    with pytest.raises(TypeError, match="bfloat16, float16 or float32"):
        rope.axis_rope(x.double(), (64,), positions=pos)
    for shape in ((6, 3, 64), (2, 6, 3, 63), (2, 6, 0, 64), (2, 6, 3, 514)):
        with pytest.raises(ValueError, match="axis_rope"):
            rope.axis_rope(torch.zeros(shape), (64,), positions=pos)
    for axes in ((), (8,) * 5, (63,), (-2,), (66,), (40, 40)):
        with pytest.raises(ValueError, match="axes"):
            rope.axis_rope(x, axes, positions=pos)
    for theta in (0.0, -1.0, math.nan, math.inf, (1.0, 2.0)):
        with pytest.raises(ValueError, match="theta"):
            rope.axis_rope(x, (64,), positions=pos, theta=theta)
    with pytest.raises(ValueError, match="norm"):
        rope.axis_rope(x, (64,), positions=pos, norm="layer")
    with pytest.raises(ValueError, match="eps"):
        rope.axis_rope(x, (64,), positions=pos, eps=-1.0)
    with pytest.raises(ValueError, match="a grid or positions"):
        rope.axis_rope(x, (64,))
    with pytest.raises(ValueError, match="a grid or positions"):
        rope.axis_rope(x, (64,), grid=(6,), positions=pos)
    with pytest.raises(ValueError, match="start goes with a grid"):
        rope.axis_rope(x, (64,), positions=pos, start=(0,))
    for grid in ((7,), (0,), (2, 3), (1 << 31,)):
        with pytest.raises(ValueError, match="grid"):
            rope.axis_rope(x, (64,), grid=grid)
    with pytest.raises(ValueError, match="start"):
        rope.axis_rope(x, (64,), grid=(6,), start=(1 << 31,))
    with pytest.raises(TypeError, match="positions"):
        rope.axis_rope(x, (64,), positions=pos.double())
    for shape in ((6,), (5, 1), (3, 6, 1), (6, 2)):
        with pytest.raises(ValueError, match="positions: shape"):
            rope.axis_rope(x, (64,), positions=torch.zeros(shape, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="no gradient for positions"):
        rope.axis_rope(x, (64,), positions=torch.zeros(6, 1, requires_grad=True))
    for norm, n in (("row", 64), ("head", 192), ("none", 64)):
        with pytest.raises(ValueError, match="weight: shape"):
            rope.axis_rope(x, (64,), positions=pos, norm=norm, weight=torch.ones(n))
    with pytest.raises(ValueError, match="at most"):
        rope.axis_rope(torch.zeros(1, 6, 129, 128), (64,), positions=pos, norm="row")
    for dy in (x[:1], x.half()):
        with pytest.raises(ValueError, match="dy: "):
            rope.axis_rope_bwd(dy, x, (64,), positions=pos)
    assert not launches


def test_residual_refuses_in_python(launches):
    from svoo_amd import norm

    x = torch.zeros(2, 3, 8)
    with pytest.raises(TypeError, match="bfloat16, float16 or float32"):
        norm.residual_norm(x.double(), x.double())
    for b in (x[:1], x.half(), x[..., :4]):
        with pytest.raises(ValueError, match="branch: "):
            norm.residual_norm(x, b)
        with pytest.raises(ValueError, match="branch: "):
            norm.gated_residual(x, b)
    for grad in (False, True):
        with pytest.raises(ValueError, match="not both"):
            norm.residual_norm(x, x, weight=torch.zeros(8, requires_grad=grad), scale=torch.zeros(8))
    for p in (torch.zeros(7), torch.zeros(3, 8), torch.zeros(2, 3, 8), torch.zeros(())):
        with pytest.raises(ValueError, match="gate: shape"):
            norm.residual_norm(x, x, p)
    with pytest.raises(ValueError, match="eps"):
        norm.residual_norm(x, x, eps=-1.0)
    with pytest.raises(ValueError, match="columns"):
        norm.residual_norm(torch.zeros(1, 16385), torch.zeros(1, 16385))
    with pytest.raises(ValueError, match="65536 batch entries"):
        norm.residual_norm(torch.zeros(65536, 8), torch.zeros(65536, 8), torch.zeros(65536, 8))
    with pytest.raises(RuntimeError, match="no backward"):
        norm.residual_norm_fwd(x, x, torch.zeros(8, requires_grad=True))
    st = torch.zeros(2, 3)
    with pytest.raises(ValueError, match="rstd: fp32"):
        norm.residual_norm_bwd(x, x, x, x, st, st.double())
    assert not launches


def test_on_the_cpu_the_operators_say_so():
    from svoo_amd import dense, norm, rope

    x = torch.zeros(1, 2, 4, 8, dtype=torch.bfloat16)
    for f in (lambda: dense.dense_attention(x, x, x), lambda: rope.axis_rope(x, (8,), grid=(2,)), lambda: norm.residual_norm(x, x),
              lambda: norm.gated_residual(x, x)):
        with pytest.raises(AssertionError, match="GPU"):
            f()


# ------------------------------------------------------------------------------------------------ records, tangents
def _operators():
    from svoo_amd import dense, norm, rope

    h = torch.randn(1, 2, 4, 64, dtype=torch.bfloat16)
    w, st, lse = torch.randn(4, 64), torch.zeros(4), torch.zeros(1, 2, 4)
    kw = dict(grid=(2,))

    def four(x):
        return x.view(1, 2, 2, 64)

    return {
        "dense_attention": lambda x: dense.dense_attention(x.bfloat16().view(1, 1, 4, 64), h[:, :1], h[:, :1]),
        "dense_attention of v": lambda x: dense.dense_attention(h[:, :1], h[:, :1], x.bfloat16().view(1, 1, 4, 64)),
        "dense_attention_fwd": lambda x: dense.dense_attention_fwd(x.bfloat16().view(1, 1, 4, 64), h[:, :1], h[:, :1])[0],
        "dense_attention_bwd": lambda x: dense.dense_attention_bwd(x.bfloat16().view(1, 1, 4, 64), h[:, :1], h[:, :1], h[:, :1],
                                                                   h[:, :1], None, lse[:, :1])[0],
        "axis_rope": lambda x: rope.axis_rope(four(x), (64,), **kw),
        "axis_rope of a weight": lambda x: rope.axis_rope(four(w), (64,), norm="head", weight=x[0], **kw),
        "axis_rope_bwd": lambda x: rope.axis_rope_bwd(four(x), four(w), (64,), **kw)[0],
        "residual_norm": lambda x: norm.residual_norm(x, w)[0], "residual_norm of a gate": lambda x: norm.residual_norm(w, w, x)[0],
        "residual_norm_fwd": lambda x: norm.residual_norm_fwd(w, x)[0], "gated_residual": lambda x: norm.gated_residual(w, x),
        "residual_norm_bwd": lambda x: norm.residual_norm_bwd(x, w, w, w, st, st)[0],
    }


NAMES = ["dense_attention", "dense_attention of v", "dense_attention_fwd", "dense_attention_bwd", "axis_rope",
         "axis_rope of a weight", "axis_rope_bwd", "residual_norm", "residual_norm of a gate", "residual_norm_fwd",
         "gated_residual", "residual_norm_bwd"]


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("grad", [False, True])
def test_tangents_are_refused(launches, name, grad):
    import torch.autograd.forward_ad as fwd

    with torch.set_grad_enabled(grad):
        f, x = _operators()[name], torch.randn(4, 64)
        with fwd.dual_level():
            with pytest.raises(RuntimeError, match="forward-mode"):
                f(fwd.make_dual(x, torch.ones_like(x)))
            assert not launches
            f(x)
            assert launches


@pytest.mark.parametrize("name", NAMES)
def test_tracing_is_refused(launches, name):
    from torch.fx.experimental.proxy_tensor import make_fx

    f, x = _operators()[name], torch.randn(4, 64)
    with torch.no_grad():
        with pytest.raises(RuntimeError, match="cannot be recorded"):
            torch.jit.trace(f, (x,), check_trace=False)
        with pytest.raises(RuntimeError, match="cannot be recorded"):
            make_fx(f)(x)
        assert not launches


# ------------------------------------------------------------------------------------------------ what the launches are given
def test_attention_operands_are_read_in_place_where_they_can_be(launches):
    from svoo_amd import dense

    def rows(t, at=0):
        launches.clear()
        dense.dense_attention(t, t, t)
        return launches[0][1][at:at + 4]

    base = torch.zeros(2, 7, 3, 64, dtype=torch.bfloat16)
    t = base.transpose(1, 2)
    assert rows(t) == (base.data_ptr(), 7 * 3 * 64, 64, 3 * 64)
    wide = torch.zeros(2, 7, 9 * 64, dtype=torch.bfloat16)[..., 192:384].unflatten(2, (3, 64)).transpose(1, 2)
    assert rows(wide) == (wide.data_ptr(), 7 * 576, 64, 576)
    assert rows(t[:1].expand(2, -1, -1, -1))[1] == 0
    one = torch.zeros(1, 1, 7, 64, dtype=torch.bfloat16).as_strided((1, 1, 7, 64), (13, 5, 64, 1))
    assert rows(one)[1:] == (0, 0, 64)  # strides of single entries do not count
    for odd in (torch.zeros(2, 3, 7, 67, dtype=torch.bfloat16)[..., :64], torch.zeros(2, 3, 64, 7, dtype=torch.bfloat16).mT,
                torch.zeros(2 * 3 * 7 * 64 + 1, dtype=torch.bfloat16)[1:].view(2, 3, 7, 64)):
        at, *strides = rows(odd)
        assert at != odd.data_ptr() and at % 16 == 0 and tuple(strides) == (3 * 7 * 64, 7 * 64, 64)
    # a head dim that is no multiple of 8 is padded, and the result cut again
    launches.clear()
    o = dense.dense_attention(*(torch.zeros(1, 2, 5, 37, dtype=torch.bfloat16) for _ in range(3)))
    assert o.shape == (1, 2, 5, 37) and launches[0][1][18] == 40
    assert o.transpose(1, 2).is_contiguous()
    scale = launches[0][1][19]
    assert scale == 37 ** -0.5


def test_attention_keeps_no_rest_without_gradients(launches):
    """What rounding o left is written for a backward pass only."""
    from svoo_amd import dense

    q = torch.zeros(1, 2, 5, 64, dtype=torch.bfloat16)
    dense.dense_attention(q, q, q)
    with torch.no_grad():
        dense.dense_attention(q.requires_grad_(), q, q)
    dense.dense_attention(q, q, q)
    assert [args[-4] is None for _, args in launches] == [True, True, False]


@pytest.mark.parametrize("gate", [None, "shared", "expanded", "own"])
@pytest.mark.parametrize("w", [None, "shared", "expanded", "own"])
def test_residual_sums_go_to_buffers_of_their_size(launches, gate, w):
    """A parameter with a row per batch entry has sums per entry, also where the entries share memory."""
    from svoo_amd import norm

    b, s, c = 3, 5, 16
    make = {"shared": torch.randn(c), "expanded": torch.randn(c).expand(b, 1, c), "own": torch.randn(b, 1, c)}
    x, st = torch.randn(b, s, c), torch.zeros(b, s)
    got = norm.residual_norm_bwd(x, x, x, x, st, st, make.get(gate), scale=make.get(w))
    a = dict(zip(RES_BWD, launches[0][1]))
    own = [k in ("expanded", "own") for k in (gate, w)]
    assert a["batch"] == (b if any(own) else 1) and a["batch"] * a["rows"] == b * s
    for key, kind, t in (("dgate", gate, got[2]), ("dw", w, got[3])):
        assert (t is None) == (kind is None) and a[key] == (None if t is None else t.data_ptr())
        if kind is not None:
            assert t.shape == make[kind].shape and bool(a[key + "_each"]) == (kind != "shared")
            assert t.numel() == (c if kind == "shared" else a["batch"] * c)
    assert a["gate_b"] == (c if gate == "own" else 0) and a["w_b"] == (c if w == "own" else 0)
