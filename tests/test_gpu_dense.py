"""Dense attention and its gradients against their definition in 64 bits, at the sizes and masks where they can go wrong."""

import math

import pytest
import torch

from train_ops_helpers import HALF, attention64, held, say

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


def make(seed, b, h, kh, sq, sk, d, dtype, device, level=1.0):
    g = torch.Generator().manual_seed(seed)
    q, k, v, dy = (torch.randn(b, s, n, d, generator=g) for s, n in ((sq, h), (sk, kh), (sk, kh), (sq, h)))
    v = v + 0.5 * torch.randn(d, generator=g)
    return [t.mul(f).to(dtype).to(device).transpose(1, 2) for t, f in ((q, level), (k, 1.0), (v, 1.0), (dy, 0.01))]


def lens(values, device):
    return None if values is None else torch.tensor(values, dtype=torch.int32, device=device)


def check(q, k, v, dy, **kw):
    from svoo_amd import dense

    want = attention64(q, k, v, dy, half=HALF[q.dtype], scale=kw.get("scale"),
                       q_lens=None if kw.get("q_lens") is None else kw["q_lens"].tolist(),
                       k_lens=None if kw.get("k_lens") is None else kw["k_lens"].tolist())
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = dense.dense_attention(*leaves, **kw)
    grads = torch.autograd.grad(o, leaves, dy)
    held(o, want["o"], "o")
    for t, name in zip(grads, ("dq", "dk", "dv")):
        held(t, want[name], name)
    o2, rest, lse = dense.dense_attention_fwd(q, k, v, **kw)
    held(lse.float(), want["lse"], "lse")
    assert torch.equal(o2, o)
    for a, b in zip(dense.dense_attention_bwd(dy, q, k, v, o2, rest, lse, **kw), grads):
        assert torch.equal(a, b)
    with torch.no_grad():
        assert torch.equal(dense.dense_attention(q, k, v, **kw), o)
    return o, grads


SIZES = [
    # b, h, kh, sq, sk, d
    (1, 1, 1, 1, 1, 128), (1, 2, 2, 1, 700, 128), (1, 2, 2, 300, 1, 64), (2, 2, 1, 33, 65, 64), (1, 3, 3, 64, 64, 128),
    (1, 2, 2, 257, 513, 128), (2, 4, 2, 256, 256, 128), (1, 4, 1, 129, 1025, 128), (1, 1, 1, 1037, 771, 64),
    (1, 2, 2, 40, 3000, 128), (1, 2, 1, 3000, 40, 128), (3, 2, 2, 31, 63, 40), (1, 2, 2, 70, 130, 80), (1, 1, 1, 65, 64, 8),
    (1, 2, 2, 50, 90, 120), (1, 2, 1, 20, 100, 37), (1, 1, 1, 9, 17, 1), (1, 1, 1, 300, 300, 127),
]


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("dtype", [BF, FP])
def test_sizes(gpu, size, dtype):
    say("sizes", size, dtype)
    check(*make(sum(size), *size, dtype, gpu))


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("q_lens,k_lens", [([100, 0, 65], [200, 130, 64]), (None, [0, 1, 200]), ([100, 1, 64], None),
                                           ([100, 50, 7], [0, 0, 0]), ([-5, 1000, 99], [1 << 30, -(1 << 31), 199])])
def test_lengths(gpu, q_lens, k_lens, d, dtype):
    """Rows behind a length may hold anything; queries without keys, and batch entries without queries, are 0."""
    say("lengths", q_lens, k_lens, d, dtype)
    q, k, v, dy = make(3, 3, 4, 2, 100, 200, d, dtype, gpu)
    for i in range(3):
        nq = 100 if q_lens is None else min(max(q_lens[i], 0), 100)
        nk = 200 if k_lens is None else min(max(k_lens[i], 0), 200)
        for t, n in ((q, nq), (dy, nq), (k, nk), (v, nk)):
            t[i, :, n:] = torch.tensor([math.nan, math.inf, -math.inf, 3e4], device=gpu).to(dtype)[
                torch.arange(t[i, :, n:].numel(), device=gpu) % 4].view(t[i, :, n:].shape)
    clean = [torch.nan_to_num(t, 0, 0, 0) for t in (q, k, v, dy)]
    from svoo_amd import dense

    want = attention64(*clean, half=HALF[dtype], q_lens=q_lens, k_lens=k_lens)
    kw = dict(q_lens=lens(q_lens, gpu), k_lens=lens(k_lens, gpu))
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = dense.dense_attention(*leaves, **kw)
    for t, name in zip((o, *torch.autograd.grad(o, leaves, dy)), ("o", "dq", "dk", "dv")):
        held(t, want[name], name)
    lse = dense.dense_attention_fwd(q, k, v, **kw)[2]
    held(lse, want["lse"], "lse")


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("sq,sk,kh", [(5, 8192, 2), (700, 4096, 1), (2048, 64, 2), (64, 65536, 1), (33, 1024, 2)])
def test_even_attention_is_exact(gpu, sq, sk, kh, dtype):
    """Keys of 0 give every key the weight 1 / N, a power of two: o is the mean of v, dv the mean of the incoming rows, and
    both are whole numbers over N here, so nothing is rounded before the result."""
    from svoo_amd import dense

    say("even", sq, sk, kh, dtype)
    g = torch.Generator().manual_seed(sq)
    q = torch.randn(1, 2, sq, 128, generator=g).to(dtype).to(gpu)
    k = torch.zeros(1, kh, sk, 128, dtype=dtype, device=gpu)
    v = torch.randint(-4, 5, (1, kh, sk, 128), generator=g).to(dtype).to(gpu)
    dy = torch.randint(-4, 5, (1, 2, sq, 128), generator=g).to(dtype).to(gpu)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    o = dense.dense_attention(*leaves)
    dv = torch.autograd.grad(o, [v], dy)[0]
    mean = v.detach().double().mean(2, keepdim=True).repeat_interleave(2 // kh, 1).expand(1, 2, sq, 128)
    assert torch.equal(o.double(), mean.to(dtype).double())
    sums = dy.double().view(1, kh, 2 // kh, sq, 128).sum((2, 3)) / sk
    assert torch.equal(dv.double(), sums[:, :, None].to(dtype).double().expand(1, kh, sk, 128))


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("sk,d,kh", [(1, 128, 1), (63, 64, 2), (65, 128, 2), (500, 128, 1), (4099, 64, 2), (3000, 120, 1)])
def test_one_key_each(gpu, sk, d, kh, dtype):
    """Each query picks one key whose score is 100 above every other: o is that key's value, dv that query's row, bit for bit."""
    from svoo_amd import dense

    say("one key", sk, d, kh, dtype)
    g = torch.Generator().manual_seed(sk)
    n = 300
    pick = torch.randint(0, sk, (n,), generator=g)
    pick[0], pick[-1] = 0, sk - 1
    # keys are signs of the bits of their number, so that another key's product is at least two lower
    bits = ((torch.arange(sk)[:, None] >> torch.arange(13)) & 1) * 2.0 - 1
    keys = torch.zeros(sk, d)
    keys[:, :13] = bits
    q = (50 * keys[pick]).expand(1, 2, n, d).to(dtype).to(gpu)
    k = keys.expand(1, kh, sk, d).to(dtype).to(gpu)
    v = torch.randn(1, kh, sk, d, generator=g).to(dtype).to(gpu)
    dy = torch.randn(1, 2, n, d, generator=g).to(dtype).to(gpu)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = dense.dense_attention(*leaves, scale=1.0)
    assert torch.equal(o, v[:, :, pick].repeat_interleave(2 // kh, 1))
    _, _, dv = torch.autograd.grad(o, leaves, dy)
    want = torch.zeros(1, kh, sk, d, dtype=torch.float64)
    want.index_add_(2, pick, dy.double().cpu().view(1, kh, 2 // kh, n, d).sum(2))
    err = (dv.double().cpu() - want).abs()
    mag = torch.zeros_like(want).index_add_(2, pick, dy.double().cpu().abs().view(1, kh, 2 // kh, n, d).sum(2))
    assert (err <= HALF[dtype] * want.abs() + 700 * 2.0 ** -23 * mag + 2.0 ** -24).all()


@pytest.mark.parametrize("level", [0.0, 1e-3, 8.0, 40.0])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_flat_and_sharp_scores(gpu, level, dtype):
    say("level", level, dtype)
    check(*make(8, 1, 2, 2, 130, 600, 128, dtype, gpu, level))


def test_large_and_small_gradients_in_fp16(gpu):
    """Incoming gradients over the whole range of fp16: dS keeps its digits by a power of two of its own."""
    q, k, v, dy = make(9, 2, 2, 1, 100, 900, 64, FP, gpu)
    for f in (1e-4, 1.0, 1000.0):
        say("gradients times", f)
        check(q, k, v, (dy.float() * f).to(FP))
    check(q, k, v, torch.zeros_like(dy))


@pytest.mark.parametrize("scale", [1e-3, 0.5, 3.0])
def test_scale(gpu, scale):
    check(*make(10, 1, 2, 2, 90, 150, 64, BF, gpu), scale=scale)


@pytest.mark.parametrize("which", range(6))
def test_strides_and_addresses(gpu, which):
    """Operands in any layout give the bits of contiguous ones."""
    from svoo_amd import dense

    b, h, s, n, d = 2, 4, 70, 90, 64
    q, k, v, dy = (t.contiguous() for t in make(11, b, h, 2, s, n, d, BF, gpu))

    def odd(t):
        if which == 0:
            return t.transpose(1, 2).contiguous().transpose(1, 2)
        if which == 1:  # a slice of a fused projection
            return torch.cat([t, t, t], 3)[..., d:2 * d]
        if which == 2:  # 2 bytes past a 16-byte address
            return torch.empty(t.numel() + 1, dtype=t.dtype, device=gpu)[1:].view(t.shape).copy_(t)
        if which == 3:  # columns apart
            return torch.stack([t, t], -1)[..., 0]
        if which == 4:  # rows in another order of dimensions
            return t.permute(2, 0, 3, 1).contiguous().permute(1, 3, 0, 2)
        return torch.nn.functional.pad(t, (0, 3))[..., :d]  # rows of 67

    want = dense.dense_attention_fwd(q, k, v)
    grads = dense.dense_attention_bwd(dy, q, k, v, *want)
    args = [odd(t) for t in (q, k, v)]
    got = dense.dense_attention_fwd(*args)
    for a, c in zip(got, want):
        assert torch.equal(a, c)
    for a, c in zip(dense.dense_attention_bwd(odd(dy), *args, odd(want[0]), odd(want[1]), want[2].mT.contiguous().mT), grads):
        assert torch.equal(a, c)


def test_broadcast_operands(gpu):
    """Keys expanded over the batch, and one incoming row for all queries."""
    q, k, v, dy = make(12, 2, 2, 2, 40, 60, 64, BF, gpu)
    check(q, k[:1].expand(2, -1, -1, -1), v[:1].expand(2, -1, -1, -1), dy[:, :, :1].expand(-1, -1, 40, -1))


def test_empty_calls(gpu):
    from svoo_amd import dense

    for b, h, kh, sq, sk in ((0, 2, 2, 5, 5), (2, 0, 0, 5, 5), (2, 2, 2, 0, 5), (2, 2, 2, 5, 0)):
        q, k, v, dy = (torch.randn(b, n, s, 64, device=gpu).to(BF).requires_grad_() for n, s in
                       ((h, sq), (kh, sk), (kh, sk), (h, sq)))
        o = dense.dense_attention(q, k, v)
        assert o.shape == q.shape and not o.any()
        for t, g in zip((q, k, v), torch.autograd.grad(o, [q, k, v], dy)):
            assert g.shape == t.shape and not g.any()


def test_only_the_gradients_asked_for(gpu):
    from svoo_amd import dense

    q, k, v, dy = make(13, 1, 2, 2, 70, 80, 64, BF, gpu)
    o, rest, lse = dense.dense_attention_fwd(q, k, v)
    want = dense.dense_attention_bwd(dy, q, k, v, o, rest, lse)
    for needs in ((True, False, False), (False, True, False), (False, False, True), (False, False, False)):
        for got, w, need in zip(dense.dense_attention_bwd(dy, q, k, v, o, rest, lse, needs=needs), want, needs):
            assert (got is None) == (not need) and (not need or torch.equal(got, w))
    frozen = k.detach()
    leaf = q.detach().requires_grad_()
    assert torch.equal(torch.autograd.grad(dense.dense_attention(leaf, frozen, v), leaf, dy)[0], want[0])


def test_gradients_against_differences(gpu):
    """The loss along a direction, by differences of float64 attention, against the kernels' gradients."""
    from svoo_amd import dense

    q, k, v, dy = make(14, 1, 2, 1, 60, 100, 64, BF, gpu)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(dense.dense_attention(*leaves), leaves, dy)
    g = torch.Generator().manual_seed(1)
    base = [t.detach().double().cpu() for t in (q, k, v)]
    for i in range(3):
        way = torch.randn(base[i].shape, generator=g).double()

        def loss(e):
            at = list(base)
            at[i] = at[i] + e * way
            return (attention64(*at)["o"][0] * dy.double().cpu()).sum()

        slope = (loss(1e-4) - loss(-1e-4)) / 2e-4
        got = (grads[i].double().cpu() * way).sum()
        # the two bounds of a sum over a random direction: each gradient's own rounding and bound
        bound = attention64(q, k, v, dy)[("dq", "dk", "dv")[i]][1]
        room = ((bound + HALF[BF] * grads[i].double().cpu().abs()) * way.abs()).sum()
        assert abs(got - slope) <= room + 1e-6 * abs(slope)


def test_not_finite_values_stay_in_their_rows(gpu):
    from svoo_amd import dense

    q, k, v, dy = make(15, 2, 2, 2, 80, 90, 64, BF, gpu)
    clean = dense.dense_attention(q, k, v)
    q2 = q.clone()
    q2[0, 1, 7, 3] = math.nan
    o = dense.dense_attention(q2, k, v)
    bad = torch.zeros(2, 2, 80, dtype=torch.bool, device=gpu)
    bad[0, 1, 7] = True
    assert o[bad].isnan().all() and torch.equal(o[~bad], clean[~bad])
    v2 = v.clone()
    v2[1, 0, 5, 9] = math.inf
    o = dense.dense_attention(q, k, v2)
    assert (o[1, 0, :, 9] == math.inf).all()
    o[1, 0, :, 9] = clean[1, 0, :, 9]
    assert torch.equal(o, clean)


def test_the_same_call_gives_the_same_bits(gpu):
    from svoo_amd import dense

    q, k, v, dy = make(16, 1, 4, 2, 900, 5000, 128, BF, gpu)
    first = dense.dense_attention_fwd(q, k, v)
    grads = dense.dense_attention_bwd(dy, q, k, v, *first)
    for _ in range(3):
        again = dense.dense_attention_fwd(q, k, v)
        assert all(torch.equal(a, b) for a, b in zip(first, again))
        assert all(torch.equal(a, b) for a, b in zip(grads, dense.dense_attention_bwd(dy, q, k, v, *again)))


def test_streams_and_two_calls_at_once(gpu):
    from svoo_amd import dense

    a, b = make(17, 1, 2, 2, 40, 9000, 128, BF, gpu), make(18, 1, 2, 2, 40, 9000, 128, BF, gpu)
    want = [dense.dense_attention_bwd(t[3], *t[:3], *dense.dense_attention_fwd(*t[:3])) for t in (a, b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(gpu) for _ in range(2)]
    got = [None, None]
    for i, (s, t) in enumerate(zip(streams, (a, b))):
        with torch.cuda.stream(s):
            got[i] = dense.dense_attention_bwd(t[3], *t[:3], *dense.dense_attention_fwd(*t[:3]))
    torch.cuda.synchronize()
    for x, y in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(x, y))


def test_captured_and_replayed(gpu):
    """A graph of both passes, replayed on new inputs, with eager calls in between."""
    from svoo_amd import dense

    args = make(19, 2, 2, 1, 300, 2000, 128, FP, gpu)
    k_lens = torch.tensor([2000, 700], dtype=torch.int32, device=gpu)

    def step(q, k, v, dy):
        o, rest, lse = dense.dense_attention_fwd(q, k, v, k_lens=k_lens)
        return [o, *dense.dense_attention_bwd(dy, q, k, v, o, rest, lse, k_lens=k_lens)]

    side = torch.cuda.Stream(gpu)
    side.wait_stream(torch.cuda.current_stream(gpu))
    with torch.cuda.stream(side):
        step(*args)
    torch.cuda.current_stream(gpu).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*args)
    for seed in (20, 21, 22):
        for t, n in zip(args, make(seed, 2, 2, 1, 300, 2000, 128, FP, gpu)):
            t.copy_(n)
        k_lens.copy_(torch.tensor([seed, 2000], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step(*args)):
            assert torch.equal(a, b)


def test_offsets_past_32_bits(gpu):
    """Rows 16 MB apart, and batch entries further: operands in a buffer of 12 GB give the bits of packed ones."""
    from svoo_amd import dense

    q, k, v, dy = (t.contiguous() for t in make(23, 2, 1, 1, 90, 350, 64, BF, gpu))
    want = dense.dense_attention_fwd(q, k, v)
    grads = dense.dense_attention_bwd(dy, q, k, v, *want)
    row = (1 << 23) - 8
    buffer = torch.empty(2 * 350 * row, dtype=BF, device=gpu)
    # every operand has 64 columns of its own in each row
    apart = [buffer.as_strided(t.shape, (350 * row, 0, row, 1), 64 * i).copy_(t) for i, t in enumerate((q, k, v, dy, want[0]))]
    got = dense.dense_attention_fwd(*apart[:3])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for a, b in zip(dense.dense_attention_bwd(apart[3], *apart[:3], apart[4], want[1], want[2]), grads):
        assert torch.equal(a, b)


def test_rows_too_far_apart_are_copied(gpu):
    from svoo_amd import dense

    q, k, v, _ = (t.contiguous() for t in make(24, 1, 1, 1, 20, 30, 64, BF, gpu))
    far = torch.empty(30 << 23, dtype=BF, device=gpu).as_strided(k.shape, (0, 0, 1 << 23, 1)).copy_(k)
    assert torch.equal(dense.dense_attention(q, far, v), dense.dense_attention(q, k, v))


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("sq,sk", [(100, 1500), (3, 9000), (600, 4000), (1700, 130)])
def test_lengths_that_leave_shares_empty(gpu, sq, sk, dtype):
    """A long axis is split into a few shares or many, of which a short sequence fills the first ones only."""
    say("shares", sq, sk, dtype)
    q, k, v, dy = make(25, 4, 2, 1, sq, sk, 64, dtype, gpu)
    check(q, k, v, dy, q_lens=lens([sq, sq, (sq + 1) // 2, 0], gpu), k_lens=lens([sk, 65, 0, sk], gpu))


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("d,sk", [(64, 70), (128, 600), (40, 1)])
def test_many_blocks(gpu, d, sk, dtype):
    """More blocks than a few rounds of all CUs, of one tile of queries each."""
    say("many blocks", d, sk, dtype)
    check(*make(26, 5, 230, 46, 9, sk, d, dtype, gpu))
