"""Gradients of a layer norm's parameters in every form that a parameter may have, against the formula in 64 bits."""

import pytest
import torch

from norm_fp8_helpers import U32, norm64, say, within

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _terms(x, dy, eps=1e-6):
    """The terms of both parameters' gradients, and the sizes that their errors are relative to."""
    n, _, _ = norm64(x.double(), 1, 0, eps)
    d = dy.double()
    return (d * n, d.abs() * (n.abs() + 1)), (d, d.abs())


FORMS = [("expanded", "expanded"), ("rows", "rows"), ("expanded", None), (None, "rows"), ("expanded", "own"), ("own", "rows"),
         ("expanded", "shared"), ("shared", "rows"), ("shared", "own"), ("own", None)]


@pytest.mark.parametrize("batch,rows,cols", [(3, 5, 16), (3, 700, 136), (2, 33, 2056), (5, 1, 999)])
@pytest.mark.parametrize("names", [("scale", "shift"), ("weight", "bias")])
def test_gradients_of_expanded_parameters(gpu, batch, rows, cols, names):
    """Parameters whose batch entries share memory, beside others: each entry's gradient, and the leaf's through autograd."""
    from svoo_amd import norm

    g = torch.Generator(device=gpu).manual_seed(cols + rows)
    x = torch.randn(batch, rows, cols, generator=g, device=gpu).to(BF16)
    dy = (0.1 * torch.randn(batch, rows, cols, generator=g, device=gpu)).to(BF16)
    terms = _terms(x, dy)
    for kinds in FORMS:
        leaves, params = [], {}
        for name, kind in zip(names, kinds):
            if kind is None:
                continue
            shape = (batch, 1, cols) if kind == "own" else (cols,)
            leaf = (0.3 * torch.randn(shape, generator=g, device=gpu)).requires_grad_()
            leaves.append((leaf, names.index(name), kind))
            params[name] = leaf.expand(batch, 1, cols) if kind == "expanded" else \
                leaf.expand(batch, cols) if kind == "rows" else leaf
        say("expanded parameters", batch, rows, cols, names, kinds)
        y = norm.layer_norm(x, **params)
        gain, offset = (torch.zeros(1, 1, cols, dtype=torch.float64, device=gpu) if name not in params else
                        params[name].detach().double().reshape(-1, 1, cols) for name in names)
        gain = gain if "weight" in params else 1 + gain
        n, _, want = norm64(x.double(), gain, offset, 1e-6)
        # as in the other tests of the forward pass: 80 U of |n| + 1, and four roundings
        within(y, want, 80 * U32 * (n.abs() + 1) * gain.abs() + 4 * U32 * (want.abs() + offset.abs()))
        # each entry's own gradient: 80 U of a term's size, one rounding per added row (and, of a parameter shared beside
        # one that is not, per entry)
        _, mean, rstd = norm.layer_norm_fwd(x, **{k: p.detach() for k, p in params.items()})
        grads = norm.layer_norm_bwd(dy, x, mean, rstd, **{k: p.detach() for k, p in params.items()})[1:]
        for name, got, (term, size), kind in zip(names, grads, terms, kinds):
            if kind is None:
                assert got is None
                continue
            over = (0, 1) if kind == "shared" else (1,)
            shape = params[name].shape
            assert got.shape == shape and got.dtype == F32
            within(got, term.sum(over).reshape(shape), ((80 + batch * rows) * U32 * size.sum(over)).reshape(shape))
        # the leaf's: the entries' sum, of as many more additions
        for (leaf, which, kind), got in zip(leaves, torch.autograd.grad(y, [leaf for leaf, _, _ in leaves], dy)):
            term, size = terms[which]
            over = (1,) if kind == "own" else (0, 1)
            assert got.shape == leaf.shape
            within(got, term.sum(over).reshape(leaf.shape),
                   ((80 + batch * rows + batch) * U32 * size.sum(over)).reshape(leaf.shape))


def test_gradients_of_expanded_16_bit_parameters(gpu):
    """The gradient has the parameter's type, one rounding from the sum."""
    from svoo_amd import norm

    g = torch.Generator(device=gpu).manual_seed(1)
    x = torch.randn(4, 9, 264, generator=g, device=gpu).to(F16)
    dy = (0.1 * torch.randn(4, 9, 264, generator=g, device=gpu)).to(F16)
    sc = torch.randn(264, generator=g, device=gpu).to(BF16).expand(4, 264)
    sh = torch.randn(4, 264, generator=g, device=gpu).to(F16)
    _, mean, rstd = norm.layer_norm_fwd(x, scale=sc, shift=sh)
    grads = norm.layer_norm_bwd(dy, x, mean, rstd, scale=sc, shift=sh)[1:]
    for got, p, (term, size) in zip(grads, (sc, sh), _terms(x, dy)):
        assert got.shape == p.shape and got.dtype == p.dtype
        within(got, term.sum(1), 100 * U32 * size.sum(1))


def _memset_nodes(graph):
    """How many nodes of a captured graph clear memory."""
    import ctypes

    hip = ctypes.CDLL("libamdhip64.so")
    h, n = ctypes.c_void_p(graph.raw_cuda_graph()), ctypes.c_size_t()
    assert hip.hipGraphGetNodes(h, None, ctypes.byref(n)) == 0
    nodes = (ctypes.c_void_p * n.value)()
    assert hip.hipGraphGetNodes(h, nodes, ctypes.byref(n)) == 0
    count = 0
    for node in nodes:
        kind = ctypes.c_int()
        assert hip.hipGraphNodeGetType(ctypes.c_void_p(node), ctypes.byref(kind)) == 0
        count += kind.value == 2  # hipGraphNodeTypeMemset
    return count


@pytest.mark.parametrize("batch,rows,cols", [(3, 21, 136), (3000, 2, 64), (20000, 1, 9), (700, 3, 1536)])
def test_shared_gradients_in_a_graph(gpu, batch, rows, cols):
    """A parameter shared by many entries beside one that is not, captured: only kernels, and every replay is the eager
    result, with eager work between."""
    from svoo_amd import norm

    g = torch.Generator(device=gpu).manual_seed(batch)
    draw = lambda *s: torch.randn(*s, generator=g, device=gpu)  # noqa: E731
    data = [(draw(batch, rows, cols).to(BF16), draw(batch, rows, cols).to(BF16), 0.3 * draw(batch, 1, cols), 0.3 * draw(cols))
            for _ in range(2)]

    def step(x, dy, sc, sh):
        y, mean, rstd = norm.layer_norm_fwd(x, scale=sc, shift=sh)
        return (y, *norm.layer_norm_bwd(dy, x, mean, rstd, scale=sc, shift=sh))

    say("shared gradients in a graph", batch, rows, cols)
    want = [step(*d) for d in data]
    for (x, dy, _, _), (_, _, dsc, dsh) in zip(data, want):
        (term, size), (d, d_size) = _terms(x, dy)
        within(dsc.view(batch, cols), term.sum(1), (80 + rows) * U32 * size.sum(1))
        within(dsh, d.sum((0, 1)), (80 + rows + batch) * U32 * d_size.sum((0, 1)))
    held = [t.clone() for t in data[0]]
    step(*held)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        out = step(*held)
    assert _memset_nodes(graph) == 0
    graph.instantiate()
    for i in range(4):
        for h, t in zip(held, data[i % 2]):
            h.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want[i % 2])), i
        assert all(torch.equal(a, b) for a, b in zip(step(*data[1]), want[1]))


@pytest.mark.parametrize("batch,cols", [((1 << 22) + 5, 9), ((1 << 24) - 1, 8)])
def test_parameters_of_millions_of_batch_entries(gpu, batch, cols):
    """A row and a parameter each: as in calls of the ends alone."""
    from svoo_amd import norm

    g = torch.Generator(device=gpu).manual_seed(cols)
    x, dy = (torch.randn(batch, cols, generator=g, device=gpu).to(BF16) for _ in range(2))
    sc, sh = (torch.randn(batch, cols, generator=g, device=gpu) for _ in range(2))
    say("millions of entries", batch, cols)
    y, mean, rstd = norm.layer_norm_fwd(x, scale=sc, shift=sh)
    grads = norm.layer_norm_bwd(dy, x, mean, rstd, scale=sc, shift=sh)
    for at in (slice(0, 100), slice(batch // 2, batch // 2 + 100), slice(batch - 100, batch)):
        y1, mean1, rstd1 = norm.layer_norm_fwd(x[at], scale=sc[at], shift=sh[at])
        assert torch.equal(y[at], y1) and torch.equal(mean[at], mean1) and torch.equal(rstd[at], rstd1)
        ends = norm.layer_norm_bwd(dy[at], x[at], mean1, rstd1, scale=sc[at], shift=sh[at])
        assert all(torch.equal(a[at], b) for a, b in zip(grads, ends))
    assert torch.equal(grads[2], dy.float())  # one row an entry
