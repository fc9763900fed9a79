"""GEMM launches that run at the same time: captured graphs, streams, and more
captured launches than there are tile counters.  Every result has the bits of
the same product run alone."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def rnd(shape, seed, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, device="cuda", generator=g) * std).to(BF)


def test_two_graphs_of_the_trained_layer(pkg, f4):
    """A graph of mxfp4_linear with its backward, launches beyond the number of
    stream counters, a second graph: both replayed at once, beside an eager product."""
    ops = pkg.ops
    t, n, k = 4096, 4096, 2048      # 256, 128 and 128 tiles: several for every CTA pair

    def inputs(i):
        return rnd((t, k), 10 * i + 1), rnd((n, k), 10 * i + 2, 0.02), rnd((t, n), 10 * i + 3, 1e-2)

    def step(x, w, dy):
        x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
        y = f4.mxfp4_linear(x, w)
        return (y.detach(), *torch.autograd.grad(y, (x, w), dy))

    held = [inputs(i) for i in range(2)]
    ref = [step(*v) for v in held]
    qa, qb = ops.mx_quantize(held[0][0]), ops.mx_quantize(held[0][1])
    torch.cuda.synchronize()
    graphs, outs = [], []
    for v in held:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(*v))
        graphs.append(graph)
        for _ in range(300):
            y = ops.mx_gemm(*qa, *qb)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for rep in range(20):
        for o in outs:
            for v in o:
                v.zero_()
        torch.cuda.synchronize()
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
                graph.replay()
        with torch.cuda.stream(streams[2]):
            for _ in range(4):
                y = ops.mx_gemm(*qa, *qb)
        torch.cuda.synchronize()
        for o, r in zip(outs, ref):
            assert all(torch.equal(a, b) for a, b in zip(o, r)), rep
        assert torch.equal(y, ref[0][0]), rep
    assert ops.device_error() == 0


def test_many_launches_on_several_streams(pkg):
    """Queues of hundreds of products on four streams that run side by side."""
    ops = pkg.ops
    sets = []
    for i in range(4):
        qa, qb = ops.mx_quantize(rnd((2400 + 300 * i, 512), i)), ops.mx_quantize(rnd((4096, 512), 10 + i))
        sets.append((qa, qb, ops.mx_gemm(*qa, *qb)))
    outs = [[torch.zeros_like(r) for _ in range(3)] for _, _, r in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for i in range(300):
        for (qa, qb, _), o, st in zip(sets, outs, streams):
            with torch.cuda.stream(st):
                ops.mx_gemm(*qa, *qb, out=o[i % 3])
    torch.cuda.synchronize()
    for (_, _, r), o in zip(sets, outs):
        assert all(torch.equal(v, r) for v in o)
    assert ops.device_error() == 0


def test_more_captured_launches_than_counters(pkg):
    """The captured launches past the last counter walk their tiles in a fixed
    order; NVFP4 and MXFP4; a graph's counters serve again after it is gone."""
    ops = pkg.ops
    xa, xb = rnd((2560, 256), 1), rnd((2304, 256), 2)     # 90 tiles
    qa, qb = ops.mx_quantize(xa), ops.mx_quantize(xb)
    na, nb = ops.quantize(xa), ops.quantize(xb)
    ref, nref = ops.mx_gemm(*qa, *qb), ops.gemm(*na, *nb)
    for rep in range(2):
        outs = [torch.zeros_like(ref) for _ in range(4)]
        nout = torch.zeros_like(nref)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for i in range(8200):
                ops.mx_gemm(*qa, *qb, out=outs[i % 4])
            ops.gemm(*na, *nb, out=nout)
        for _ in range(2):
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, ref) for o in outs) and torch.equal(nout, nref)
        assert torch.equal(ops.mx_gemm(*qa, *qb), ref)
        del graph
    assert ops.device_error() == 0


def test_large_products_behind_dependent_launches(pkg):
    """Captured together: few-token products, which start while the kernel before
    them still runs, each right before a product of several tiles per CTA pair."""
    ops = pkg.ops
    w1, w2 = ops.mx_quantize(rnd((2048, 2048), 1, 0.02)), ops.mx_quantize(rnd((8192, 2048), 2, 0.02))
    tok, big = rnd((8, 2048), 3), ops.mx_quantize(rnd((2400, 2048), 4))
    more = rnd((100, 2048), 5)

    def chain():
        out = []
        for x in (tok, more):
            out += [ops.mx_linear(x, *w1), ops.mx_gemm(*big, *w2)]
        return out

    ref = chain()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(chain())
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for rep in range(10):
        for o in outs:
            for v in o:
                v.zero_()
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for o in outs:
            assert all(torch.equal(a, b) for a, b in zip(o, ref)), rep
    assert ops.device_error() == 0
