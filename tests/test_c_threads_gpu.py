"""The C ABI from several host threads (ctypes gives up the interpreter lock
during a call): calls of different sizes that run the same kernel, each thread
on its stream; and one captured graph that holds two sizes of a kernel."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def rnd(shape, seed, std=1.0, dtype=BF):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, device="cuda", generator=g) * std).to(dtype)


def linear_call(pkg, m, n, k):
    """(a call on a stream, its outputs)"""
    lib, ops = pkg._lib.load(), pkg.ops
    x = rnd((m, k), m + k)
    qw, sw = ops.mx_quantize(rnd((n, k), n, 0.05))
    qx, sx = ops.mx_quantize(x)
    y = torch.zeros(m, n, device="cuda", dtype=BF)
    keep = (x, qw, sw, qx, sx)
    args = (x.data_ptr(), qw.data_ptr(), sw.data_ptr(), None, qx.data_ptr(), sx.data_ptr(), y.data_ptr(), m, n, k, k)
    return (lambda st, keep=keep: lib.nvfp4b200_mx_linear(*args, st)), [y]


def norm_calls(pkg, t, d, dtype=BF):
    lib, ops = pkg._lib.load(), pkg.ops
    code = {BF: 0, torch.float32: 1}[dtype]
    b, x, dy, dn = (rnd((t, d), i, 1.0, dtype) for i in range(4))
    gp, gn = rnd((d,), 5, 1.0, dtype), rnd((d,), 6, 1.0, dtype)
    y, n, ib, iy = ops.sandwich_norm(b, x, gp, None, gn)
    outs = [torch.zeros_like(b), torch.zeros_like(b), torch.zeros(d, device="cuda"), torch.zeros(d, device="cuda"),
            torch.zeros_like(b), torch.zeros_like(b), torch.zeros(t, device="cuda"), torch.zeros(t, device="cuda")]
    words = torch.zeros(1, dtype=torch.int64)
    import ctypes
    w = ctypes.c_int64()
    assert lib.nvfp4b200_sandwich_norm_bwd_ws(t, d, 0, ctypes.byref(w)) == 0
    ws = torch.empty(w.value, device="cuda")
    keep = (b, x, dy, dn, gp, gn, y, ib, iy, ws, words)
    bwd = (dy.data_ptr(), dn.data_ptr(), b.data_ptr(), y.data_ptr(), ib.data_ptr(), iy.data_ptr(), gp.data_ptr(), None, gn.data_ptr(),
           outs[0].data_ptr(), outs[1].data_ptr(), outs[2].data_ptr(), None, outs[3].data_ptr(), ws.data_ptr(), w.value, code, t, d, 0,
           d, d, d, d, 1.0, 1.0)
    fwd = (b.data_ptr(), x.data_ptr(), gp.data_ptr(), None, gn.data_ptr(), outs[4].data_ptr(), outs[5].data_ptr(), outs[6].data_ptr(),
           outs[7].data_ptr(), code, t, d, 0, d, d, 1.0, 1.0, 1e-6)
    return (lambda st, keep=keep: lib.nvfp4b200_sandwich_norm_bwd(*bwd, st) or lib.nvfp4b200_sandwich_norm(*fwd, st)), outs


def sets(pkg):
    """Pairs of sizes that run one kernel with different amounts of shared memory."""
    return {
        "product": [linear_call(pkg, 16, 4096, 2048), linear_call(pkg, 16, 4096, 16384), linear_call(pkg, 16, 1024, 8192)],
        "product, tokens inside": [linear_call(pkg, 1, 4096, 2048), linear_call(pkg, 1, 4096, 16384), linear_call(pkg, 1, 1024, 32768)],
        "norms": [norm_calls(pkg, 64, 2072), norm_calls(pkg, 64, 2552), norm_calls(pkg, 64, 2304)],
        "norms, odd widths": [norm_calls(pkg, 64, 2071), norm_calls(pkg, 64, 2553), norm_calls(pkg, 64, 2303)],
        "norms, long rows": [norm_calls(pkg, 64, 5128), norm_calls(pkg, 64, 8192), norm_calls(pkg, 64, 6144)],
    }


@pytest.mark.parametrize("name", ["product", "product, tokens inside", "norms", "norms, odd widths", "norms, long rows"])
def test_sizes_from_several_threads(pkg, name):
    calls = sets(pkg)[name]
    want = []
    for call, outs in calls:
        assert call(torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()
        want.append([o.clone() for o in outs])
        for o in outs:
            o.zero_()
    torch.cuda.synchronize()
    bad = []

    def work(call):
        st = torch.cuda.Stream()
        for _ in range(1500):
            rc = call(st.cuda_stream)
            if rc:
                bad.append(rc)
        st.synchronize()

    threads = [threading.Thread(target=work, args=(c,)) for c, _ in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not bad, (len(bad), bad[:3])
    for (_, outs), ref in zip(calls, want):
        assert all(torch.equal(o, r) for o, r in zip(outs, ref))
    assert pkg.ops.device_error() == 0


def test_two_sizes_in_one_graph(pkg):
    """The larger size first, then the smaller, captured; the smaller once more before
    the graph runs."""
    calls = [c for pair in sets(pkg).values() for c in sorted(pair, key=lambda c: -c[1][0].numel())]
    want = []
    for call, outs in calls:
        assert call(torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()
        want.append([o.clone() for o in outs])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for call, _ in calls:
            assert call(torch.cuda.current_stream().cuda_stream) == 0
    for call, _ in reversed(calls):
        assert call(torch.cuda.current_stream().cuda_stream) == 0
    for rep in range(3):
        for _, outs in calls:
            for o in outs:
                o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for (_, outs), ref in zip(calls, want):
            assert all(torch.equal(o, r) for o, r in zip(outs, ref)), rep
    assert pkg.ops.device_error() == 0
