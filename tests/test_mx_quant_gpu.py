"""GPU parity of the MXFP4 quantizers, the way back, and the MXFP4 linear layer.

Quantizers: every code and nibble equals the numpy restatement
(oracle/mx_oracle.py), except the nibbles of a block that holds an infinity or
a NaN, which mean nothing.  The products of the factors (row scale, norm
weight) are rounded once each in fp32, in that order, so the restatement takes
them in float32 and stays exact.  Products: within one bf16 rounding (2^-8
relative) of the float64 product of the same operands, plus 2^-20 of the sum
of the terms' magnitudes for fp32 accumulation (fp32 outputs: the latter only).
"""
import numpy as np
import pytest
import torch

from oracle import mx_oracle as mxo, nvfp4_oracle as orc

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def host(t):
    return t.detach().cpu().view(torch.uint8).numpy()


def f64(t):
    return t.detach().double().cpu().numpy()


def make(r, c, dtype, seed=0, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed + 31 * r + c)
    x = torch.randn(r, c, device="cuda", generator=g)
    return (x * torch.exp(spread * torch.randn(r, c, device="cuda", generator=g))).to(dtype)


def same(q, s, oq, os_, rows, k):
    """Codes equal everywhere, nibbles equal outside NaN blocks."""
    assert np.array_equal(host(s), os_)
    flat = os_.reshape(-1)
    rr, cc = np.meshgrid(np.arange(rows), np.arange(k // 32), indexing="ij")
    good = flat[orc.swizzle_offset(rr, cc, os_.shape[1])] != 255
    good = np.repeat(good, 16, axis=1)
    assert np.array_equal(host(q).reshape(rows, k // 2)[good], oq[good])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("r,c", [(1, 32), (3, 64), (31, 96), (32, 128), (33, 160), (127, 352), (129, 1024), (260, 2080)])
def test_orientations(pkg, r, c, dtype):
    x = make(r, c, dtype)
    x[0, :32] = 0
    ops = pkg.ops
    oq, os_ = mxo.quantize(f64(x))
    oqt, ost = mxo.quantize_t(f64(x))
    pr = -(-r // 32) * 32
    q, s = ops.mx_quantize(x)
    same(q, s, oq, os_, r, c)
    qt, st = ops.mx_quantize_t(x)
    same(qt, st, oqt, ost, c, pr)
    both = ops.mx_quantize_both(x)
    for a, b in zip(both, (q, s, qt, st)):
        assert torch.equal(a, b)
    for dt in (torch.bfloat16, torch.float32):
        assert np.array_equal(f64(ops.mx_dequantize(q, s, dt)), orc.dequant_mxfp4(oq, os_, r, c))
        assert np.array_equal(f64(ops.mx_dequantize(qt, st, dt)), orc.dequant_mxfp4(oqt, ost, c, pr))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("with_row,with_gamma", [(True, True), (True, False), (False, True)])
def test_factors(pkg, dtype, with_row, with_gamma):
    r, c = 77, 416
    x = make(r, c, dtype, 5)
    row = torch.rand(r, device="cuda") + 0.3 if with_row else None
    gam = (torch.randn(c, device="cuda") * 0.2 + 1).to(torch.bfloat16) if with_gamma else None
    v = x.float().cpu().numpy()
    if with_row:
        v = v * row.cpu().numpy()[:, None]
    if with_gamma:
        v = v * gam.float().cpu().numpy()
    assert v.dtype == np.float32
    q, s, qt, st = pkg.ops.mx_quantize_both(x, row_scale=row, gamma=gam)
    same(q, s, *mxo.quantize(v), r, c)
    same(qt, st, *mxo.quantize_t(v), c, 96)


def test_ties_extremes_and_non_finite(pkg):
    """Every tie point and its neighbours at several exponents, signed zeros,
    subnormals, the largest values, infinities and NaN."""
    rows = []
    for e in (-126, -30, -3, 0, 5, 100):
        t = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=np.float32)
        vals = np.concatenate([t, np.nextafter(t, np.float32(9)), np.nextafter(t, np.float32(0)), -t, [6.0, -0.0, 0.0, 7.9]])
        rows.append(np.ldexp(vals.astype(np.float32), e))
    rows.append(np.float32([3.4e38, -3.4e38, 1e38] + [0] * 29))
    rows.append(np.float32([1e-45, 1e-40, 1.2e-38, -1e-39] + [0] * 28))
    rows.append(np.float32([np.inf] + [1] * 31))
    rows.append(np.float32([1] * 31 + [np.nan]))
    rows.append(np.float32([-np.inf, np.nan] + [3] * 30))
    x = np.stack([np.concatenate([r, np.roll(r, 5)]) for r in rows]).astype(np.float32)
    for dt in (torch.float32, torch.bfloat16):
        t = torch.from_numpy(x).to(dt).cuda()
        q, s, qt, st = pkg.ops.mx_quantize_both(t)
        v = f64(t)
        same(q, s, *mxo.quantize(v), *x.shape)
        same(qt, st, *mxo.quantize_t(v), x.shape[1], 32)
        d = f64(pkg.ops.mx_dequantize(q, s))
        ref = orc.dequant_mxfp4(*mxo.quantize(v), *x.shape)
        bad = ~np.isfinite(v).reshape(len(x), 2, 32).all(2)
        assert np.array_equal(np.isnan(d), np.repeat(bad, 32, axis=1))
        assert np.array_equal(d[~np.isnan(d)], ref[~np.isnan(d)])


def test_strided_misaligned_and_transposed_inputs(pkg):
    big = make(70, 512, torch.bfloat16, 9)
    for x in (big[:, 64:192], big[3:40, 128:256], big[:, ::2][:, :128], big[:64, :].t(), big.view(-1)[1:1 + 64 * 96].view(64, 96),
              big[:1, :64].expand(40, 64)):
        q, s, qt, st = pkg.ops.mx_quantize_both(x)
        r, c = x.shape
        same(q, s, *mxo.quantize(f64(x)), r, c)
        same(qt, st, *mxo.quantize_t(f64(x)), c, -(-r // 32) * 32)


def test_out_tensors_and_no_rows(pkg):
    ops = pkg.ops
    x = make(40, 96, torch.bfloat16, 2)
    q, s = ops.mx_quantize(x)
    out = (torch.full_like(q, 7), torch.full_like(s, 7))
    ops.mx_quantize(x, out=out)
    assert torch.equal(out[0], q) and torch.equal(out[1], s)
    qt, st = ops.mx_quantize_t(x)
    out = (torch.full_like(qt, 7), torch.full_like(st, 7))
    ops.mx_quantize_t(x, out=out)
    assert torch.equal(out[0], qt) and torch.equal(out[1], st)
    q, s, qt, st = ops.mx_quantize_both(x[:0])
    assert q.shape == (0, 48) and qt.shape == (96, 0)
    assert ops.mx_dequantize(q, s).shape == (0, 96) and ops.mx_dequantize(qt, st).shape == (96, 0)
    assert pkg.ops.mx_linear(x[:0], *ops.mx_quantize(make(24, 96, torch.bfloat16))).shape == (0, 24)


def test_wide_and_long(pkg):
    """Many row tiles and odd tails: sampled rows of 70001 x 1056 against the restatement."""
    x = make(70001, 1056, torch.bfloat16, 3)
    q, s, qt, st = pkg.ops.mx_quantize_both(x)
    d = pkg.ops.mx_dequantize(q, s)
    dt = pkg.ops.mx_dequantize(qt, st)
    rows = torch.tensor([0, 1, 127, 128, 65535, 65536, 69999, 70000], device="cuda")
    ref = orc.dequant_mxfp4(*mxo.quantize(f64(x[rows])), len(rows), 1056)
    assert np.array_equal(f64(d[rows]), ref)
    cols = torch.tensor([0, 5, 1023, 1024, 1055], device="cuda")
    sub = f64(x[:, cols])
    ref = orc.dequant_mxfp4(*mxo.quantize_t(sub), len(cols), 70016)
    assert np.array_equal(f64(dt[cols]), ref)


def test_offsets_past_32_bits(pkg):
    """More than 2^31 elements: sampled rows and columns of both orientations."""
    r, c = 66000, 32768
    x = torch.empty(r, c, device="cuda", dtype=torch.bfloat16)
    for lo in range(0, r, 11000):
        x[lo:lo + 11000] = make(11000, c, torch.bfloat16, lo)
    rows = torch.tensor([0, 65535, 65536, 65999], device="cuda")
    cols = torch.tensor([0, 17, 32767], device="cuda")
    q, s, qt, st = pkg.ops.mx_quantize_both(x)
    xr, xc = f64(x[rows]), f64(x[:, cols])
    del x
    d = pkg.ops.mx_dequantize(q, s)
    assert np.array_equal(f64(d[rows]), orc.dequant_mxfp4(*mxo.quantize(xr), len(rows), c))
    del d, q, s
    d = pkg.ops.mx_dequantize(qt, st)
    assert np.array_equal(f64(d[cols]), orc.dequant_mxfp4(*mxo.quantize_t(xc), len(cols), d.shape[1]))


def product(qa, sa, qb, sb, m, n, k):
    a = orc.dequant_mxfp4(host(qa), host(sa), m, k)
    b = orc.dequant_mxfp4(host(qb), host(sb), n, k)
    return a @ b.T, np.abs(a) @ np.abs(b).T


def check(d, ref, mag, bf16=True):
    tol = (np.abs(ref) * 2.0 ** -8 if bf16 else 0) + mag * 2.0 ** -20 + 1e-30
    err = np.abs(f64(d) - ref)
    assert (err <= tol).all(), float((err - tol).max())


@pytest.mark.parametrize("m,n,k", [(1, 8, 32), (1, 4096, 1024), (2, 264, 96), (3, 520, 4096), (7, 1000, 352), (8, 2048, 2048),
                                   (9, 128, 14336), (16, 136, 512), (17, 640, 1056), (31, 256, 256), (33, 384, 640),
                                   (64, 1032, 288), (65, 136, 1024), (129, 256, 96), (300, 520, 1024), (257, 4096, 2048), (1000, 1024, 512),
                                                   (700, 4608, 256)])
@pytest.mark.parametrize("with_bias", [False, True])
def test_mx_linear(pkg, m, n, k, with_bias):
    ops = pkg.ops
    x, w = make(m, k, torch.bfloat16, 1), make(n, k, torch.bfloat16, 2) * 0.05
    bias = (torch.randn(n, device="cuda") * 3).to(torch.bfloat16) if with_bias else None
    qw, sw = ops.mx_quantize(w)
    y = ops.mx_linear(x, qw, sw, bias=bias)
    assert ops.device_error() == 0
    ref, mag = product(*ops.mx_quantize(x), qw, sw, m, n, k)
    if with_bias:
        ref, mag = ref + f64(bias), mag + np.abs(f64(bias))
    assert y.dtype == torch.bfloat16 and y.shape == (m, n)
    check(y, ref, mag)
    y3 = ops.mx_linear(x.view(1, m, k), qw, sw, bias=bias)
    assert y3.shape == (1, m, n) and torch.equal(y3[0], y)


def test_mx_linear_strided_input_and_nan_rows(pkg):
    """A row that holds a NaN gives a NaN row and leaves the others alone."""
    ops = pkg.ops
    big = make(12, 1024, torch.bfloat16, 8)
    big[2, 700] = float("nan")
    big[5, 513] = float("inf")
    w = make(256, 512, torch.bfloat16, 4)
    qw, sw = ops.mx_quantize(w)
    y = ops.mx_linear(big[:, 512:], qw, sw)
    ref = ops.mx_linear(torch.nan_to_num(big[:, 512:], 0, 0, 0).contiguous(), qw, sw)
    bad = torch.zeros(12, dtype=torch.bool, device="cuda")
    bad[[2, 5]] = True
    assert torch.isnan(y[bad]).all() and torch.equal(y[~bad], ref[~bad])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t,n,k", [(1, 32, 64), (5, 96, 32), (33, 160, 256), (200, 288, 512), (777, 512, 288)])
def test_linear_forward_backward(pkg, f4, t, n, k, dtype):
    ops = pkg.ops
    x = make(t, k, dtype, 1).requires_grad_()
    w = (make(n, k, dtype, 2) * 0.05).requires_grad_()
    bias = torch.randn(n, device="cuda").to(dtype).requires_grad_()
    dy = make(t, n, dtype, 3)
    y = f4.mxfp4_linear(x, w, bias)
    dx, dw, db = torch.autograd.grad(y, (x, w, bias), dy)
    bf = dtype == torch.bfloat16
    pt = -(-t // 32) * 32
    xd, wd = x.detach(), w.detach()
    b16 = f64(bias.detach().to(torch.bfloat16))
    ref, mag = product(*ops.mx_quantize(xd), *ops.mx_quantize(wd), t, n, k)
    check(y, ref + b16, mag + np.abs(b16), bf)
    ref, mag = product(*ops.mx_quantize(dy), *ops.mx_quantize_t(wd), t, k, n)
    check(dx, ref, mag, bf)
    ref, mag = product(*ops.mx_quantize_t(dy), *ops.mx_quantize_t(xd), n, k, pt)
    check(dw, ref, mag, bf)
    ref = f64(dy).sum(0)
    assert (np.abs(f64(db) - ref) <= np.abs(ref) * (2.0 ** -8 if bf else 0) + np.abs(f64(dy)).sum(0) * 2.0 ** -18).all()
    assert y.dtype == dx.dtype == dw.dtype == dtype


def test_linear_module(pkg, f4):
    """Batched inputs, only some gradients, no tokens, frozen and thawed."""
    lin = f4.MXFP4Linear(128, 96, device="cuda")
    x = make(6, 128, torch.bfloat16, 1).view(2, 3, 128)
    y = lin(x)
    y.add_(1)                                  # the result may be changed in place
    y.sum().backward()
    assert lin.weight.grad.shape == (96, 128) and lin.bias.grad is not None
    lin.weight.requires_grad_(False)
    xg = x.clone().requires_grad_()
    lin(xg).sum().backward()
    assert xg.grad.shape == x.shape
    empty = torch.empty(0, 128, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    lin.weight.requires_grad_(True)
    lin.weight.grad = None
    lin(empty).sum().backward()
    assert empty.grad.shape == (0, 128) and (lin.weight.grad == 0).all()
    with torch.no_grad():
        ref = lin(x)
        lin.freeze()
        assert torch.equal(lin(x), ref)
        lin.weight.add_(1.0)
        assert torch.equal(lin(x), ref)        # held until thawed
        assert not torch.equal(lin.thaw()(x), ref)
        lin.freeze().load_state_dict(lin.state_dict())
        assert lin._held is None
    lin.freeze()
    with pytest.raises(RuntimeError):
        lin(xg)


def test_no_second_derivative(pkg, f4):
    x = make(32, 64, torch.bfloat16, 1).requires_grad_()
    w = make(32, 64, torch.bfloat16, 2).requires_grad_()
    y = f4.mxfp4_linear(x, w)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y.sum(), x, create_graph=True)
    with torch.no_grad():
        assert not f4.mxfp4_linear(x, w).requires_grad


def test_backward_twice_and_saved_tensor_hooks(pkg, f4):
    """retain_graph, and hooks that move what is kept (offloading): the same bits."""
    x = make(40, 64, torch.bfloat16, 1).requires_grad_()
    w = make(32, 64, torch.bfloat16, 2).requires_grad_()
    dy = make(40, 32, torch.bfloat16, 3)
    y = f4.mxfp4_linear(x, w)
    first = torch.autograd.grad(y, (x, w), dy, retain_graph=True)
    again = torch.autograd.grad(y, (x, w), dy)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.cuda()):
        z = f4.mxfp4_linear(x, w)
    moved = torch.autograd.grad(z, (x, w), dy)
    for a, b, c in zip(first, again, moved):
        assert torch.equal(a, b) and torch.equal(a, c)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y, (x, w), dy)     # freed


def test_gemm_forms(pkg):
    """fp32 store and accumulate, residual, ReLU epilogue, strided output."""
    ops = pkg.ops
    m, n, k = 150, 264, 320
    qa, sa = ops.mx_quantize(make(m, k, torch.bfloat16, 1))
    qb, sb = ops.mx_quantize(make(n, k, torch.bfloat16, 2))
    ref, mag = product(qa, sa, qb, sb, m, n, k)
    d = ops.mx_gemm(qa, sa, qb, sb, out_dtype=torch.float32)
    check(d, ref, mag, False)
    ops.mx_gemm(qa, sa, qb, sb, out=d, accumulate=True)
    check(d, 2 * ref, 2 * mag, False)
    res = make(m, n, torch.bfloat16, 3)
    check(ops.mx_gemm(qa, sa, qb, sb, residual=res), ref + f64(res), mag + np.abs(f64(res)))
    check(ops.mx_gemm(qa, sa, qb, sb, epilogue=ops.EPI_RELU), np.maximum(ref, 0), mag)
    wide = torch.full((m, 2 * n), 9.0, device="cuda", dtype=torch.bfloat16)
    ops.mx_gemm(qa, sa, qb, sb, out=wide[:, :n])
    check(wide[:, :n], ref, mag)
    assert (wide[:, n:] == 9).all()
    assert torch.equal(ops.mx_gemm(qa, sa, qb, sb), ops.mxfp4_mm(qa, sa, qb, sb))


def test_refusals(pkg, f4):
    ops = pkg.ops
    x = make(8, 64, torch.bfloat16)
    q, s = ops.mx_quantize(x)
    for call in (lambda: ops.mx_quantize(x[:, :40]), lambda: ops.mx_quantize_t(x[:, :12]), lambda: ops.mx_quantize(x[0]),
                 lambda: ops.mx_quantize(x.double()), lambda: ops.mx_quantize(x, gamma=x[0, :32]),
                 lambda: ops.mx_quantize(x, row_scale=torch.ones(3, device="cuda")),
                 lambda: ops.mx_quantize(x, out=(q[:4], s)), lambda: ops.mx_dequantize(q, s, torch.float16),
                 lambda: ops.mx_dequantize(q, s[:64]), lambda: ops.mx_gemm(q, s, q[:, :16], s),
                 lambda: ops.mx_gemm(q[:4], s, q[:4], s[:64]), lambda: ops.mx_gemm(q, s, q[:5].contiguous(), s),
                 lambda: ops.mx_linear(x[:, :32], q, s), lambda: ops.mx_linear(x.float(), q, s),
                 lambda: ops.mx_gemm(q, s, q, s, accumulate=True), lambda: f4.mxfp4_linear(x.half(), x.half()),
                 lambda: f4.mxfp4_linear(x.clone().requires_grad_(), make(40, 64, torch.bfloat16))):
        with pytest.raises(RuntimeError):
            call()


def test_other_stream_and_graph(pkg, f4):
    """On a stream of its own, and captured and replayed with new inputs."""
    ops = pkg.ops
    x, w = make(37, 512, torch.bfloat16, 1), make(640, 512, torch.bfloat16, 2)
    qw, sw = ops.mx_quantize(w)
    ref = ops.mx_linear(x, qw, sw)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        y = ops.mx_linear(x, qw, sw)
    torch.cuda.current_stream().wait_stream(st)
    assert torch.equal(y, ref)
    buf = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.mx_linear(buf, qw, sw)
        both = ops.mx_quantize_both(buf)
    for seed in (5, 6):
        new = make(37, 512, torch.bfloat16, seed)
        buf.copy_(new)
        graph.replay()
        assert torch.equal(out, ops.mx_linear(new, qw, sw))
        for a, b in zip(both, ops.mx_quantize_both(new)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("m", [1, 5, 12, 13, 40])
def test_linear_right_after_its_operands(pkg, m):
    """The product is launched while the kernel before it may still run: weights
    and tokens written just before must be the ones it reads, call after call,
    eagerly and replayed."""
    ops = pkg.ops
    n, k = 1024, 2048
    ws = [make(n, k, torch.bfloat16, s) for s in (1, 2, 3)]
    xs = [make(m, k, torch.bfloat16, s) for s in (4, 5, 6)]
    held = [ops.mx_quantize(w) for w in ws]
    torch.cuda.synchronize()
    ref = []
    for x, h in zip(xs, held):
        ref.append(ops.mx_linear(x, *h))
        torch.cuda.synchronize()
    buf_w, buf_x = ws[0].clone(), xs[0].clone()
    out = (torch.empty_like(held[0][0]), torch.empty_like(held[0][1]))

    def step(i):
        buf_w.copy_(ws[i])
        ops.mx_quantize(buf_w, out=out)          # the weights, just before
        y = ops.mx_linear(xs[i], *out)
        buf_x.copy_(xs[i])                       # the tokens, just before
        return y, ops.mx_linear(buf_x, *out)

    for rep in range(20):
        i = rep % 3
        for y in step(i):
            assert torch.equal(y, ref[i]), rep
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ys = [y for i in range(3) for y in step(i)]
    for _ in range(5):
        for y in ys:
            y.zero_()
        graph.replay()
        assert all(torch.equal(y, ref[j // 2]) for j, y in enumerate(ys))
    assert ops.device_error() == 0


def test_linear_on_two_streams_at_once(pkg):
    """Few-token products of both forms and a large one side by side."""
    ops = pkg.ops
    w = ops.mx_quantize(make(4096, 4096, torch.bfloat16, 1))
    xs = [make(m, 4096, torch.bfloat16, m) for m in (1, 30, 100, 300)]
    ref = [ops.mx_linear(x, *w) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    for _ in range(10):
        got = []
        for x, st in zip(xs, streams):
            with torch.cuda.stream(st):
                got.append(ops.mx_linear(x, *w))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, ref))
    assert ops.device_error() == 0


def test_no_output_features(pkg, f4):
    """A weight of no rows: an empty result, and gradients of zeros."""
    for shape in ((2, 3, 64), (5, 64), (0, 2, 64)):
        x = torch.randn(shape, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        w = torch.empty(0, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        b = torch.empty(0, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        y = f4.mxfp4_linear(x, w, b)
        assert y.shape == (*shape[:-1], 0)
        y.sum().backward()
        assert (x.grad == 0).all() and x.grad.shape == x.shape and w.grad.shape == w.shape and b.grad.shape == b.shape


@pytest.mark.parametrize("m", [1, 8, 37])
def test_chain_in_a_graph(pkg, m):
    """Layers one after another, captured: each result is the next call's input,
    its memory is used again two calls later, and every call may start early."""
    ops = pkg.ops
    k = 2048
    ws = [ops.mx_quantize(make(k, k, torch.bfloat16, s, 0.0) * k ** -0.5) for s in range(12)]
    xs = [make(m, k, torch.bfloat16, 20 + s, 0.0) for s in range(3)]
    ref = []
    for x in xs:
        for w in ws:
            x = ops.mx_linear(x, *w)
            torch.cuda.synchronize()
        ref.append(x)
        assert x.float().norm() > 0
    hold = xs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = hold
        for w in ws:
            y = ops.mx_linear(y, *w)
    for rep in range(30):
        hold.copy_(xs[rep % 3])
        graph.replay()
        assert torch.equal(y, ref[rep % 3]), rep
        z = xs[rep % 3]
        for w in ws:
            z = ops.mx_linear(z, *w)
        assert torch.equal(z, ref[rep % 3]), rep
