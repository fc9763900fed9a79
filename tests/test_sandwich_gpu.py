"""GPU parity of the norms after and before a block (sandwich_norm) and their
backward, against the formulas in float64 and against differences.

Tolerances.  A row's mean of squares, or of products, adds at most 16 terms in
a thread, 5 steps over lanes and up to 32 over warps: 53 roundings of 2^-24 of
the terms' magnitude, below 2^-18; rsqrtf adds two units in the last place.
Every element after that is a handful of fp32 products.  So each result is
within 2^-17 of the sum of its terms' magnitudes, plus the rounding to the
stored type (eps/2 relative, fp16: or half its smallest subnormal).  Column
sums of T rows add at most T further roundings, taken as (T + 64) * 2^-24 of
the sum of magnitudes."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF, HF, FL = torch.bfloat16, torch.float16, torch.float32
F32 = 2.0 ** -17


def rnd(shape, seed, dtype=FL, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, device="cuda", generator=g) * std).to(dtype)


def half_step(v, dtype):
    f = torch.finfo(dtype)
    return v.abs() * (f.eps / 2) + f.smallest_normal * f.eps / 2


def close(got, ref, mag, dtype=FL, extra=F32):
    tol = mag * extra + half_step(ref, dtype) + half_step(mag * extra, dtype)
    err = (got.double() - ref).abs()
    assert (err <= tol).all(), float((err / tol.clamp(min=1e-300)).max())


def expand(gate, t):
    return 1.0 if gate is None else gate.double().reshape(-1, gate.shape[-1]).repeat_interleave(t // gate.reshape(-1, gate.shape[-1]).shape[0], 0)


def one(p):
    return 1.0 if p is None else p.double()


def forward64(b, x, gp, gate, gn, al, s, eps):
    b, x = b.double(), x.double()
    ib = (b.square().mean(1) + eps).rsqrt()
    branch = s * expand(gate, b.shape[0]) * (b * ib[:, None]) * one(gp)
    return al * x + branch, ib, (al * x).abs() + branch.abs()


def backward64(dy, dn, b, y, ib, iy, gp, gate, gn, al, s):
    """Values, and the same with every difference turned into a sum (magnitudes)."""
    out = []
    for f in (lambda v: v, lambda v: v.abs()):
        sign = 1 if not out else -1
        t = f(dy.double()) if dy is not None else torch.zeros_like(b, dtype=torch.float64)
        dpre = None
        if dn is not None:
            yh, v = f(y.double() * iy.double()[:, None]), f(dn.double() * one(gn))
            t = t + iy.double()[:, None] * (v - sign * yh * (v * yh).mean(1, keepdim=True))
            dpre = (f(dn.double()) * yh).sum(0)
        bh = f(b.double() * ib.double()[:, None])
        g = expand(gate, b.shape[0])
        g = f(g) if gate is not None else g
        p = f(one(gp)) if gp is not None else 1.0
        e = abs(s) if sign < 0 else s
        u = e * t * g * p
        db = ib.double()[:, None] * (u - sign * bh * (u * bh).mean(1, keepdim=True))
        each = e * t * bh
        dgate = None if gate is None else (each * p).reshape(gate.reshape(-1, b.shape[1]).shape[0], -1, b.shape[1]).sum(1)
        out.append(dict(dx=(abs(al) if sign < 0 else al) * t, db=db, dgamma_post=(each * g).sum(0), dgate=dgate, dgamma_pre=dpre))
    return out


CASES = [  # t, d, groups, gamma_post, gamma_pre/pre
    (1, 1, 0, True, True), (1, 4096, 1, True, True), (5, 64, 5, True, True), (3, 333, 1, True, True),
    (16, 520, 4, False, True), (77, 1000, 7, True, False), (130, 2048, 1, True, True), (64, 4096, 16, True, True),
    (33, 5000, 0, True, True), (20, 8192, 2, True, True), (9, 16384, 3, True, True), (7, 16383, 1, True, True),
    (2000, 96, 1000, True, True), (1200, 256, 2, True, True), (1500, 8200, 1, True, True), (700, 12296, 7, True, True),
    (400, 16384, 0, True, False), (333, 1536, 3, True, True), (901, 2560, 1, True, True), (640, 5120, 1, True, True),
    (320, 5888, 0, True, True), (77, 1480, 1, True, False), (50, 2488, 50, True, True), (4099, 40, 1, True, True), (600, 512, 600, False, False)]


@pytest.mark.parametrize("dtype", [BF, HF, FL])
@pytest.mark.parametrize("t,d,g,post,pre", CASES)
def test_forward_backward(pkg, t, d, g, post, pre, dtype):
    ops = pkg.ops
    b, x = rnd((t, d), 1, dtype, 2.0), rnd((t, d), 2, dtype)
    gp = rnd((d,), 3, dtype, 0.3) + 1 if post else None
    gate = rnd((g, d), 4, dtype) if g else None
    gn = rnd((d,), 5, dtype, 0.3) + 1 if pre else None
    al, s, eps = 0.9, -1.3, 1e-5
    y, n, ib, iy = ops.sandwich_norm(b, x, gp, gate, gn, residual_scale=al, branch_scale=s, eps=eps)
    ry, rib, mag = forward64(b, x, gp, gate, gn, al, s, eps)
    close(ib, rib, rib)
    close(y, ry, mag, dtype)
    if pre:
        # y is off by at most F32 * mag before its rounding; its root mean square by that of the same
        riy = (ry.square().mean(1) + eps).rsqrt()
        off = riy * (mag.square().mean(1) + eps).sqrt()
        close(iy, riy, riy * (1 + off))
        close(n, ry * riy[:, None] * gn.double(), (mag * (1 + off[:, None])) * riy[:, None] * gn.double().abs(), dtype)
    else:
        assert n is None and iy is None
    dy, dn = rnd((t, d), 6, dtype, 0.1), (rnd((t, d), 7, dtype, 0.1) if pre else None)
    kw = dict(dn=dn, y=y, inv_y=iy, gamma_pre=gn) if pre else {}
    got = ops.sandwich_norm_bwd(dy, b, ib, gp, gate, residual_scale=al, branch_scale=s, **kw)
    ref, big = backward64(dy, dn, b, y, ib, iy, gp, gate, gn, al, s)
    for k in ("dx", "db"):
        close(got[k], ref[k], big[k], dtype)
    for k in ("dgamma_post", "dgate", "dgamma_pre"):
        if ref[k] is None or (k == "dgamma_pre" and not pre):
            assert got[k] is None
        else:
            close(got[k], ref[k], big[k], extra=F32 + (t + 64) * 2.0 ** -24)
    again = ops.sandwich_norm_bwd(dy, b, ib, gp, gate, residual_scale=al, branch_scale=s, **kw)
    assert all((got[k] is None) == (again[k] is None) and (got[k] is None or torch.equal(got[k], again[k])) for k in got)
    if pre:   # only the next norm's gradient
        only = ops.sandwich_norm_bwd(None, b, ib, gp, gate, residual_scale=al, branch_scale=s, **kw)
        zero = ops.sandwich_norm_bwd(torch.zeros_like(b), b, ib, gp, gate, residual_scale=al, branch_scale=s, **kw)
        assert all(only[k] is None or torch.equal(only[k], zero[k]) for k in only)


def test_strides_and_misaligned(pkg):
    """Row-strided inputs, inputs that start off a 16-byte boundary, transposed ones: the same bits."""
    ops = pkg.ops
    t, d = 37, 264
    big = rnd((t, 3 * d), 1, BF)
    odd = rnd((t, 3 * d + 1), 6, BF)
    for b, x in ((odd[:, :d], odd[:, 2 * d:3 * d]), (big[:, :d], big[:, 2 * d:]), (big[:, 1:d + 1], big[:, d + 3:2 * d + 3]),
                 (rnd((d, t), 2, BF).t(), big[:, :d]), (big[:1, :d].expand(t, d), big[:, d:2 * d])):
        gp, gate, gn = rnd((d,), 3, BF), rnd((1, d), 4, BF), rnd((d,), 5, BF)
        got = ops.sandwich_norm(b, x, gp, gate, gn)
        bc, xc = b.contiguous(), x.contiguous()
        y, n, ib, iy = ops.sandwich_norm(bc, xc, gp, gate, gn)
        ry, rib, mag = forward64(b, x, gp, gate, gn, 1.0, 1.0, 1e-6)
        close(got[0], ry, mag, BF)
        close(got[2], rib, rib)
        dy, dn = big[:, 5:d + 5], big[:, d + 8:2 * d + 8]
        g = ops.sandwich_norm_bwd(dy, b, ib, gp, gate, dn=dn, y=y, inv_y=iy, gamma_pre=gn)
        ref, mg = backward64(dy, dn, b, y, ib, iy, gp, gate, gn, 1.0, 1.0)
        for k in ("dx", "db"):
            close(g[k], ref[k], mg[k], BF)
        for k in ("dgamma_post", "dgate", "dgamma_pre"):
            close(g[k], ref[k], mg[k], extra=F32 + (t + 64) * 2.0 ** -24)


@pytest.mark.parametrize("dtype", [BF, HF, FL])
@pytest.mark.parametrize("t,d", [(1, 3), (2, 7), (9, 1), (500, 5), (300, 67), (1000, 1001), (401, 4097), (97, 8191), (700, 2050),
                                 (500, 9001), (311, 16383), (2, 8193), (450, 1501), (301, 5003), (290, 6001)])
def test_widths_of_no_multiple(pkg, t, d, dtype):
    """Unaligned rows, many of them, the tensors ending with their storage: forward and
    backward against float64, and nothing read beside them (neighbours are NaN)."""
    ops = pkg.ops

    def lone(seed, std=1.0):   # a [t, d] view that starts 16-byte aligned, NaN before and after
        flat = torch.full((t * d + 32,), math.nan, device="cuda", dtype=dtype)
        flat[16:16 + t * d] = rnd((t * d,), seed, dtype, std)
        return flat[16:16 + t * d].view(t, d)

    b, x, dy, dn = lone(1, 2.0), lone(2), lone(3, 0.1), lone(4, 0.1)
    gp, gate, gn = rnd((d,), 5, dtype, 0.3) + 1, rnd((1, d), 6, dtype), rnd((d,), 7, dtype, 0.3) + 1
    y, n, ib, iy = ops.sandwich_norm(b, x, gp, gate, gn, branch_scale=0.7)
    ry, rib, mag = forward64(b, x, gp, gate, gn, 1.0, 0.7, 1e-6)
    close(ib, rib, rib)
    close(y, ry, mag, dtype)
    riy = (ry.square().mean(1) + 1e-6).rsqrt()
    off = riy * (mag.square().mean(1) + 1e-6).sqrt()
    close(n, ry * riy[:, None] * gn.double(), (mag * (1 + off[:, None])) * riy[:, None] * gn.double().abs(), dtype)
    for kw in (dict(dn=dn, y=y, inv_y=iy, gamma_pre=gn), {}):
        got = ops.sandwich_norm_bwd(dy, b, ib, gp, gate, branch_scale=0.7, **kw)
        ref, big = backward64(dy, kw.get("dn"), b, y, ib, iy, gp, gate, gn, 1.0, 0.7)
        for k in ("dx", "db"):
            close(got[k], ref[k], big[k], dtype)
        for k in ("dgamma_post", "dgate", "dgamma_pre"):
            if got[k] is not None:
                close(got[k], ref[k], big[k], extra=F32 + (t + 64) * 2.0 ** -24)
    assert ops.device_error() == 0


@pytest.mark.parametrize("dtype", [BF, FL])
@pytest.mark.parametrize("per,d", [(1, 4096), (1, 1001), (3, 1001), (2, 96), (7, 520), (1, 7), (5, 4104), (1, 8191), (40, 2048), (1, 12288), (3, 16384), (2, 9001)])
def test_many_gates(pkg, per, d, dtype):
    """More groups of rows than CTAs: a CTA walks several groups, and the last one fewer."""
    ops = pkg.ops
    groups = (5000 if d < 100 else 1900 if d < 1100 else 701 if d < 8192 else 233) // (1 if per < 8 else 4)
    t = groups * per
    b, y, dy, dn = (rnd((t, d), i, dtype, s) for i, s in ((1, 2.0), (2, 1.0), (3, 0.1), (4, 0.1)))
    gp, gate, gn = rnd((d,), 5, dtype, 0.3) + 1, rnd((groups, d), 6, dtype), rnd((d,), 7, dtype, 0.3) + 1
    ib, iy = rnd((t,), 8).abs() + 0.1, rnd((t,), 9).abs() + 0.1
    for kw in (dict(dn=dn, y=y, inv_y=iy, gamma_pre=gn), {}):
        for w in (gp, None):
            got = ops.sandwich_norm_bwd(dy, b, ib, w, gate, residual_scale=0.5, branch_scale=-0.7, **kw)
            ref, big = backward64(dy, kw.get("dn"), b, y, ib, iy, w, gate, gn, 0.5, -0.7)
            for k in ("dx", "db"):
                close(got[k], ref[k], big[k], dtype)
            for k in ("dgamma_post", "dgate", "dgamma_pre"):
                if got[k] is not None:
                    close(got[k], ref[k], big[k], extra=F32 + (t + 64) * 2.0 ** -24)
            again = ops.sandwich_norm_bwd(dy, b, ib, w, gate, residual_scale=0.5, branch_scale=-0.7, **kw)
            assert all(got[k] is None or torch.equal(got[k], again[k]) for k in got)
    assert ops.device_error() == 0


def test_zero_rows_and_no_rows(pkg):
    ops = pkg.ops
    b = torch.zeros(3, 64, device="cuda", dtype=BF)
    x = rnd((3, 64), 1, BF)
    y, n, ib, iy = ops.sandwich_norm(b, x, pre=True)
    assert torch.equal(y, x) and torch.allclose(ib, torch.full_like(ib, 1e3), rtol=1e-6)
    g = ops.sandwich_norm_bwd(x, b, ib)
    assert torch.equal(g["dx"], x) and torch.isfinite(g["db"]).all() and (g["dgamma_post"] == 0).all()
    e = b[:0]
    gate = rnd((1, 64), 2, BF)
    y, n, ib, iy = ops.sandwich_norm(e, e, gate=gate, pre=True)
    assert y.shape == n.shape == (0, 64) and ib.shape == iy.shape == (0,)
    g = ops.sandwich_norm_bwd(e, e, ib, gate=gate, dn=e, y=e, inv_y=iy)
    assert (g["dgate"] == 0).all() and (g["dgamma_pre"] == 0).all() and g["db"].shape == (0, 64)


def test_non_finite_rows_stay_apart(pkg):
    """A row with a NaN or an infinity touches no other row."""
    b, x = rnd((40, 512), 1, BF), rnd((40, 512), 2, BF)
    ref = pkg.ops.sandwich_norm(b, x, pre=True)
    b2 = b.clone()
    b2[3, 100], b2[17, 0] = math.nan, math.inf
    got = pkg.ops.sandwich_norm(b2, x, pre=True)
    ok = torch.ones(40, dtype=torch.bool, device="cuda")
    ok[[3, 17]] = False
    for a, r in zip(got, ref):
        assert torch.equal(a[ok], r[ok])
    assert torch.isnan(got[0][3]).all()


@pytest.mark.parametrize("shape,gshape", [((6, 128), (128,)), ((2, 5, 96), (2, 96)), ((2, 3, 64), (2, 1, 64)), ((4, 72), None)])
def test_autograd_against_differences(pkg, shape, gshape):
    """Directional differences of a scalar loss in float64 against the kernel's fp32 gradients."""
    import importlib
    mlp = importlib.import_module("nvfp4_b200.mlp")
    d = shape[-1]
    leaves = [rnd(shape, 1), rnd(shape, 2), rnd((d,), 3, FL, 0.3) + 1, rnd(gshape, 4) if gshape else None, rnd((d,), 5, FL, 0.3) + 1]
    cy, cn = rnd(shape, 8).double(), rnd(shape, 9).double()
    al, s, eps = 0.8, 0.7, 1e-5

    def loss64(b, x, gp, gate, gn):
        t = b.numel() // d
        y, _, _ = forward64(b.reshape(t, d), x.reshape(t, d), gp, None if gate is None else gate.reshape(-1, d), gn, al, s, eps)
        n = y * (y.square().mean(1, keepdim=True) + eps).rsqrt() * gn.double()
        return (y * cy.reshape(t, d)).sum() + (n * cn.reshape(t, d)).sum()

    for p in leaves:
        if p is not None:
            p.requires_grad_()
    y, n = mlp.sandwich_norm(leaves[0], leaves[1], leaves[2], leaves[3], leaves[4], residual_scale=al, branch_scale=s, eps=eps)
    ((y * cy.float()).sum() + (n * cn.float()).sum()).backward()
    h = 1e-5
    with torch.no_grad():
        for i, p in enumerate(leaves):
            if p is None:
                continue
            assert p.grad.shape == p.shape and p.grad.dtype == p.dtype
            u = rnd(tuple(p.shape), 50 + i).double()
            at = lambda e: [None if q is None else (q.double() + e * u if q is p else q.double()) for q in leaves]
            diff = (loss64(*at(h)) - loss64(*at(-h))) / (2 * h)
            dot = (p.grad.double() * u).sum()
            assert abs(diff - dot) <= 1e-4 * (p.grad.double().abs() * u.abs()).sum()


def test_autograd_partial_use(pkg):
    """Only y, only n, no gradient for the parameters; results changed in place."""
    import importlib
    mlp = importlib.import_module("nvfp4_b200.mlp")
    b, x = rnd((2, 4, 64), 1, BF), rnd((2, 4, 64), 2, BF)
    gp = (rnd((64,), 3, BF) + 1)
    bb = b.clone().requires_grad_()
    y = mlp.sandwich_norm(bb, x, gp)
    y.mul_(2)
    y.sum().backward()
    assert bb.grad.shape == b.shape
    bb.grad = None
    _, n = mlp.sandwich_norm(bb, x, gp, pre=True)
    n.float().square().sum().backward()
    assert torch.isfinite(bb.grad).all()


def test_mlp_block_with_post_norm(pkg):
    """NVFP4SwiGLUMLP(post_norm=True): the forward is the plain block's output through
    the norm; gradients reach every parameter; without the option nothing changes."""
    import importlib
    mlp = importlib.import_module("nvfp4_b200.mlp")
    torch.manual_seed(0)
    plain = mlp.NVFP4SwiGLUMLP(256, 512, device="cuda")
    blk = mlp.NVFP4SwiGLUMLP(256, 512, device="cuda", post_norm=True, gate=True, residual_scale=0.9, branch_scale=0.5)
    blk.load_state_dict(plain.state_dict(), strict=False)
    x = rnd((2, 64, 256), 1, BF).requires_grad_()
    qw = mlp.quantize_weights(plain.w_gu.detach(), plain.w_down.detach())
    zero = torch.zeros(128, 256, device="cuda", dtype=BF)
    with torch.no_grad():
        blk.gate.copy_(rnd((256,), 2, BF))
        _, sv = mlp.block_forward(x.detach().view(128, 256), blk.gamma.detach(), qw,
                                  post=mlp.PostNorm(blk.post_gamma, blk.gate, 0.9, 0.5))
        want = pkg.ops.sandwich_norm(sv.b, x.detach().view(128, 256), blk.post_gamma, blk.gate, residual_scale=0.9,
                                     branch_scale=0.5)[0]
    y = blk(x)
    assert torch.equal(y.view(128, 256), want)
    dy = rnd((2, 64, 256), 3, BF, 1e-2)
    y.backward(dy)
    ref = pkg.ops.sandwich_norm_bwd(dy.view(128, 256), sv.b, sv.inv_b, blk.post_gamma.detach(), blk.gate.detach(),
                                    residual_scale=0.9, branch_scale=0.5)
    assert torch.equal(blk.gate.grad, ref["dgate"][0].to(BF)) and torch.equal(blk.post_gamma.grad, ref["dgamma_post"].to(BF))
    for p in blk.parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all() and p.grad.abs().sum() > 0
    # the block's part of dx is what the plain backward gives for db
    dx0 = mlp.block_backward(ref["db"], blk.gamma.detach(), qw, mlp.Saved(*[getattr(sv, k) for k in ("x", "inv_rms", "g_xn", "gu", "h", "g_h")]),
                             torch.zeros(256, device="cuda"), torch.empty_like(plain.w_gu), torch.empty_like(plain.w_down), False)
    branch = dx0.double() - ref["db"].double()
    total = branch + ref["dx"].double()
    # two roundings to bf16 apart (dx0, and the result itself), each half a step
    assert ((x.grad.view(128, 256).double() - total).abs()
            <= half_step(dx0.double(), BF) + half_step(total, BF) + half_step(half_step(dx0.double(), BF), BF) + 1e-12).all()


def test_refusals(pkg):
    ops = pkg.ops
    b = rnd((6, 64), 1, BF)
    inv = torch.ones(6, device="cuda")
    for call in (lambda: ops.sandwich_norm(b, b.float()), lambda: ops.sandwich_norm(b, b[:5]), lambda: ops.sandwich_norm(b[0], b[0]),
                 lambda: ops.sandwich_norm(b, b, gamma_post=b[0, :32]), lambda: ops.sandwich_norm(b, b, gate=rnd((4, 64), 2, BF)),
                 lambda: ops.sandwich_norm(b, b, gate=rnd((1, 64), 2)), lambda: ops.sandwich_norm(b, b, gamma_pre=b[0], pre=False),
                 lambda: ops.sandwich_norm(rnd((2, 16385), 1), rnd((2, 16385), 1)), lambda: ops.sandwich_norm(b.double(), b.double()),
                 lambda: ops.sandwich_norm_bwd(None, b, inv), lambda: ops.sandwich_norm_bwd(b, b, inv, dn=b),
                 lambda: ops.sandwich_norm_bwd(b, b, inv[:5]), lambda: ops.sandwich_norm_bwd(b, b, inv, gamma_pre=b[0]),
                 lambda: ops.sandwich_norm_bwd(b.float(), b, inv)):
        with pytest.raises(RuntimeError):
            call()


def test_graph_with_backward(pkg):
    """Forward and backward captured and replayed with new inputs, beside an eager call on another stream."""
    ops = pkg.ops
    t, d = 48, 1024
    b, x, dy, dn = (rnd((t, d), i, BF) for i in range(4))
    gp, gate, gn = rnd((d,), 5, BF), rnd((4, d), 6, BF), rnd((d,), 7, BF)

    def both(b, x, dy, dn):
        y, n, ib, iy = ops.sandwich_norm(b, x, gp, gate, gn)
        g = ops.sandwich_norm_bwd(dy, b, ib, gp, gate, dn=dn, y=y, inv_y=iy, gamma_pre=gn)
        return [y, n, ib, iy] + [g[k] for k in sorted(g)]
    both(b, x, dy, dn)
    bufs = [v.clone() for v in (b, x, dy, dn)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both(*bufs)
    for seed in (20, 30):
        new = [rnd((t, d), seed + i, BF) for i in range(4)]
        for buf, v in zip(bufs, new):
            buf.copy_(v)
        graph.replay()
        assert all(torch.equal(a, r) for a, r in zip(out, both(*new)))
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        other = both(b, x, dy, dn)
    torch.cuda.current_stream().wait_stream(st)
    assert all(torch.equal(a, r) for a, r in zip(other, both(b, x, dy, dn)))


def test_layer_step_together(pkg, f4):
    """The operators as a training step uses them: MXFP4 linear layers around the
    two norms, loss, backward, clipping and AdamW; one step equals the same step
    made of its parts in float64 within the products' tolerances."""
    import importlib
    mlp = importlib.import_module("nvfp4_b200.mlp")
    torch.manual_seed(1)
    d, t = 256, 70
    up, down = f4.MXFP4Linear(d, 2 * d, bias=False, device="cuda"), f4.MXFP4Linear(2 * d, d, bias=False, device="cuda")
    head = f4.MXFP4Linear(d, 64, bias=True, device="cuda")
    gp, gate, gn = (torch.nn.Parameter(rnd((d,), 10 + i, BF, 0.1) + 1) for i in range(3))
    params = [up.weight, down.weight, head.weight, head.bias, gp, gate, gn]
    x, dz = rnd((t, d), 1, BF), rnd((t, 64), 2, BF, 0.5)
    b = down(torch.relu(up(x)))
    y, n = mlp.sandwich_norm(b, x, gp, gate, gn, branch_scale=0.5)
    (head(n).float() * dz.float()).sum().add(y.float().square().mean()).backward()
    grads = [p.grad for p in params]
    norm = pkg.ops.clip_grad_norm(grads, 0.5)
    ref = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
    assert norm.item() > 0.5 and abs(ref - 0.5) <= 0.5 * 2.0 ** -8       # clipped to 0.5, each value rounded to bf16
    before = [p.detach().clone() for p in params]
    for p, g in zip(params, grads):
        m, v = torch.zeros(p.numel(), device="cuda"), torch.zeros(p.numel(), device="cuda")
        pkg.ops.adamw_step(p.data.view(-1), g.view(-1), m, v, lr=1e-2, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.0, step=1)
    assert all(not torch.equal(p, q) and torch.isfinite(p).all() for p, q in zip(params, before))
    assert pkg.ops.device_error() == 0


def test_offsets_past_32_bits(pkg):
    """More than 2^31 elements, forward and backward: the last rows against the same
    rows alone."""
    ops = pkg.ops
    t, d = 133000, 16384
    b = torch.empty(t, d, device="cuda", dtype=BF)
    for lo in range(0, t, 13300):
        b[lo:lo + 13300] = rnd((13300, d), lo, BF)
    x, gp, gn = b.flip(0), rnd((d,), 1, BF), rnd((d,), 2, BF)
    gate = rnd((2, d), 3, BF)
    y, n, ib, iy = ops.sandwich_norm(b, x, gp, gate, gn)
    last = slice(t - 40, t)
    y2, n2, ib2, iy2 = ops.sandwich_norm(b[last], x[last], gp, gate[1:], gn)
    for a, r in ((y, y2), (n, n2), (ib, ib2), (iy, iy2)):
        assert torch.equal(a[last], r)
    del n
    g = ops.sandwich_norm_bwd(x, b, ib, gp, gate, dn=b, y=y, inv_y=iy, gamma_pre=gn)
    g2 = ops.sandwich_norm_bwd(x[last], b[last], ib2, gp, gate[1:], dn=b[last], y=y2, inv_y=iy2, gamma_pre=gn)
    for k in ("dx", "db"):
        assert torch.equal(g[k][last], g2[k])
    assert all(torch.isfinite(g[k]).all() for k in ("dgamma_post", "dgate", "dgamma_pre"))
