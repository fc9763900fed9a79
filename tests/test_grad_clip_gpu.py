"""GPU parity of the global gradient norm, clipping and the clipped AdamW steps.

Squares are summed in fp32 over 8 elements (relative error at most 8 * 2^-24 =
2^-21, of positive terms) and in fp64 after that, the norm is rounded to fp32
once: relative error at most 2^-22 + 2^-24 < 2^-21.  A clipped value is two
fp32 roundings (factor, product) away from g * coef, plus the rounding to its
type: half a step, eps/2 relative, or half the smallest subnormal."""
import math

import numpy as np
import pytest
import torch

from oracle import adamw_oracle

pytestmark = pytest.mark.gpu
REL = 2.0 ** -21


def tensors(sizes, dtypes, seed=0, std=1e-2):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(s, device="cuda", generator=g) * std).to(dtypes[i % len(dtypes)]) for i, s in enumerate(sizes)]


def ref_norm(grads, kind=2):
    parts = [g.double().abs() for g in grads if g.numel()]
    if not parts:
        return 0.0
    if kind == 2:
        return math.sqrt(sum(float(p.square().sum()) for p in parts))
    return max(float(p.max()) for p in parts)


def check_scaled(out, grads, factor):
    for o, g in zip(out, grads):
        ref = g.double() * factor
        f = torch.finfo(o.dtype)
        tol = ref.abs() * (f.eps / 2 + 2.0 ** -20) + f.smallest_normal * f.eps / 2
        assert ((o.double() - ref).abs() <= tol).all()


BF, HF, FL = torch.bfloat16, torch.float16, torch.float32
LISTS = [([7], [BF]), ([1], [FL]), ([(3, 5), (), 8], [HF, FL, BF]), ([4096, 0, 4097, 12289], [BF, FL]),
         ([(257, 515), (515,), (1030, 257)] * 4, [FL, BF, HF]), ([33] * 300, [BF, FL, HF]),
         ([(4096, 2304), (1000, 2311)], [BF]), ([20_000_003, 5], [FL, BF])]


@pytest.mark.parametrize("sizes,dtypes", LISTS)
@pytest.mark.parametrize("kind", [2, math.inf])
def test_norm(pkg, sizes, dtypes, kind):
    grads = tensors(sizes, dtypes)
    n = pkg.ops.grad_norm(grads, norm_type=kind)
    ref = ref_norm(grads, kind)
    assert n.shape == (1,) and n.dtype == torch.float32
    assert abs(n.item() - ref) <= REL * ref
    assert abs(pkg.ops.grad_norm(grads, kind, grad_scale=-0.25).item() - 0.25 * ref) <= REL * ref
    assert torch.equal(n, pkg.ops.grad_norm(grads, norm_type=kind))


@pytest.mark.parametrize("sizes,dtypes", LISTS)
@pytest.mark.parametrize("max_norm", [0.05, 1e6])
def test_clip_in_place_and_out(pkg, sizes, dtypes, max_norm):
    grads = tensors(sizes, dtypes, 1)
    norm = ref_norm(grads)
    coef = min(1.0, max_norm / (norm + 1e-6))
    out = [torch.full_like(g, 5, dtype=d) for g, d in zip(grads, [BF, FL, HF] * 200)]
    n = pkg.ops.clip_grad_norm(grads, max_norm, out=out)
    assert abs(n.item() - norm) <= REL * norm
    check_scaled(out, grads, coef)
    scaled = [torch.empty_like(g) for g in grads]
    pkg.ops.clip_grad_norm(grads, max_norm, grad_scale=0.5, out=scaled)
    check_scaled(scaled, grads, 0.5 * min(1.0, max_norm / (0.5 * norm + 1e-6)))
    keep = [g.clone() for g in grads]
    assert torch.equal(pkg.ops.clip_grad_norm(grads, max_norm), n)
    if coef < 1:
        check_scaled(grads, keep, coef)
    else:
        assert all(torch.equal(a, b) for a, b in zip(grads, keep))


def test_offsets_past_32_bits(pkg):
    """One gradient of more than 2^31 elements, misaligned and not."""
    big = torch.full((2 ** 31 + 4099,), 0.5, device="cuda", dtype=BF)
    for g in (big, big[1:]):
        ref = 0.5 * math.sqrt(g.numel())
        n = pkg.ops.clip_grad_norm(g, ref / 4, out=[g.new_empty(g.shape)])
        assert abs(n.item() - ref) <= REL * ref
    big[-1] = 2000.0
    n = pkg.ops.clip_grad_norm(big, 1e9, math.inf)
    assert n.item() == 2000.0
    pkg.ops.clip_grad_norm(big, 1000.0, math.inf)          # halves every value exactly, to within the 1e-6
    assert big[-1].item() == 1000.0 and big[0].item() == 0.25 and big[2 ** 31 + 7].item() == 0.25


def test_misaligned_views_and_layouts(pkg):
    """Views at odd offsets of one buffer, transposed and permuted gradients."""
    flat = tensors([10_007], [BF])[0]
    grads = [flat[1:4000], flat[4001:4009], flat[4100:4100 + 64 * 65].view(64, 65).t()]
    big = tensors([(6, 4, 10)], [FL], 2)[0].permute(2, 0, 1)
    grads.append(big)
    keep = [g.clone() for g in grads]
    rest = flat.clone()
    norm = ref_norm(grads)
    bucket = torch.zeros(4999, device="cuda", dtype=FL)
    out = [bucket[1:4000], bucket[4001:4009], torch.empty_like(grads[2]), torch.empty_like(big)]
    n = pkg.ops.clip_grad_norm(grads, 0.1, out=out)
    assert abs(n.item() - norm) <= REL * norm
    check_scaled(out, keep, 0.1 / (norm + 1e-6))
    assert bucket[0] == 0 and bucket[4000] == 0 and (bucket[4009:] == 0).all()
    pkg.ops.clip_grad_norm(grads, 0.1)
    check_scaled(grads, keep, 0.1 / (norm + 1e-6))
    inside = torch.zeros(10_007, dtype=torch.bool, device="cuda")
    inside[1:4000] = inside[4001:4009] = inside[4100:4100 + 64 * 65] = True
    assert torch.equal(flat[~inside], rest[~inside])


@pytest.mark.parametrize("src", [BF, HF, FL])
@pytest.mark.parametrize("dst", [BF, HF, FL])
def test_every_alignment(pkg, src, dst):
    """Views at every offset within 16 bytes on either side, short and past a chunk's
    length: each value right, nothing written beside them."""
    for n in (1, 6, 7, 8, 9, 23, 300, 12345):
        a, b = tensors([n + 9], [src], n)[0], torch.full((n + 18,), 7.0, device="cuda", dtype=dst)
        for i in range(0, 9, 1 if n < 400 else 3):
            for j in range(9):
                b.fill_(7.0)
                g, o = a[i:i + n], b[j + 1:j + 1 + n]
                norm = pkg.ops.clip_grad_norm([g], 0.01, out=[o])
                ref = ref_norm([g])
                assert abs(norm.item() - ref) <= REL * ref
                check_scaled([o], [g], min(1.0, 0.01 / (ref + 1e-6)))
                assert (b[:j + 1] == 7).all() and (b[j + 1 + n:] == 7).all()


@pytest.mark.parametrize("scale", [1e-38, 1e-30, 1e-22, 1e18, 1e30, 3e38])
def test_extreme_magnitudes(pkg, scale):
    """Squares that fp32 cannot hold, alone and beside ordinary ones."""
    g = torch.tensor([1.0, -0.5, 0.25] * 1000, device="cuda") * scale
    for grads in ([g], [g, tensors([100], [FL])[0]], [g.to(BF)]):
        ref = ref_norm(grads)
        got = pkg.ops.grad_norm(grads).item()
        if ref > 3.4028235e38:
            assert got == math.inf
            n, c = pkg.ops.grad_norm_coef(grads, 1e38)
            assert abs(c.item() - 1e38 / ref) <= 2.0 ** -20 * 1e38 / ref   # the factor comes from the fp64 norm
        else:
            # fp32 rounding of the norm, or of a subnormal one
            assert abs(got - ref) <= REL * ref + 2.0 ** -150


def test_non_finite(pkg):
    g = tensors([5000, 300], [BF, FL], 4)
    g[1][7] = math.inf
    out = [torch.empty_like(t) for t in g]
    assert pkg.ops.clip_grad_norm(g, 1.0, out=out).item() == math.inf
    assert (out[0] == 0).all() and torch.isnan(out[1][7]) and torch.isnan(out[1]).sum() == 1
    g[0][4999] = math.nan
    for kind in (2, math.inf):
        assert math.isnan(pkg.ops.clip_grad_norm(g, 1.0, kind, out=out).item())
        assert all(torch.isnan(o).all() for o in out)


def test_degenerate_lists(pkg):
    ops = pkg.ops
    assert ops.grad_norm([]).item() == 0 and ops.clip_grad_norm([], 1.0).item() == 0
    e = torch.empty(0, 4, device="cuda")
    assert ops.clip_grad_norm([e], 1.0).item() == 0
    z = torch.zeros(1000, device="cuda", dtype=BF)
    n, c = ops.grad_norm_coef([z], 1.0)
    assert n.item() == 0 and c.item() == 1
    one = tensors([100], [FL])[0]
    assert ops.grad_norm(one).item() == ops.grad_norm([one]).item()
    twice = ops.grad_norm([one, one]).item()       # a list counts what it holds
    assert abs(twice - math.sqrt(2) * ref_norm([one])) <= 2 * REL * twice
    zero = one.clone()
    ops.clip_grad_norm([zero], 0.0)
    assert (zero == 0).all()


def test_refusals(pkg):
    ops = pkg.ops
    a, b = tensors([64, 64], [BF])
    w = tensors([(8, 8)], [FL])[0]
    for call in (lambda: ops.grad_norm([a.double()]), lambda: ops.grad_norm([w[:, ::2]]), lambda: ops.grad_norm([a], 1),
                 lambda: ops.clip_grad_norm([a], -1.0), lambda: ops.clip_grad_norm([a], math.nan),
                 lambda: ops.clip_grad_norm([a, a], 1.0), lambda: ops.clip_grad_norm([a, b], 1.0, out=[a]),
                 lambda: ops.clip_grad_norm([a, b], 1.0, out=[b, a]), lambda: ops.clip_grad_norm([a[:40], a[32:]], 1.0),
                 lambda: ops.clip_grad_norm([w], 1.0, out=[torch.empty(8, 8, device="cuda").t()]),
                 lambda: ops.clip_grad_norm([a, a.cpu()], 1.0), lambda: ops.grad_norm([a.to(torch.int16)]),
                 lambda: ops.grad_norm_finish(torch.ones(1, device="cuda"), 1.0)):
        keep = a.clone()
        with pytest.raises(RuntimeError):
            call()
        assert torch.equal(a, keep)


def test_shard_totals(pkg):
    """Totals of the shards, summed (or their maximum), give the whole list's norm and factor."""
    grads = tensors([5000, 777, 12345], [BF, FL])
    for kind in (2, math.inf):
        totals = torch.cat([pkg.ops.grad_norm_total([g], kind) for g in grads])
        n, c = pkg.ops.grad_norm_finish(totals, 0.3, kind, grad_scale=0.5)
        whole, coef = pkg.ops.grad_norm_coef(grads, 0.3, kind, grad_scale=0.5)
        assert abs(n.item() - whole.item()) <= 2 * REL * whole.item() and abs(c.item() - coef.item()) <= 2.0 ** -20


def test_streams_and_two_graphs(pkg):
    """Two captured graphs replayed at once on two streams share nothing."""
    ops = pkg.ops
    sets = [tensors([100_003, 50_000], [BF, FL], s) for s in (1, 2)]
    outs = [[torch.empty_like(t) for t in s] for s in sets]
    graphs, norms = [], []
    for s, o in zip(sets, outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            norms.append(ops.clip_grad_norm(s, 0.5, out=o))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(20):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for s, o, n in zip(sets, outs, norms):
        ref = ref_norm(s)
        assert abs(n.item() - ref) <= REL * ref
        check_scaled(o, s, min(1.0, 0.5 / (ref + 1e-6)))


HP = dict(lr=3e-3, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.1)


@pytest.mark.parametrize("n", [5, 1001])
@pytest.mark.parametrize("coef", [1.0, 0.25, 0.3])
def test_adamw_takes_the_factor(pkg, n, coef):
    """clip is one more factor: the same bits as that grad_scale in fp32."""
    g = tensors([n], [BF], 3, 0.1)[0]
    w = torch.randn(n, device="cuda")
    c = torch.tensor([coef], device="cuda")
    both = float(np.float32(0.5) * np.float32(coef))
    for master in (True, False):
        got = []
        for kw in (dict(grad_scale=0.5, clip=c), dict(grad_scale=both)):
            p, ww, m, v = w.to(BF), w.clone(), torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
            for step in (1, 2):
                if master:
                    pkg.ops.adamw_master_step(p, ww, g, m, v, step=step, **HP, **kw)
                else:
                    pkg.ops.adamw_step(p, g, m, v, step=step, **HP, **kw)
            got.append((p, ww, m, v))
        assert all(torch.equal(a, b) for a, b in zip(*got))
    # and against the float32 oracle
    op, om, ov = p.cpu(), None, None
    start = w.to(BF).cpu().view(torch.int16).numpy().view(np.uint16)
    z = np.zeros(n, np.float32)
    bits = lambda t: t.cpu().view(torch.int16).numpy().view(np.uint16)
    o1 = adamw_oracle.adamw_bf16(start, bits(g), z, z, step=1, grad_scale=both, **HP)
    o2 = adamw_oracle.adamw_bf16(o1[0], bits(g), o1[1], o1[2], step=2, grad_scale=both, **HP)
    assert np.array_equal(bits(got[0][0]), o2[0])


@pytest.mark.parametrize("micro", [512, 256])
def test_trainer_clips(pkg, micro):
    """max_grad_norm in the trainer: the norm it reports is that of its gradients,
    and the moments after one step are those of the scaled gradients."""
    import importlib
    mlp = importlib.import_module("nvfp4_b200.mlp")
    t, d, f = 512, 256, 512
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(t, d, device="cuda", generator=g).to(BF)
    dy = (torch.randn(t, d, device="cuda", generator=g) * 1e-2).to(BF)
    free = mlp.NVFP4MLPStackTrainer(2, d, f, micro_tokens=micro, max_local_tokens=t)
    free.step(x, dy)
    grads = [g for b in free.blocks for g in ((b.grad,) if micro == t else (b.grad_gamma32, b.acc_gu, b.acc_down))]
    norm = ref_norm(grads)
    assert free.grad_norm is None
    for max_norm in (norm / 3, norm * 3):
        tr = mlp.NVFP4MLPStackTrainer(2, d, f, micro_tokens=micro, max_local_tokens=t,
                                      adam=mlp.AdamConfig(max_grad_norm=max_norm))
        tr.step(x, dy)
        # gamma's gradient is summed by atomics, whose order may change its last bits between the runs
        assert abs(tr.grad_norm.item() - norm) <= 1e-4 * norm
        coef = min(1.0, max_norm / norm)
        for a, b in zip(tr.blocks, free.blocks):
            lo = d   # past gamma
            assert (a.m[lo:] - coef * b.m[lo:]).abs().max() <= 2e-4 * coef * b.m[lo:].abs().max()


def test_writes_are_counted(pkg):
    """A tensor that autograd saved and clipping then wrote: its backward is
    refused, as after any change in place.  Tensors of inference mode count nothing."""
    for out in (False, True):
        p = torch.randn(100, device="cuda", requires_grad=True)
        t = torch.randn(100, device="cuda")
        loss = (p * t).sum()
        pkg.ops.clip_grad_norm([torch.randn(100, device="cuda")] if out else [t], 0.5, out=[t] if out else None)
        with pytest.raises(RuntimeError, match="inplace"):
            loss.backward()
    with torch.inference_mode():
        t = torch.randn(100, device="cuda")
        ref = t.double().norm().item()
        assert abs(pkg.ops.clip_grad_norm([t], 0.5).item() - ref) <= REL * ref
    assert t.norm().item() < 0.51


def test_two_threads(pkg):
    """Calls from several host threads, each on its stream, as from one."""
    import threading
    lists = [tensors([(257, 515), 33, 100_003 * (i + 1)], [FL, BF, HF], seed=i) for i in range(4)]
    ref = [pkg.ops.grad_norm(g) for g in lists]
    torch.cuda.synchronize()
    got = [[] for _ in lists]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                got[i].append(pkg.ops.grad_norm(lists[i]))
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(len(g) == 50 and all(torch.equal(v, r) for v in g) for g, r in zip(got, ref))
