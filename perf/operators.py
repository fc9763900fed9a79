"""What the training and serving operators beside the NVFP4 path are measured on.

Six calls: an MXFP4 linear layer with held weights (``mx_linear``), the same
layer trained (``mx_train``: forward, dgrad and wgrad with MXFP4 operands),
the MXFP4 quantizer in both orientations (``mx_quant``), the global gradient
norm with clipping into communication buckets (``clip``), and the norms after
and before a block fused with its gate and residual scale (``norm_fwd``,
``norm_bwd``).

``run`` computes each with elementary torch operations in 32 bits (64 where
32 lose what matters), or, where ``own`` is true, with the package's entry
points.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-6


def listed():
    return [
        # one token through a down projection of the 4096 x 14336 MLP: serving, the weight stream and latency count
        {"name": "linear_token", "op": "mx_linear", "m": 1, "n": 4096, "k": 14336, "bias": False},
        # a ragged decode batch through its gate/up projection
        {"name": "linear_batch", "op": "mx_linear", "m": 37, "n": 28672, "k": 4096, "bias": True},
        # a whole micro-batch of tokens through the up projection: tensor-core rate
        {"name": "linear_prefill", "op": "mx_linear", "m": 16384, "n": 14336, "k": 4096, "bias": False},
        # a small layer on a token count that fills no block: every launch counts
        {"name": "train_ragged", "op": "mx_train", "t": 777, "n": 2048, "k": 1024},
        # the training step of the down projection on one micro-batch
        {"name": "train_microbatch", "op": "mx_train", "t": 16384, "n": 4096, "k": 14336},
        # both operand orientations of a small fp32 matrix with an odd row count
        {"name": "quant_small", "op": "mx_quant", "r": 333, "c": 512, "dtype": "f32", "scaled": False},
        # both orientations of normalised activations: 1/RMS and norm weight applied on the way
        {"name": "quant_activations", "op": "mx_quant", "r": 32768, "c": 4096, "dtype": "bf16", "scaled": True},
        # fp32 micro-batch accumulators of a small odd-sized stack, clipped into bf16 buckets
        {"name": "clip_small_odd", "op": "clip", "blocks": 6, "d": 257, "f": 515, "dtype": "f32", "max_norm": 1.0},
        # bf16 gradients of a four-block 4096 x 14336 stack
        {"name": "clip_stack", "op": "clip", "blocks": 4, "d": 4096, "f": 14336, "dtype": "bf16", "max_norm": 1.0},
        # a handful of decoded tokens: post-norm, channel gate, residual, next pre-norm
        {"name": "norm_tokens", "op": "norm_fwd", "t": 5, "d": 4096, "groups": 1, "dtype": "bf16", "next": True},
        # a micro-batch, wide rows, no gate
        {"name": "norm_microbatch", "op": "norm_fwd", "t": 16384, "d": 8192, "groups": 0, "dtype": "bf16", "next": True},
        # its backward where eight sequences each bring a gate of their own
        {"name": "norm_backward", "op": "norm_bwd", "t": 16000, "d": 4096, "groups": 8, "dtype": "bf16", "next": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["mx_linear", "mx_train", "mx_quant", "clip", "norm_fwd", "norm_bwd"])
    if op in ("mx_linear", "mx_train"):
        most = 16384 * 14336 * 4096
        while True:
            t, n, k = _log(rng, 1, 16384), _log(rng, 256, 28672), _log(rng, 256, 14336)
            n, k = n // 32 * 32, k // 32 * 32
            if op == "mx_linear":
                n += rng.choice([0, 8, 16, 24])   # any multiple of 8 output features
            if t * n * k <= most // (1 if op == "mx_linear" else 3):
                break
        if op == "mx_linear":
            return {"op": op, "m": t, "n": n, "k": k, "bias": rng.random() < 0.5}
        return {"op": op, "t": t, "n": n, "k": k}
    if op == "mx_quant":
        while True:
            r, c = _log(rng, 1, 32768), _log(rng, 32, 16384) // 32 * 32
            if r * c <= 32768 * 4096:
                return {"op": op, "r": r, "c": c, "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]),
                        "scaled": rng.random() < 0.5}
    if op == "clip":
        while True:
            b, d, f = _log(rng, 1, 48), _log(rng, 64, 4096), _log(rng, 64, 14336)
            if 3 * b * d * f <= 3 * 4 * 4096 * 14336:
                return {"op": op, "blocks": b, "d": d, "f": f, "dtype": rng.choice(["bf16", "f32"]),
                        "max_norm": rng.choice([0.1, 1.0, 1e4])}
    while True:
        g, per, d = rng.choice([0, 1, 1, 2, 5, 16]), _log(rng, 1, 16384), _log(rng, 64, 8192)
        d = d if rng.random() < 0.3 else d // 8 * 8
        t = per * max(g, 1)
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        if t * d * (2 if dtype == "f32" else 1) <= (16384 * 8192 if op == "norm_fwd" else 16000 * 4096):
            return {"op": op, "t": t, "d": d, "groups": g, "dtype": dtype, "next": rng.random() < 0.8}


def work(case):
    op = case["op"]
    if op == "mx_linear":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": 2 * m * k + n * k * 17 / 32 + 2 * m * n, "flops": 2 * m * n * k}
    if op == "mx_train":
        t, n, k = case["t"], case["n"], case["k"]
        return {"bytes": 2 * 2 * (t * k + n * k + t * n), "flops": 3 * 2 * t * n * k}
    if op == "mx_quant":
        r, c = case["r"], case["c"]
        return {"bytes": r * c * (4 if case["dtype"] == "f32" else 2) + 2 * c * (r + -(-r // 32) * 32), "flops": 0}
    if op == "clip":
        n = case["blocks"] * (case["d"] + 3 * case["d"] * case["f"])
        return {"bytes": n * ((2 if case["dtype"] == "bf16" else 4) + 2), "flops": 3 * n}
    t, d = case["t"], case["d"]
    size = 4 if case["dtype"] == "f32" else 2
    if op == "norm_fwd":
        return {"bytes": t * d * size * (4 if case["next"] else 3), "flops": 10 * t * d}
    return {"bytes": t * d * size * (6 if case["next"] else 4), "flops": 20 * t * d}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _normal(gen, shape, std=1.0, dtype=torch.float32):
    return (torch.randn(shape, device=DEV, generator=gen) * std).to(dtype)


def _activations(gen, shape, dtype=torch.bfloat16):
    """Token activations: normal values, some channels far larger than the rest."""
    x = torch.randn(shape, device=DEV, generator=gen)
    x *= torch.exp(0.5 * torch.randn(shape[-1], device=DEV, generator=gen))
    return x.to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    op = case["op"]
    if op == "mx_linear":
        m, n, k = case["m"], case["n"], case["k"]
        q = torch.randint(0, 256, (n, k // 2), device=DEV, generator=gen, dtype=torch.uint8)
        # one scale exponent per row and 32-block, stored in 128 x 4 atoms as the product reads them
        s = torch.randint(118, 124, (n, k // 32), device=DEV, generator=gen, dtype=torch.uint8)
        return {"op": op, "x": _activations(gen, (m, k)), "qw": q, "sw": _swizzle(s),
                "bias": _normal(gen, (n,), 1.0, torch.bfloat16) if case["bias"] else None}
    if op == "mx_train":
        t, n, k = case["t"], case["n"], case["k"]
        return {"op": op, "x": _activations(gen, (t, k)).requires_grad_(),
                "w": _normal(gen, (n, k), 0.02, torch.bfloat16).requires_grad_(),
                "dy": _normal(gen, (t, n), 1e-3, torch.bfloat16)}
    if op == "mx_quant":
        x = _activations(gen, (case["r"], case["c"]), DTYPES[case["dtype"]])
        row = gamma = None
        if case["scaled"]:
            row = torch.rsqrt(x.float().square().mean(1) + EPS)
            gamma = _normal(gen, (case["c"],), 0.1, torch.bfloat16) + 1
        return {"op": op, "x": x, "row_scale": row, "gamma": gamma}
    if op == "clip":
        d, f, dt = case["d"], case["f"], DTYPES[case["dtype"]]
        grads, buckets = [], []
        for _ in range(case["blocks"]):
            grads += [_normal(gen, (d,), 1e-2), _normal(gen, (2 * f, d), 1e-3, dt), _normal(gen, (d, f), 1e-3, dt)]
            buckets.append(torch.empty(d + 3 * d * f, device=DEV, dtype=torch.bfloat16))
        out = [v for b in buckets for v in (b[:d], b[d:d + 2 * d * f].view(2 * f, d), b[d + 2 * d * f:].view(d, f))]
        return {"op": op, "grads": grads, "buckets": buckets, "out": out, "max_norm": case["max_norm"]}
    t, d, g, dt = case["t"], case["d"], case["groups"], DTYPES[case["dtype"]]
    st = {"op": op, "b": _activations(gen, (t, d), dt), "gamma_post": _normal(gen, (d,), 0.1, dt) + 1,
          "gate": _normal(gen, (g, d), 0.5, dt) if g else None, "alpha": 1.0, "branch": 0.7,
          "gamma_pre": _normal(gen, (d,), 0.1, dt) + 1 if case["next"] else None}
    if op == "norm_fwd":
        st["x"] = _activations(gen, (t, d), dt)
        return st
    st["dy"] = _normal(gen, (t, d), 1e-2, dt)
    st["inv_b"] = torch.rsqrt(st["b"].float().square().mean(1) + EPS)
    if case["next"]:
        st["y"] = _activations(gen, (t, d), dt)
        st["inv_y"] = torch.rsqrt(st["y"].float().square().mean(1) + EPS)
        st["dn"] = _normal(gen, (t, d), 1e-2, dt)
    return st


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

_pkg = None


def _ops():
    """The package, imported the way its README says; only where ``own`` is true."""
    global _pkg
    if _pkg is None:
        import importlib
        import __graft_entry__
        __graft_entry__.import_package()
        _pkg = (importlib.import_module("nvfp4_b200.ops"), importlib.import_module("nvfp4_b200.float4utils"))
    return _pkg


def run(st):
    return (_run_own if own else _run_plain)(st)


def _run_own(st):
    ops, f4 = _ops()
    op = st["op"]
    if op == "mx_linear":
        return ops.mx_linear(st["x"], st["qw"], st["sw"], bias=st["bias"])
    if op == "mx_train":
        y = f4.mxfp4_linear(st["x"], st["w"])
        dx, dw = torch.autograd.grad(y, (st["x"], st["w"]), st["dy"])
        return {"y": y.detach(), "dx": dx, "dw": dw}
    if op == "mx_quant":
        q, s, qt, s_t = ops.mx_quantize_both(st["x"], row_scale=st["row_scale"], gamma=st["gamma"])
        return {"rows": ops.mx_dequantize(q, s), "cols": ops.mx_dequantize(qt, s_t)}
    if op == "clip":
        norm = ops.clip_grad_norm(st["grads"], st["max_norm"], out=st["out"])
        return {"norm": norm, "buckets": st["buckets"]}
    if op == "norm_fwd":
        y, n, inv_b, inv_y = ops.sandwich_norm(st["b"], st["x"], st["gamma_post"], st["gate"], st["gamma_pre"],
                                               residual_scale=st["alpha"], branch_scale=st["branch"], eps=EPS)
        return {"y": y, "n": n, "inv_b": inv_b, "inv_y": inv_y}
    if st["gamma_pre"] is not None:
        more = dict(dn=st["dn"], y=st["y"], inv_y=st["inv_y"], gamma_pre=st["gamma_pre"])
    else:
        more = {}
    return ops.sandwich_norm_bwd(st["dy"], st["b"], st["inv_b"], st["gamma_post"], st["gate"],
                                 residual_scale=st["alpha"], branch_scale=st["branch"], **more)


def _swizzle(s):
    """Block scales [rows, blocks] -> the padded 128 x 4-atom layout [round_up(rows, 128), round_up(blocks, 4)]."""
    r, c = s.shape
    pr, pc = -(-r // 128) * 128, -(-c // 4) * 4
    full = s.new_zeros((pr, pc))
    full[:r, :c] = s
    return full.view(pr // 128, 4, 32, pc // 4, 4).permute(0, 3, 2, 1, 4).reshape(pr, pc)


def _unswizzle(s, r, c):
    pr, pc = s.shape
    return s.view(pr // 128, pc // 4, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(pr, pc)[:r, :c]


def _power(e):
    """2^e in fp32 for integer e >= -127."""
    return torch.where(e > -127, (e + 127) << 23, torch.full_like(e, 1 << 22)).view(torch.float32)


def _mx(v):
    """The values that MXFP4 blocks of 32 along the last dimension stand for, in fp32."""
    b = v.reshape(*v.shape[:-1], -1, 32)
    amax = b.abs().amax(-1, keepdim=True)
    e = torch.where(amax > 0, torch.frexp(amax).exponent - 3, -127).clamp(min=-127).int()
    a = (b * ((127 - e) << 23).view(torch.float32))
    m = a.abs().clamp(max=6.0)
    step = torch.where(m < 2, 0.5, torch.where(m < 4, 1.0, 2.0))
    return (torch.copysign(torch.round(m / step) * step, a) * _power(e)).reshape(v.shape)


def _mx_t(v):
    """The same for the transpose, its rows (v's first dimension) filled up with zeros to whole blocks."""
    return _mx(torch.nn.functional.pad(v, (0, 0, 0, -v.shape[0] % 32)).t().contiguous())


def _codes(q):
    lo, hi = q & 15, q >> 4
    c = torch.stack((lo, hi), -1).reshape(q.shape[0], -1).long()
    table = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], device=q.device)
    return table[c]


def _run_plain(st):
    op = st["op"]
    if op == "mx_linear":
        n, k = st["qw"].shape[0], 2 * st["qw"].shape[1]
        scale = _power(_unswizzle(st["sw"], n, k // 32).int() - 127)
        w = (_codes(st["qw"]).view(n, k // 32, 32) * scale[..., None]).view(n, k)
        y = _mx(st["x"].float()) @ w.t()
        return (y if st["bias"] is None else y + st["bias"].float()).to(torch.bfloat16)
    if op == "mx_train":
        x, w, dy = st["x"].detach().float(), st["w"].detach().float(), st["dy"].float()
        return {"y": (_mx(x) @ _mx(w).t()).to(torch.bfloat16), "dx": (_mx(dy) @ _mx_t(w).t()).to(torch.bfloat16),
                "dw": (_mx_t(dy) @ _mx_t(x).t()).to(torch.bfloat16)}
    if op == "mx_quant":
        v = st["x"].float()
        if st["row_scale"] is not None:
            v = (v * st["row_scale"][:, None]) * st["gamma"].float()
        return {"rows": _mx(v).to(torch.bfloat16), "cols": _mx_t(v).to(torch.bfloat16)}
    if op == "clip":
        norm = torch.stack([g.double().square().sum() for g in st["grads"]]).sum().sqrt()
        coef = (st["max_norm"] / (norm + 1e-6)).clamp(max=1.0).float()
        flat = [(g.float() * coef).to(torch.bfloat16).reshape(-1) for g in st["grads"]]
        return {"norm": norm.float().reshape(1),
                "buckets": [torch.cat(flat[i:i + 3]) for i in range(0, len(flat), 3)]}
    b, gp = st["b"].float(), st["gamma_post"].float()
    gate = 1.0 if st["gate"] is None else st["gate"].float().repeat_interleave(b.shape[0] // st["gate"].shape[0], 0)
    if op == "norm_fwd":
        inv_b = torch.rsqrt(b.square().mean(1) + EPS)
        y = st["alpha"] * st["x"].float() + st["branch"] * gate * (b * inv_b[:, None] * gp)
        n = inv_y = None
        if st["gamma_pre"] is not None:
            inv_y = torch.rsqrt(y.square().mean(1) + EPS)
            n = (y * inv_y[:, None] * st["gamma_pre"].float()).to(st["b"].dtype)
        return {"y": y.to(st["b"].dtype), "n": n, "inv_b": inv_b, "inv_y": inv_y}
    total, dpre = st["dy"].float(), None
    if st["gamma_pre"] is not None:
        yn, dn = st["y"].float() * st["inv_y"][:, None], st["dn"].float()
        v = dn * st["gamma_pre"].float()
        total = total + st["inv_y"][:, None] * (v - yn * (v * yn).mean(1, keepdim=True))
        dpre = (dn * yn).sum(0)
    bn = b * st["inv_b"][:, None]
    u = st["branch"] * total * gate * gp
    db = st["inv_b"][:, None] * (u - bn * (u * bn).mean(1, keepdim=True))
    each = st["branch"] * total * bn
    dgate = None
    if st["gate"] is not None:
        dgate = (each * gp).view(st["gate"].shape[0], -1, b.shape[1]).sum(1)
    return {"dx": (st["alpha"] * total).to(st["b"].dtype), "db": db.to(st["b"].dtype),
            "dgamma_post": (each * gate).sum(0), "dgate": dgate, "dgamma_pre": dpre}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _blocks64(v):
    """MXFP4 along the last dimension in 64 bits: the shared exponent is
    floor(log2(amax)) - 2, not below -127; each value goes to the nearest
    point of the grid, ties to the point of even index, 6 at most."""
    grid = torch.tensor(_GRID, device=v.device, dtype=torch.float64)
    out = torch.empty_like(v)
    rows = max(1, (1 << 26) // v.shape[1])
    for lo in range(0, v.shape[0], rows):   # in pieces, for memory
        w = v[lo:lo + rows].unflatten(1, (-1, 32))
        top = w.abs().amax(2, keepdim=True)
        field = (top.view(torch.int64) >> 52) & 0x7FF
        e = (field - 1023 - 2).clamp(min=-127)
        x = w.abs() * ((1023 - e) << 52).view(torch.float64)
        hi = torch.searchsorted(grid, x).clamp(max=7)
        below = (hi - 1).clamp(min=0)
        du, dl = grid[hi] - x, x - grid[below]
        pick = torch.where((du < dl) | ((du == dl) & (hi % 2 == 0)), hi, below)
        out[lo:lo + rows] = (torch.sign(w) * grid[pick] * ((1023 + e) << 52).view(torch.float64)).flatten(1)
    return out


def _cols64(v):
    r = -(-v.shape[0] // 32) * 32
    full = v.new_zeros((r, v.shape[1]))
    full[:v.shape[0]] = v
    return _blocks64(full.T.contiguous())


def exact(case, seed):
    st = prepare(case, seed)
    f64 = lambda t: t.detach().double()  # noqa: E731
    op = case["op"]
    if op == "mx_linear":
        n, k = case["n"], case["k"]
        idx = torch.empty((n, k), device=DEV, dtype=torch.uint8)
        idx[:, 0::2], idx[:, 1::2] = st["qw"] % 16, st["qw"] // 16
        w = torch.tensor(_GRID, device=DEV, dtype=torch.float64)[(idx % 8).int()]
        w[idx >= 8] *= -1
        r, c = torch.arange(n, device=DEV)[:, None], torch.arange(k // 32, device=DEV)[None]
        at = (r // 128 * (st["sw"].shape[1] // 4) + c // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + c % 4
        s = torch.exp2(st["sw"].flatten()[at].double() - 127)
        y = _blocks64(f64(st["x"])) @ (w * s.repeat_interleave(32, 1)).T
        return y if st["bias"] is None else y + f64(st["bias"])
    if op == "mx_train":
        x, w, dy = f64(st["x"]), f64(st["w"]), f64(st["dy"])
        return {"y": _blocks64(x) @ _blocks64(w).T, "dx": _blocks64(dy) @ _cols64(w).T, "dw": _cols64(dy) @ _cols64(x).T}
    if op == "mx_quant":
        v = f64(st["x"])
        if case["scaled"]:
            v = v * f64(st["row_scale"]).unsqueeze(1) * f64(st["gamma"])
        return {"rows": _blocks64(v), "cols": _cols64(v)}
    if op == "clip":
        total = 0.0
        for g in st["grads"]:
            total += float(torch.linalg.vector_norm(f64(g))) ** 2
        norm = math.sqrt(total)
        c = min(1.0, case["max_norm"] / (norm + 1e-6))
        return {"norm": torch.tensor([norm], dtype=torch.float64, device=DEV),
                "buckets": [torch.cat([f64(g).flatten() for g in st["grads"][i:i + 3]]) * c
                            for i in range(0, len(st["grads"]), 3)]}
    t, d, g = case["t"], case["d"], case["groups"]
    b, gp = f64(st["b"]), f64(st["gamma_post"])
    gate = f64(st["gate"]) if g else torch.ones((1, d), device=DEV, dtype=torch.float64)
    rows = t // gate.shape[0]
    by = lambda z: z.view(-1, rows, d)  # noqa: E731
    if op == "norm_fwd":
        ib = (b.pow(2).sum(1) / d + EPS).pow(-0.5)
        branch = by(b * ib.view(t, 1) * gp) * gate[:, None] * st["branch"]
        y = branch.view(t, d) + f64(st["x"]) * st["alpha"]
        if not case["next"]:
            return {"y": y, "n": None, "inv_b": ib, "inv_y": None}
        iy = (y.pow(2).sum(1) / d + EPS).pow(-0.5)
        return {"y": y, "n": y * iy.view(t, 1) * f64(st["gamma_pre"]), "inv_b": ib, "inv_y": iy}
    up, dpre = f64(st["dy"]), None
    if case["next"]:
        iy, dn = f64(st["inv_y"]).view(t, 1), f64(st["dn"])
        yh = f64(st["y"]) * iy
        dyh = dn * f64(st["gamma_pre"])
        up = up + iy * dyh - iy * yh * ((dyh * yh).sum(1, keepdim=True) / d)
        dpre = torch.einsum("td,td->d", dn, yh)
    ib = f64(st["inv_b"]).view(t, 1)
    bh = b * ib
    dbh = (by(up) * (gate * gp * st["branch"])[:, None]).view(t, d)
    db = ib * dbh - ib * bh * ((dbh * bh).sum(1, keepdim=True) / d)
    sums = torch.einsum("grd,grd->gd", by(up), by(bh)) * st["branch"]
    return {"dx": up * st["alpha"], "db": db, "dgamma_post": (sums * gate).sum(0), "dgate": sums * gp if g else None,
            "dgamma_pre": dpre}
