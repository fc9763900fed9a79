"""One training step of MXFP4 linear layers around the two norms, with clipping
and AdamW, part by part: every activation, gradient and updated parameter
against float64 (AdamW: against the float32 oracle, bit for bit) on the values
that reached the part.  Tolerances as derived in test_mx_quant_gpu.py (products),
test_sandwich_gpu.py (norms) and test_grad_clip_gpu.py (clipping)."""
import importlib
import math

import numpy as np
import pytest
import torch

from oracle import adamw_oracle
from test_grad_clip_gpu import REL, check_scaled
from test_mx_quant_gpu import check, f64, product
from test_sandwich_gpu import BF, F32, backward64, close, forward64, rnd

pytestmark = pytest.mark.gpu
HP = dict(lr=1e-2, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.1)


def bits(t):
    return t.detach().cpu().view(torch.int16).numpy().view(np.uint16)


@pytest.mark.parametrize("t,groups", [(70, 1), (96, 4)])
def test_step(pkg, f4, t, groups):
    ops = pkg.ops
    mlp = importlib.import_module("nvfp4_b200.mlp")
    torch.manual_seed(1)
    d, f, c = 256, 512, 64
    up, down = f4.MXFP4Linear(d, f, bias=False, device="cuda"), f4.MXFP4Linear(f, d, bias=False, device="cuda")
    head = f4.MXFP4Linear(d, c, bias=True, device="cuda")
    gp, gn = (torch.nn.Parameter(rnd((d,), 10 + i, BF, 0.1) + 1) for i in range(2))
    gate = torch.nn.Parameter(rnd((groups, d), 12, BF, 0.1) + 1)
    params = [up.weight, down.weight, head.weight, head.bias, gp, gate, gn]
    x, dz = rnd((t, d), 1, BF), rnd((t, c), 2, BF, 0.5)
    al, s, eps = 0.9, 0.5, 1e-6

    a = up(x)
    r = torch.relu(a)
    b = down(r)
    y, n = mlp.sandwich_norm(b, x, gp, gate, gn, residual_scale=al, branch_scale=s, eps=eps)
    z = head(n)
    for v in (a, r, b, y, n, z):
        v.retain_grad()
    (z.float() * dz.float()).sum().add(y.float().square().mean() * 50).backward()

    # forward
    mul = lambda p, q: product(*ops.mx_quantize(p.detach()), *ops.mx_quantize(q.detach()), p.shape[0], q.shape[0], p.shape[1])
    check(a, *mul(x, up.weight))
    check(b, *mul(r, down.weight))
    ry, rib, mag = forward64(b.detach(), x, gp.detach(), gate.detach(), gn.detach(), al, s, eps)
    close(y.detach(), ry, mag, BF)
    riy = (ry.square().mean(1) + eps).rsqrt()
    off = riy * (mag.square().mean(1) + eps).sqrt()
    close(n.detach(), ry * riy[:, None] * gn.double(), (mag * (1 + off[:, None])) * riy[:, None] * gn.double().abs(), BF)
    ref, big = mul(n, head.weight)
    bias = f64(head.bias)
    check(z, ref + bias, big + np.abs(bias))

    # backward
    assert torch.equal(z.grad, dz)

    def layer_back(dy, inp, weight, din):
        rows, pr = dy.shape[0], -(-dy.shape[0] // 32) * 32
        n_, k_ = weight.shape
        w = weight.detach()
        check(din, *product(*ops.mx_quantize(dy), *ops.mx_quantize_t(w), rows, k_, n_))
        check(weight.grad, *product(*ops.mx_quantize_t(dy), *ops.mx_quantize_t(inp.detach()), n_, k_, pr))

    layer_back(dz, n, head.weight, n.grad)
    ref = f64(dz).sum(0)
    assert (np.abs(f64(head.bias.grad) - ref) <= np.abs(ref) * 2.0 ** -8 + np.abs(f64(dz)).sum(0) * 2.0 ** -18).all()
    want = y.detach().double() * (100.0 / y.numel())
    assert ((y.grad.double() - want).abs() <= want.abs() * (2.0 ** -8 + 2.0 ** -20) + 2.0 ** -133).all()   # three fp32 products, one bf16 rounding
    ib, iy = ops.sandwich_norm(b.detach(), x, gp.detach(), gate.detach(), gn.detach(), residual_scale=al, branch_scale=s, eps=eps)[2:]
    ref, big = backward64(y.grad, n.grad, b.detach(), y.detach(), ib, iy, gp.detach(), gate.detach(), gn.detach(), al, s)
    close(b.grad, ref["db"], big["db"], BF)
    for p, k in ((gp, "dgamma_post"), (gate, "dgate"), (gn, "dgamma_pre")):
        close(p.grad, ref[k], big[k], BF, extra=F32 + (t + 64) * 2.0 ** -24)
    layer_back(b.grad, r, down.weight, r.grad)
    assert torch.equal(a.grad, r.grad * (a.detach() > 0))
    dn_up = a.grad
    pr = -(-t // 32) * 32
    check(up.weight.grad, *product(*ops.mx_quantize_t(dn_up), *ops.mx_quantize_t(x), f, d, pr))

    # clipping
    grads = [p.grad for p in params]
    keep = [g.clone() for g in grads]
    norm = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
    got = ops.clip_grad_norm(grads, norm / 3)
    assert abs(got.item() - norm) <= REL * norm
    check_scaled(grads, keep, 1 / 3 * norm / (norm + 1e-6))

    # AdamW: two steps with the clipped gradients
    for p, g in zip(params, grads):
        m, v = torch.zeros(p.numel(), device="cuda"), torch.zeros(p.numel(), device="cuda")
        q, om, ov = bits(p).reshape(-1), np.zeros(p.numel(), np.float32), np.zeros(p.numel(), np.float32)
        for step in (1, 2):
            ops.adamw_step(p.data.view(-1), g.view(-1), m, v, step=step, **HP)
            q, om, ov = adamw_oracle.adamw_bf16(q, bits(g).reshape(-1), om, ov, step=step, **HP)
        assert np.array_equal(bits(p).reshape(-1), q)
    assert ops.device_error() == 0
