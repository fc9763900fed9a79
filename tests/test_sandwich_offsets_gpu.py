"""The norms on tensors that start off a 16-byte boundary (slices of flat
buffers), at every number of threads a row can take, with one gate, a gate per
few rows and none: the kernels that read single elements straight from global
memory.  Tolerances as derived in test_sandwich_gpu.py; there too a row's
thread adds at most 16 terms."""
import math

import pytest
import torch

from test_sandwich_gpu import BF, F32, FL, HF, backward64, close, forward64, rnd

pytestmark = pytest.mark.gpu


def beside(t, d, seed, dtype, std=1.0):
    """[t, d] one element past a 16-byte boundary, with NaN around it."""
    flat = torch.full((t * d + 32,), math.nan, device="cuda", dtype=dtype)
    flat[17:17 + t * d] = rnd((t * d,), seed, dtype, std)
    v = flat[17:17 + t * d].view(t, d)
    assert v.data_ptr() % 16 != 0
    return v


WIDTHS = [7, 512, 1000, 1024, 1536, 2048, 2560, 4096, 4097, 5120, 6144, 8192, 8193, 12296, 16384]


@pytest.mark.parametrize("dtype", [BF, HF, FL])
@pytest.mark.parametrize("d", WIDTHS)
@pytest.mark.parametrize("form", ["one gate", "many gates", "no gate"])
def test_forward_backward(pkg, d, form, dtype):
    ops = pkg.ops
    per, groups = {"one gate": (301, 1), "many gates": (2, 500 if d <= 8192 else 250), "no gate": (150, 1)}[form]
    t = per * groups
    b, x, dy, dn = (beside(t, d, i, dtype, s) for i, s in ((1, 2.0), (2, 1.0), (3, 0.1), (4, 0.1)))
    gp, gn = rnd((d,), 5, dtype, 0.3) + 1, rnd((d,), 7, dtype, 0.3) + 1
    gate = None if form == "no gate" else rnd((groups, d), 6, dtype)
    y, n, ib, iy = ops.sandwich_norm(b, x, gp, gate, gn, residual_scale=0.9, branch_scale=0.7)
    ry, rib, mag = forward64(b, x, gp, gate, gn, 0.9, 0.7, 1e-6)
    close(ib, rib, rib)
    close(y, ry, mag, dtype)
    riy = (ry.square().mean(1) + 1e-6).rsqrt()
    off = riy * (mag.square().mean(1) + 1e-6).sqrt()
    close(n, ry * riy[:, None] * gn.double(), (mag * (1 + off[:, None])) * riy[:, None] * gn.double().abs(), dtype)
    for kw in (dict(dn=dn, y=y, inv_y=iy, gamma_pre=gn), {}):
        got = ops.sandwich_norm_bwd(dy, b, ib, gp, gate, residual_scale=0.9, branch_scale=0.7, **kw)
        ref, big = backward64(dy, kw.get("dn"), b, y, ib, iy, gp, gate, gn, 0.9, 0.7)
        for k in ("dx", "db"):
            close(got[k], ref[k], big[k], dtype)
        for k in ("dgamma_post", "dgate", "dgamma_pre"):
            if got[k] is not None:
                close(got[k], ref[k], big[k], extra=F32 + (t + 64) * 2.0 ** -24)
        again = ops.sandwich_norm_bwd(dy, b, ib, gp, gate, residual_scale=0.9, branch_scale=0.7, **kw)
        assert all(got[k] is None or torch.equal(got[k], again[k]) for k in got)
    assert ops.device_error() == 0
