"""Clipping at the ends of its arguments' ranges: limits that are infinite (or
past fp32), which measure the norm and clip nothing, with finite and infinite
gradients."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("max_norm", [math.inf, 1e39, 1e300, 1.0])
@pytest.mark.parametrize("kind", [2, math.inf])
def test_infinite_norm(pkg, max_norm, kind):
    """An infinite norm makes every output 0, NaN where the gradient was infinite."""
    ops = pkg.ops
    for bad in (math.inf, -math.inf):
        g = [torch.randn(5000, device="cuda").to(torch.bfloat16), torch.randn(300, device="cuda")]
        g[1][7] = bad
        out = [torch.full_like(t, 3) for t in g]
        assert ops.clip_grad_norm(g, max_norm, kind, out=out).item() == math.inf
        assert (out[0] == 0).all() and torch.isnan(out[1][7]) and torch.isnan(out[1]).sum() == 1
        n, c = ops.grad_norm_coef(g, max_norm, kind)
        assert n.item() == math.inf and c.item() == 0
        total = torch.cat([ops.grad_norm_total([t], kind) for t in g])
        n, c = ops.grad_norm_finish(total, max_norm, kind)
        assert n.item() == math.inf and c.item() == 0
        g[0][0] = math.nan
        n, c = ops.grad_norm_coef(g, max_norm, kind)
        assert math.isnan(n.item()) and math.isnan(c.item())


@pytest.mark.parametrize("max_norm", [math.inf, 1e39, 1e300])
def test_no_limit_changes_nothing(pkg, max_norm):
    ops = pkg.ops
    g = [torch.randn(5000, device="cuda").to(torch.bfloat16), torch.randn(300, device="cuda") * 1e30]
    keep = [t.clone() for t in g]
    n = ops.clip_grad_norm(g, max_norm)
    assert math.isfinite(n.item()) and all(torch.equal(a, b) for a, b in zip(g, keep))
    assert ops.grad_norm_coef(g, max_norm)[1].item() == 1
