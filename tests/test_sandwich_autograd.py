"""The autograd function around the sandwich norms, on CPU with a plain stand-in
for the two kernels: shapes, what may change in place, which gradients come."""
import importlib
import os
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
import __graft_entry__ as graft  # noqa: E402

graft.import_package()
mlp = importlib.import_module("nvfp4_b200.mlp")


def _parts(b, x, gp, gate, gn, alpha, s, eps, pre):
    t, d = b.shape
    inv_b = torch.rsqrt(b.square().mean(1) + eps)
    u = b * inv_b[:, None]
    if gp is not None:
        u = u * gp
    if gate is not None:
        g = gate.reshape(-1, d)
        u = u * g.repeat_interleave(t // g.shape[0], 0)
    y = alpha * x + s * u
    if not pre:
        return y, None, inv_b, None
    inv_y = torch.rsqrt(y.square().mean(1) + eps)
    n = y * inv_y[:, None]
    return y, n if gn is None else n * gn, inv_b, inv_y


@pytest.fixture
def plain(monkeypatch):
    """fp64 stand-ins; the backward rebuilds what it needs from the y it is handed."""
    seen = {}

    def fwd(b, x, gp, gate, gn, *, residual_scale, branch_scale, eps, pre):
        pre = gn is not None if pre is None else pre
        seen.update(x=x.clone(), args=(residual_scale, branch_scale, eps, pre))
        with torch.no_grad():
            return _parts(b, x, gp, gate, gn, *seen["args"])

    def bwd(dy, b, inv_b, gp, gate, *, dn=None, y=None, inv_y=None, gamma_pre=None, residual_scale, branch_scale):
        assert b.dim() == 2 and all(t is None or t.shape == b.shape for t in (dy, dn, y))
        leaves = [None if t is None else t.detach().clone().requires_grad_() for t in (seen["x"], b, gp, gate, gamma_pre)]
        with torch.enable_grad():
            out = _parts(leaves[1], leaves[0], leaves[2], leaves[3], leaves[4], *seen["args"])
            if y is not None:
                assert torch.equal(out[0], y)
            pairs = [(o, g) for o, g in zip(out[:2], (dy, dn)) if g is not None]
            wrt = [t for t in leaves if t is not None]
            grads = iter(torch.autograd.grad([o for o, _ in pairs], wrt, [g for _, g in pairs], allow_unused=True))
        vals = [None if t is None else next(grads) for t in leaves]
        return dict(zip(("dx", "db", "dgamma_post", "dgate", "dgamma_pre"), vals))

    monkeypatch.setattr(mlp.ops, "sandwich_norm", fwd)
    monkeypatch.setattr(mlp.ops, "sandwich_norm_bwd", bwd)


def _inputs(shape, pre=True):
    gen = torch.Generator().manual_seed(5)
    d = shape[-1]
    new = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64).requires_grad_()
    return new(*shape), new(*shape), new(d), new(shape[0], d), new(d) if pre else None


@pytest.mark.parametrize("shape", [(6, 8), (2, 3, 8), (2, 1, 3, 8)])
def test_gradients_against_differences(plain, shape):
    assert torch.autograd.gradcheck(
        lambda *a: mlp.sandwich_norm(*a, residual_scale=0.75, branch_scale=-0.5), _inputs(shape))


@pytest.mark.parametrize("shape", [(6, 8), (2, 3, 8)])
def test_changes_in_place(plain, shape):
    """y is read again by the backward of n: a change of it in between is refused,
    a change of n, or of y where there is no n, is taken into account."""
    ins = _inputs(shape)
    y, n = mlp.sandwich_norm(*ins)
    y.mul_(2)
    with pytest.raises(RuntimeError, match="inplace"):
        (y.sum() + n.sum()).backward()
    y, n = mlp.sandwich_norm(*ins)
    n.mul_(2)
    got = torch.autograd.grad(n.sum(), ins[0])[0]
    ref = torch.autograd.grad(2 * mlp.sandwich_norm(*ins)[1].sum(), ins[0])[0]
    assert torch.equal(got, ref)
    ins = _inputs(shape, pre=False)
    y = mlp.sandwich_norm(*ins)
    y.mul_(2)
    got = torch.autograd.grad(y.sum(), ins[0])[0]
    ref = torch.autograd.grad(2 * mlp.sandwich_norm(*ins).sum(), ins[0])[0]
    assert torch.equal(got, ref)
