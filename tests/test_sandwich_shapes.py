"""mlp.sandwich_norm with a residual stream of another shape than the block's
output: the same rows laid out otherwise get their gradient in their own shape,
rows of another width are refused.  On CPU with plain stand-ins."""
import pytest
import torch

from test_sandwich_autograd import mlp, plain  # noqa: F401  (the fixture)


@pytest.mark.parametrize("bshape,xshape", [((2, 3, 8), (6, 8)), ((6, 8), (2, 3, 8)), ((2, 3, 8), (3, 2, 8)), ((8,), (1, 8))])
@pytest.mark.parametrize("pre", [False, True])
def test_gradients_in_their_own_shapes(plain, bshape, xshape, pre):  # noqa: F811
    gen = torch.Generator().manual_seed(3)
    b, x = (torch.randn(s, generator=gen, dtype=torch.float64).requires_grad_() for s in (bshape, xshape))
    out = mlp.sandwich_norm(b, x, pre=pre)
    outs = out if pre else (out,)
    assert all(o.shape == b.shape for o in outs)
    ups = [torch.randn(bshape, generator=gen, dtype=torch.float64) for _ in outs]
    gb, gx = torch.autograd.grad(outs, (b, x), ups)
    assert gb.shape == b.shape and gx.shape == x.shape
    same = x.detach().reshape(bshape).requires_grad_()
    out = mlp.sandwich_norm(b, same, pre=pre)
    rb, rx = torch.autograd.grad(out if pre else (out,), (b, same), ups)
    assert torch.equal(gb, rb) and torch.equal(gx, rx.reshape(xshape))


def test_rows_of_another_width(plain):  # noqa: F811
    b, x = torch.randn(4, 8, dtype=torch.float64), torch.randn(2, 16, dtype=torch.float64)
    for args in ((b, x), (x, b)):
        with pytest.raises(RuntimeError, match="width"):
            mlp.sandwich_norm(*args)
