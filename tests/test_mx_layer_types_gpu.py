"""The MXFP4 layer's types: what a gradient is rounded to on its way.  Tolerances
as in test_mx_quant_gpu.py: 2^-20 of the sum of the terms' magnitudes for fp32
accumulation, and half a step of the type that the result is stored in."""
import numpy as np
import pytest
import torch

from test_mx_quant_gpu import f64, make, product

pytestmark = pytest.mark.gpu


def within(got, ref, mag):
    f = torch.finfo(got.dtype)
    acc = mag * 2.0 ** -20
    tol = acc + (np.abs(ref) + acc) * (f.eps / 2) + f.smallest_normal * f.eps / 2
    err = np.abs(f64(got) - ref)
    assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("xtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("wtype", [torch.bfloat16, torch.float16, torch.float32])
def test_weight_gradient_has_the_weights_precision(pkg, f4, xtype, wtype):
    """Rounded once, to the weight's type: an fp16 weight's gradient has 11 significant bits."""
    ops = pkg.ops
    t, n, k = 77, 96, 160
    x, w, dy = make(t, k, xtype, 1), (make(n, k, wtype, 2) * 0.05).requires_grad_(), make(t, n, xtype, 3) * 0.1
    dw, = torch.autograd.grad(f4.mxfp4_linear(x, w), w, dy)
    assert dw.dtype == wtype
    within(dw, *product(*ops.mx_quantize_t(dy), *ops.mx_quantize_t(x), n, k, 96))


@pytest.mark.parametrize("m", [1, 37, 300])
def test_bias_that_starts_anywhere(pkg, f4, m):
    """A slice of a flat buffer off a 16-byte boundary, and a strided one: the bits of a bias of its own."""
    ops = pkg.ops
    n, k = 264, 128
    flat = make(1, 3 * n, torch.bfloat16, 9).view(-1)
    x, w = make(m, k, torch.bfloat16, 1), make(n, k, torch.bfloat16, 2)
    (qx, sx), (qw, sw) = ops.mx_quantize(x), ops.mx_quantize(w)
    for bias in (flat[3:3 + n], flat[8:8 + n], flat[:2 * n:2]):
        own = bias.clone()
        assert torch.equal(ops.mx_linear(x, qw, sw, bias=bias), ops.mx_linear(x, qw, sw, bias=own))
        assert torch.equal(ops.mx_gemm(qx, sx, qw, sw, bias=bias), ops.mx_gemm(qx, sx, qw, sw, bias=own))
        assert torch.equal(f4.mxfp4_linear(x, w, bias), f4.mxfp4_linear(x, w, own))
    lone = torch.nn.Parameter(flat[5:5 + n])
    f4.mxfp4_linear(x[:, :k], w[:256], lone[:256]).sum().backward()
    assert lone.grad is not None and (lone.grad[:256] != 0).all()
