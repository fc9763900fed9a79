"""The few-token product where the last tile of weight rows is partly filled and
K is cut over a cluster: some lanes of a warp have rows to write, others none."""
import numpy as np
import pytest
import torch

from test_mx_quant_gpu import check, f64, make, product

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m", [1, 5, 12, 13, 40, 100])
@pytest.mark.parametrize("n", [8, 120, 136, 264, 1016])
def test_ragged_rows_with_k_in_parts(pkg, m, n):
    ops = pkg.ops
    k = 8192                                   # 32 stages: 8 parts
    x, w = make(m, k, torch.bfloat16, 1), make(n, k, torch.bfloat16, 2) * 0.05
    bias = (torch.randn(n, device="cuda") * 3).to(torch.bfloat16)
    qw, sw = ops.mx_quantize(w)
    y = ops.mx_linear(x, qw, sw, bias=bias)
    ref, mag = product(*ops.mx_quantize(x), qw, sw, m, n, k)
    check(y, ref + f64(bias), mag + np.abs(f64(bias)))
    for _ in range(20):
        assert torch.equal(ops.mx_linear(x, qw, sw, bias=bias), y)
    assert ops.device_error() == 0
