"""The C ABI from a host thread that has made no CUDA call yet: the entry points
whose operands travel by tensor maps, which the driver encodes only where a
context is current."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def calls(pkg):
    lib, ops = pkg._lib.load(), pkg.ops
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(256, 512, device="cuda", generator=g).to(BF)
    w = torch.randn(128, 512, device="cuda", generator=g).to(BF)
    (q, s), (qw, sw) = ops.mx_quantize(x), ops.mx_quantize(w)
    (nq, ns), (nqw, nsw) = ops.quantize(x), ops.quantize(w)
    y = torch.zeros(256, 128, device="cuda", dtype=BF)
    qt, st = ops.quantize_t(x)
    qt0, st0 = torch.zeros_like(qt), torch.zeros_like(st)
    p = lambda t: t.data_ptr()
    one, mx = ops.mx_linear(x[:1], qw, sw), ops.mx_gemm(q, s, qw, sw)
    return {
        "mx_linear": (lambda k=(x, qw, sw): lib.nvfp4b200_mx_linear(p(x), p(qw), p(sw), None, None, None, p(y), 1, 128, 512, 512, None),
                      y[:1], one),
        "mx_gemm": (lambda k=(q, s, qw, sw): lib.nvfp4b200_mx_gemm(p(q), p(qw), p(s), p(sw), None, None, p(y), 0, 0, 0, 256, 128, 512, 128,
                                                                  None), y, mx),
        "nvfp4_mm": (lambda k=(nq, ns, nqw, nsw): lib.nvfp4b200_nvfp4_mm(p(nq), p(nqw), p(ns), p(nsw), None, None, p(y), 256, 128, 512,
                                                                        None), y, ops.gemm(nq, ns, nqw, nsw)),
        "quantize_t": (lambda k=x: lib.nvfp4b200_quant_nvfp4_t(p(x), None, None, p(qt0), p(st0), 256, 512, None, None), qt0, qt),
    }


@pytest.mark.parametrize("name", ["mx_linear", "mx_gemm", "nvfp4_mm", "quantize_t"])
def test_first_call_of_a_thread(pkg, name):
    call, out, ref = calls(pkg)[name]
    torch.cuda.synchronize()
    rc = []
    t = threading.Thread(target=lambda: rc.append(call()))
    t.start()
    t.join()
    torch.cuda.synchronize()
    assert rc == [0]
    assert torch.equal(out, ref)
