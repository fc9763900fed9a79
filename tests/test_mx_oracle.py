"""CPU tests of the MXFP4 quantizer's restatement (oracle/mx_oracle.py)
against hand-worked values, and of the argument checks that need no device."""
import numpy as np
import pytest
import torch

from oracle import mx_oracle as mxo, nvfp4_oracle as orc


def test_grid_ties_go_to_even_codes():
    ties = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    assert mxo.encode(ties).tolist() == [0, 2, 2, 4, 4, 6, 6]
    assert mxo.encode(np.nextafter(ties, 9)).tolist() == [1, 2, 3, 4, 5, 6, 7]
    assert mxo.encode(np.nextafter(ties, 0)).tolist() == [0, 1, 2, 3, 4, 5, 6]
    assert mxo.encode(np.array([6.0, 6.9, 7.99])).tolist() == [7, 7, 7]


@pytest.mark.parametrize("amax,code", [(1.0, 125), (1.99, 125), (2.0, 126), (6.0, 127), (7.9, 127), (8.0, 128),
                                       (2.0 ** -125, 0), (2.0 ** -124, 1), (1e-40, 0), (0.0, 0),
                                       (3.3e38, 252)])
def test_block_exponents(amax, code):
    v = np.zeros((1, 32))
    v[0, 7] = amax
    _, s = mxo.quantize(v)
    assert s.reshape(-1)[0] == code


def test_round_trip_keeps_representable_values():
    rng = np.random.default_rng(0)
    v = mxo.GRID[rng.integers(0, 8, (5, 64))] * rng.choice([-1, 1], (5, 64))
    v[:, 0::32] = 6.0
    v *= np.ldexp(1.0, rng.integers(-20, 20, (5, 2))).repeat(32, 1)
    q, s = mxo.quantize(v)
    assert np.array_equal(orc.dequant_mxfp4(q, s, 5, 64), v)


def test_non_finite_blocks_become_nan():
    v = np.ones((1, 96))
    v[0, 3], v[0, 40] = np.inf, np.nan
    q, s = mxo.quantize(v)
    d = orc.dequant_mxfp4(q, s, 1, 96)
    assert np.isnan(d[0, :64]).all() and (d[0, 64:] == 1).all()


def test_transpose_pads_rows_with_zeros():
    v = np.random.default_rng(1).standard_normal((5, 8))
    q, s = mxo.quantize_t(v)
    d = orc.dequant_mxfp4(q, s, 8, 32)
    assert (d[:, 5:] == 0).all() and np.abs(d[:, :5] - v.T).max() <= np.abs(v).max() / 4


def test_wrappers_refuse_host_tensors(pkg, f4):
    import importlib
    mlp = importlib.import_module("nvfp4_b200.mlp")
    ops = pkg.ops
    x = torch.zeros(32, 64, dtype=torch.bfloat16)
    u8 = torch.zeros(32, 32, dtype=torch.uint8)
    for call in (lambda: ops.mx_quantize(x), lambda: ops.mx_quantize_t(x), lambda: ops.mx_quantize_both(x),
                 lambda: ops.mx_dequantize(u8, u8), lambda: ops.mx_gemm(u8, u8, u8, u8),
                 lambda: ops.mx_linear(x, u8, u8), lambda: f4.mxfp4mm(x, x), lambda: f4.mxfp4_linear(x, x),
                 lambda: ops.grad_norm([x]), lambda: ops.clip_grad_norm([x], 1.0), lambda: ops.sandwich_norm(x, x),
                 lambda: ops.sandwich_norm_bwd(x, x, x[:, 0].float()), lambda: mlp.sandwich_norm(x, x)):
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(ValueError):
        mlp.NVFP4SwiGLUMLP(64, 128, gate=True)


FAKE = 1 << 20            # 16-byte aligned, never dereferenced: validation fails first
MIS = FAKE + 2


def _ptrs(*p):
    import ctypes
    return (ctypes.c_void_p * len(p))(*p)


def _ints(*v):
    import ctypes
    return (ctypes.c_int * len(v))(*v)


def _longs(*v):
    import ctypes
    return (ctypes.c_int64 * len(v))(*v)


def _norm(L, grads, dts, outs, odts, lens, count, kind=2, scale=1.0, mx=1.0, ws=FAKE, words=4096, norm=FAKE):
    return L.nvfp4b200_grad_norm(grads, dts, outs, odts, lens, count, kind, scale, mx, ws, words, norm, None, None, None)


def _fwd(L, b=FAKE, x=FAKE, gp=None, gate=None, gn=None, y=FAKE, n=None, ib=FAKE, iy=None, dt=0, rows=4, d=64, g=0,
         ldb=64, ldx=64):
    return L.nvfp4b200_sandwich_norm(b, x, gp, gate, gn, y, n, ib, iy, dt, rows, d, g, ldb, ldx, 1.0, 1.0, 1e-6, None)


def _bwd(L, dy=FAKE, dn=None, b=FAKE, y=None, ib=FAKE, iy=None, gate=None, gn=None, dx=FAKE, dgate=None, dgn=None,
         dt=0, rows=4, d=64, g=0, ld=64):
    return L.nvfp4b200_sandwich_norm_bwd(dy, dn, b, y, ib, iy, None, gate, gn, dx, FAKE, FAKE, dgate, dgn, FAKE, 1 << 30,
                                         dt, rows, d, g, ld, ld, ld, ld, 1.0, 1.0, None)


@pytest.mark.parametrize("call,expected", [
    (lambda L: L.nvfp4b200_mx_quant(None, 0, None, None, FAKE, FAKE, None, None, 4, 64, 64, None), 1),
    (lambda L: L.nvfp4b200_mx_quant(FAKE, 0, None, None, None, None, None, None, 4, 64, 64, None), 1),   # no output
    (lambda L: L.nvfp4b200_mx_quant(FAKE, 0, None, None, FAKE, None, None, None, 4, 64, 64, None), 1),   # q without s
    (lambda L: L.nvfp4b200_mx_quant(FAKE, 3, None, None, FAKE, FAKE, None, None, 4, 64, 64, None), 1),   # dtype
    (lambda L: L.nvfp4b200_mx_quant(FAKE, 0, None, None, FAKE, FAKE, None, None, 4, 48, 48, None), 2),   # k % 32
    (lambda L: L.nvfp4b200_mx_quant(FAKE, 0, None, None, None, None, FAKE, FAKE, 4, 44, 48, None), 2),   # cols % 8
    (lambda L: L.nvfp4b200_mx_quant(FAKE, 0, None, None, FAKE, FAKE, None, None, 4, 64, 68, None), 2),   # ldx % 8
    (lambda L: L.nvfp4b200_mx_quant(FAKE, 0, None, None, FAKE, FAKE, None, None, 4, 64, 32, None), 2),   # ldx < cols
    (lambda L: L.nvfp4b200_mx_quant(FAKE, 0, None, None, FAKE, FAKE, None, None, -1, 64, 64, None), 2),
    (lambda L: L.nvfp4b200_mx_quant(MIS, 0, None, None, FAKE, FAKE, None, None, 4, 64, 64, None), 3),
    (lambda L: L.nvfp4b200_mx_quant(FAKE, 0, None, MIS, FAKE, FAKE, None, None, 4, 64, 64, None), 3),
    (lambda L: L.nvfp4b200_mx_dequant(FAKE, FAKE, FAKE, 2, 4, 64, None), 1),                             # fp16 out
    (lambda L: L.nvfp4b200_mx_dequant(FAKE, FAKE, FAKE, 0, 4, 48, None), 2),
    (lambda L: L.nvfp4b200_mx_dequant(FAKE, FAKE, MIS, 0, 4, 64, None), 3),
    (lambda L: L.nvfp4b200_mx_gemm(FAKE, FAKE, FAKE, FAKE, None, None, FAKE, 0, 1, 0, 8, 8, 64, 8, None), 1),  # accumulate bf16
    (lambda L: L.nvfp4b200_mx_gemm(FAKE, FAKE, FAKE, FAKE, None, FAKE, FAKE, 1, 0, 0, 8, 8, 64, 8, None), 1),  # residual fp32
    (lambda L: L.nvfp4b200_mx_gemm(FAKE, FAKE, FAKE, FAKE, None, None, FAKE, 0, 0, 0, 8, 12, 64, 16, None), 2),
    (lambda L: _norm(L, _ptrs(FAKE), _ints(0), None, None, _longs(8), 1, kind=1), 1),                    # norm type
    (lambda L: _norm(L, _ptrs(FAKE), _ints(7), None, None, _longs(8), 1), 1),                            # dtype
    (lambda L: _norm(L, _ptrs(FAKE), _ints(0), None, None, _longs(-8), 1), 2),
    (lambda L: _norm(L, _ptrs(None), _ints(0), None, None, _longs(8), 1), 1),
    (lambda L: _norm(L, _ptrs(FAKE + 1), _ints(0), None, None, _longs(8), 1), 3),
    (lambda L: _norm(L, _ptrs(FAKE), _ints(0), None, None, _longs(8), 1, mx=-1.0), 1),
    (lambda L: _norm(L, _ptrs(FAKE), _ints(0), None, None, _longs(8), 1, mx=float("nan")), 1),
    (lambda L: _norm(L, _ptrs(FAKE), _ints(0), None, None, _longs(8), 1, norm=None), 1),                 # no output
    # the same output twice; outputs that overlap; an output over another gradient; a shifted copy onto itself
    (lambda L: _norm(L, _ptrs(FAKE, FAKE), _ints(0, 0), _ptrs(FAKE, FAKE), _ints(0, 0), _longs(8, 8), 2), 1),
    (lambda L: _norm(L, _ptrs(FAKE, FAKE + 512), _ints(0, 0), _ptrs(FAKE + 1024, FAKE + 1038), _ints(0, 0),
                     _longs(8, 8), 2), 1),
    (lambda L: _norm(L, _ptrs(FAKE, FAKE + 512), _ints(0, 0), _ptrs(FAKE + 512, FAKE + 1024), _ints(0, 0),
                     _longs(8, 8), 2), 1),
    (lambda L: _norm(L, _ptrs(FAKE), _ints(0), _ptrs(FAKE + 2), _ints(0), _longs(8), 1), 1),
    (lambda L: _norm(L, _ptrs(FAKE), _ints(1), _ptrs(FAKE), _ints(0), _longs(8), 1), 1),   # in place, other type
    (lambda L: L.nvfp4b200_grad_norm_finish(None, 1, 2, 1.0, 1.0, FAKE, FAKE, None), 1),
    (lambda L: L.nvfp4b200_grad_norm_finish(FAKE, -1, 2, 1.0, 1.0, FAKE, FAKE, None), 2),
    (lambda L: L.nvfp4b200_grad_norm_finish(FAKE + 4, 1, 2, 1.0, 1.0, FAKE, FAKE, None), 3),
    (lambda L: _fwd(L, b=None), 1),
    (lambda L: _fwd(L, n=FAKE), 1),                     # n without inv_y
    (lambda L: _fwd(L, gn=FAKE), 1),                    # gamma_pre without n
    (lambda L: _fwd(L, dt=5), 1),
    (lambda L: _fwd(L, gate=FAKE, g=3), 2),             # rows % groups
    (lambda L: _fwd(L, gate=FAKE), 2),                  # a gate without groups
    (lambda L: _fwd(L, d=16385, ldb=16385, ldx=16385), 2),
    (lambda L: _fwd(L, ldb=63), 2),
    (lambda L: _fwd(L, b=FAKE + 1), 3),
    (lambda L: _fwd(L, dt=1, x=MIS), 3),
    (lambda L: _bwd(L, dy=None), 1),                    # neither gradient
    (lambda L: _bwd(L, dn=FAKE), 1),                    # dn without y
    (lambda L: _bwd(L, gn=FAKE), 1),
    (lambda L: _bwd(L, dgn=FAKE), 1),
    (lambda L: _bwd(L, dgate=FAKE), 1),
    (lambda L: _bwd(L, gate=FAKE, g=3), 2),
    (lambda L: _bwd(L, ld=32), 2),
    (lambda L: _bwd(L, dx=FAKE + 1), 3),
    (lambda L: L.nvfp4b200_sandwich_norm_bwd_ws(4, 64, 3, None), 1),
    (lambda L: L.nvfp4b200_adamw_step_clipped(FAKE, FAKE, 0, FAKE, FAKE, 8, 1e-3, .9, .95, 1e-8, 0., 1., 1., 1.,
                                              MIS, None), 3),
    (lambda L: L.nvfp4b200_adamw_master_step_clipped(FAKE, None, FAKE, 0, FAKE, FAKE, 8, 1., .1, .95, .05, 1e-8, 1e-3,
                                                     1., 1., None, None, None), 1),
])
def test_c_entry_points_refuse(pkg, call, expected):
    assert call(pkg._lib.load()) == expected


def test_torch_binding_shares_the_cpp_runtime(pkg):
    """libtorch throws and formats through the shared libstdc++; a binding with a copy
    of its own crashes when a refusal's message is put together."""
    with open(pkg._build.BINDING_PATH, "rb") as f:
        assert b"libstdc++.so.6" in f.read()


def test_torch_binding_fails_loudly_when_missing(pkg, monkeypatch, tmp_path):
    monkeypatch.setattr(pkg._build, "BINDING_PATH", str(tmp_path / "missing.so"))
    with pytest.raises(pkg.NVFP4Error):
        pkg._bind.load()
