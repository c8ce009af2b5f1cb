"""The microscaled and expert entry points of the C ABI: sizes and refusals, without a device; and the oracle the GPU tests use."""
import ctypes

import numpy as np
import pytest

from apsi_b200 import _lib, build
from oracle import microscale as ora

MX, NV = _lib.FMT_MXFP4, _lib.FMT_NVFP4


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def test_constants_match_the_header():
    text = open(build.ROOT + "/include/apsi_lowbit.h").read()
    for name, val in (("LB_FMT_MXFP4", MX), ("LB_FMT_NVFP4", NV), ("LB_MX_MAX_GROUPS", _lib.MX_MAX_GROUPS),
                      ("LB_MX_PARTIALS", _lib.MX_PARTIALS), ("LB_DEVERR_BAD_INDEX", _lib.DEVERR_BAD_INDEX)):
        assert f"#define {name} {val}" in text


def test_sizes(lib):
    assert [lib.lb_mx_row_bytes(k) for k in (0, 1, 32, 33, 4096)] == [-1, 16, 16, 32, 2048]
    assert lib.lb_mx_scale_bytes(MX, 128, 256, 0, 0) == 1024 and lib.lb_mx_scale_bytes(NV, 128, 256, 0, 0) == 2048
    assert lib.lb_mx_scale_bytes(MX, 129, 257, 0, 0) == 2 * 2 * 1024
    assert lib.lb_mx_scale_bytes(MX, 6, 32, 3, 2) == 3 * 1024                 # a row block of each matrix
    assert lib.lb_mx_scale_bytes(MX, 300, 32, 5, 0) == (2 + 5) * 1024         # as many as any five groups of 300 rows need
    assert lib.lb_mx_scale_bytes(MX, 3, 32, 5, 0) == 3 * 1024
    assert lib.lb_mx_scale_bytes(9, 3, 32, 0, 0) == -1 and lib.lb_mx_scale_bytes(MX, 3, 0, 0, 0) == -1
    n = ctypes.c_size_t(0)
    assert lib.lb_moe_route_workspace_size(65, 8, ctypes.byref(n)) == 0 and n.value == 2 * 8 * 4
    assert lib.lb_moe_route_workspace_size(64, 8, ctypes.byref(n)) == 0 and n.value == 0
    from apsi_b200 import microscale
    for fmt, f in _lib.MICROSCALED_FMT.items():
        for R, K, G, per in ((0, 5, 0, 0), (1, 1, 0, 0), (300, 1000, 0, 0), (300, 1000, 7, 0), (3, 64, 7, 0), (12, 256, 4, 3)):
            assert microscale._scale_bytes(fmt, R, K, G, per) == lib.lb_mx_scale_bytes(f, R, K, G, per)
            assert microscale._row_bytes(K) == lib.lb_mx_row_bytes(K)


def test_refusals_before_a_device_is_touched(lib):
    p, odd, null = ctypes.c_void_p(1 << 20), ctypes.c_void_p((1 << 20) + 8), ctypes.c_void_p(0)
    E, A = _lib.LB_E_ARG, _lib.LB_E_ALIGN

    def quant(fmt=MX, x=p, dt=1, Rin=4, K=64, ldx=64, rows=null, R=4, off=null, G=0, per=0, t=null, auto=null, c=p, s=p):
        return lib.lb_mx_quant(fmt, x, dt, Rin, K, ldx, rows, R, off, G, per, t, auto, c, s, null)
    assert quant(fmt=9) == E and quant(dt=3) == E and quant(K=0) == E and quant(ldx=63) == E and quant(R=3) == E
    assert quant(G=1025, off=p) == E and quant(G=2) == E and quant(G=3, per=2) == E and quant(per=2) == E and quant(fmt=NV) == E
    assert quant(c=null) == E and quant(x=null) == E and quant(s=odd) == A and quant(x=ctypes.c_void_p((1 << 20) + 1)) == A
    assert quant(Rin=0, R=0) == 0                                              # nothing to do

    def dequant(fmt=MX, c=p, s=p, R=4, K=64, out=p, dt=0, ldo=64):
        return lib.lb_mx_dequant(fmt, c, s, null, R, K, null, 0, 0, out, dt, ldo, null)
    assert dequant(fmt=2) == E and dequant(dt=5) == E and dequant(ldo=63) == E and dequant(out=null) == E and dequant(c=odd) == A
    assert lib.lb_mx_scales(MX, p, 1, 1, 4, 64, p, 1, null) == E               # two blocks a row
    assert lib.lb_mx_scales(MX, p, 2, 1, 4, 64, odd, 1, null) == A

    def linear(fmt=MX, xc=p, xs=p, M=4, K=64, wc=p, ws=p, N=8, bias=null, y=p, ldy=8):
        return lib.lb_mx_linear(fmt, xc, xs, null, M, K, wc, ws, null, N, bias, 0, y, ldy, null)
    assert linear(fmt=9) == E and linear(N=0) == E and linear(ldy=7) == E and linear(y=null) == E and linear(ws=null) == E
    assert linear(xc=odd) == A and linear(ws=odd) == A and linear(y=ctypes.c_void_p((1 << 20) + 1)) == A and linear(M=0) == 0

    def grouped(G=2, off=p, N=8):
        return lib.lb_mx_linear_grouped(MX, p, p, null, 4, 64, off, G, p, p, null, N, null, 0, p, 8, null)
    assert grouped(G=0) == E and grouped(off=null) == E and grouped(G=1025) == E and grouped(N=9) == E
    assert grouped(off=ctypes.c_void_p((1 << 20) + 2)) == A

    def route(dt=0, T=100, E_=8, ld=8, k=2, w=p, off=p, ws=p, n=1 << 10):
        return lib.lb_moe_route(p, dt, T, E_, ld, k, 1, w, p, off, p, p, ws, n, null)
    assert route(dt=4) == E and route(E_=0) == E and route(E_=1025, ld=1025) == E and route(ld=7) == E and route(k=0) == E
    assert route(k=9) == E and route(w=null) == E and route(off=null) == E and route(ws=null) == _lib.LB_E_WORKSPACE
    assert route(n=63) == _lib.LB_E_WORKSPACE

    def combine(z=p, rows=8, ldz=16, w=p, s=p, T=4, k=2, H=16, y=p, ldy=16):
        return lib.lb_moe_combine(z, rows, ldz, w, s, T, k, H, 0, y, ldy, null)
    assert combine(H=0) == E and combine(ldz=15) == E and combine(ldy=15) == E and combine(k=0) == E and combine(z=null) == E
    assert combine(w=ctypes.c_void_p((1 << 20) + 2)) == A and combine(T=0) == 0


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_oracle_properties(fmt):
    """Values on the grid stay; any other is rounded to a nearest one of its block; packing and unpacking agree."""
    g = np.random.default_rng(1)
    x = g.standard_normal((20, 96)) * np.exp(2 * g.standard_normal((20, 1)))
    x = x.astype(np.float32)
    code, byte, val = ora.quantize(x, fmt, 0.5)
    packed = code[:, 0::2] | (code[:, 1::2] << 4)
    assert np.array_equal(ora.values(packed, byte, 96, fmt, 0.5), val)
    again = ora.quantize(val, fmt, 0.5)[2]
    if fmt == "mxfp4":                       # the largest value of a block keeps its binade, so the scale stays
        assert np.array_equal(again, val)
    d = np.repeat(2.0 ** (byte - 127.0) if fmt == "mxfp4" else ora.E4M3[byte] * 0.5, ora.BLOCK[fmt], 1)
    grid = np.concatenate([-ora.GRID[::-1], ora.GRID])
    best = np.abs(np.clip(x / d, -6, 6)[..., None] - grid).min(-1)
    assert np.allclose(np.abs(np.clip(x / d, -6, 6) - val / d), best, rtol=0, atol=1e-12)


def test_oracle_routing():
    w, chosen, offsets, rows, slots = ora.route(np.array([[1.0, 3, 3, 0], [5, -np.inf, np.nan, 4]]), 2, True)
    assert chosen.tolist() == [[1, 2], [0, 3]] and offsets.tolist() == [0, 1, 2, 3, 4]
    assert rows.tolist() == [1, 0, 0, 1] and slots.tolist() == [[1, 2], [0, 3]]
    assert np.allclose(w, [[0.5, 0.5], [1 / (1 + np.exp(-1)), 1 / (1 + np.exp(1))]])
