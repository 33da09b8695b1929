"""The C ABI of the norms around a block's end and of the 8-bit product's epilogue rejects bad arguments
before any device call (so this runs without a GPU)."""
import ctypes

import pytest

from _helpers import CAPI_LIB

OK, INVALID, DTYPE = 0, 1, 2
F32, F16, BF16 = 0, 1, 2
i64, p, c_int, c_float = ctypes.c_int64, ctypes.c_void_p, ctypes.c_int, ctypes.c_float


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(CAPI_LIB)
    lib.k1_last_error.restype = ctypes.c_char_p
    ins = [p, i64, p, i64, p, p, c_int, i64, p, c_int, c_int, i64, i64, c_float, c_float, c_float]
    lib.k1_sandwich_rmsnorm.argtypes = ins + [p, p, p, p, p]
    lib.k1_sandwich_rmsnorm_fp8.argtypes = ins + [p, p, p, p]
    lib.k1_sandwich_rmsnorm_backward.argtypes = [p, i64, p, i64, p, i64, p, i64, p, p, c_int, i64, p, c_int, c_int, p, p,
                                                 i64, i64, c_float, c_float, p, p, p, p, p, p, ctypes.c_size_t, p]
    lib.k1_sandwich_rmsnorm_workspace_bytes.argtypes = [i64, i64, c_int]
    lib.k1_sandwich_rmsnorm_workspace_bytes.restype = ctypes.c_size_t
    lib.k1_fp8_linear_epilogue.argtypes = [p, i64, p, p, i64, p, i64, i64, i64, p, c_int, c_int, p, i64, p, i64, c_int, p]
    return lib


def forward(lib, x=1024, xs=64, r=2048, rs=64, wp=4096, gate=8192, kind=1, gstride=64, w=4096, wd=BF16, d=BF16, n=4, h=64,
            bs=1.0, rscale=1.0, eps=1e-6, s=16384, y=32768):
    return lib.k1_sandwich_rmsnorm(x, xs, r, rs, wp, gate, kind, gstride, w, wd, d, n, h, bs, rscale, eps, s, y, None, None,
                                   None)


def forward8(lib, x=1024, xs=64, r=2048, rs=64, wp=4096, gate=8192, kind=1, gstride=64, w=4096, wd=BF16, d=BF16, n=4, h=64,
             bs=1.0, rscale=1.0, eps=1e-6, s=16384, y=32768, scales=65536):
    return lib.k1_sandwich_rmsnorm_fp8(x, xs, r, rs, wp, gate, kind, gstride, w, wd, d, n, h, bs, rscale, eps, s, y, scales,
                                       None)


def backward(lib, x=1024, xs=64, wp=4096, gate=8192, kind=1, gstride=64, w=4096, wd=BF16, d=BF16, n=4, h=64, bs=1.0,
             rscale=1.0, gy=1024, gys=64, gs=1024, gss=64, s=1024, ss=64, saved=4096, dx=2048, dr=2048, dwp=2048, dg=2048,
             dw=2048, ws=0, size=0):
    return lib.k1_sandwich_rmsnorm_backward(gy, gys, gs, gss, s, ss, x, xs, wp, gate, kind, gstride, w, wd, d, saved, saved,
                                            n, h, bs, rscale, dx, dr, dwp, dg, dw, ws, size, None)


def test_norms_refuse(lib):
    err = lambda: lib.k1_last_error().decode()
    nan, inf = float("nan"), float("inf")
    for call in (forward, forward8, backward):
        assert call(lib, d=7) == DTYPE and "bf16, fp16, or fp32" in err()
        assert call(lib, wd=F16) == DTYPE and "weight" in err()
        assert call(lib, n=-1) == INVALID and "n_rows" in err()
        for h in (0, 16385):
            assert call(lib, h=h) == INVALID and "hidden" in err()
        for kind in (-1, 4):
            assert call(lib, kind=kind) == INVALID and "gate_kind" in err()
        for bad in (nan, inf, -inf):
            assert call(lib, bs=bad) == INVALID and "finite" in err()
            assert call(lib, rscale=bad) == INVALID and "finite" in err()
        for name in ("x", "wp", "w", "gate", "s"):
            assert call(lib, **{name: 0}) == INVALID and "NULL" in err(), name
        for name in ("x", "wp", "w", "gate", "s"):
            assert call(lib, **{name: 1025}) == INVALID and "aligned" in err(), name
        assert call(lib, xs=-1) == INVALID and "strides" in err()
        assert call(lib, kind=3, gstride=-1) == INVALID and "strides" in err()
    for call in (forward, forward8):
        for eps in (0.0, -1.0, nan, inf):
            assert call(lib, eps=eps) == INVALID and "eps" in err()
        assert call(lib, r=0) == INVALID and "NULL" in err()
        assert call(lib, r=2049) == INVALID and "aligned" in err()
        assert call(lib, rs=-64) == INVALID and "strides" in err()
        assert call(lib, y=0) == INVALID and "NULL" in err()
        assert call(lib, n=0, x=0, r=0, s=0, y=0) == OK
    assert forward(lib, y=32769) == INVALID and "aligned" in err()
    assert forward8(lib, scales=0) == INVALID and "NULL" in err()
    assert backward(lib, saved=0) == INVALID and "NULL" in err()
    for name in ("gy", "gs", "dx", "dr", "dwp", "dw", "dg"):
        assert backward(lib, **{name: 2049}) == INVALID and "aligned" in err(), name
    for name in ("gys", "gss", "ss"):
        assert backward(lib, **{name: -1}) == INVALID and "strides" in err(), name
    # nothing wanted: nothing done
    assert backward(lib, dx=0, dr=0, dwp=0, dg=0, dw=0) == OK
    assert lib.k1_sandwich_rmsnorm_workspace_bytes(-1, 64, 0) == 0
    assert lib.k1_sandwich_rmsnorm_workspace_bytes(4, 0, 0) == 0
    assert lib.k1_sandwich_rmsnorm_workspace_bytes(4, 16385, 0) == 0
    assert lib.k1_sandwich_rmsnorm_workspace_bytes(4, 64, -1) == 0


def product(lib, x=1024, xs=256, xsc=2048, w=4096, ws=256, wsc=8192, m=4, k=256, n=100, bias=16384, bd=BF16, act=1,
            res=32768, rs=100, y=65536, ys=100, out=BF16):
    return lib.k1_fp8_linear_epilogue(x, xs, xsc, w, ws, wsc, m, k, n, bias, bd, act, res, rs, y, ys, out, None)


def test_product_refuses(lib):
    err = lambda: lib.k1_last_error().decode()
    assert product(lib, out=7) == DTYPE and "output" in err()
    for act in (-1, 5):
        assert product(lib, act=act) == INVALID and "activation" in err()
    assert product(lib, m=-1) == INVALID and product(lib, n=-1) == INVALID
    for k in (0, 8, 100, 32784):
        assert product(lib, k=k) == INVALID and "inner" in err()
    for name in ("x", "xsc", "w", "wsc", "y"):
        assert product(lib, **{name: 0}) == INVALID and "NULL" in err(), name
    assert product(lib, ys=99) == INVALID and "y_stride" in err()
    assert product(lib, bd=F16) == DTYPE and "bias" in err()
    assert product(lib, rs=99) == INVALID and "residual_stride" in err()
    for name in ("bias", "res", "y"):
        assert product(lib, **{name: 16385}) == INVALID and "aligned" in err(), name
    assert product(lib, bias=16386, bd=F32) == INVALID and "aligned" in err()
    assert product(lib, m=0, x=0, y=0, res=0) == OK
