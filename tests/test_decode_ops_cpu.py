"""The decoding-step entry points of the C ABI reject bad arguments before any device call
(so this runs without a GPU), and the package exports the operators."""
import ctypes

import pytest
import torch

import kernel_opt
from _helpers import CAPI_LIB

OK, INVALID, DTYPE = 0, 1, 2
F32, F16, BF16 = 0, 1, 2
i64, p, c_int, c_float, c_double = (ctypes.c_int64, ctypes.c_void_p, ctypes.c_int, ctypes.c_float,
                                    ctypes.c_double)


class Sampling(ctypes.Structure):
    _fields_ = [("temperature_rows", p), ("top_k_rows", p), ("top_p_rows", p), ("min_p_rows", p),
                ("temperature", c_double), ("top_k", c_int), ("top_p", c_float), ("min_p", c_float)]


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(CAPI_LIB)
    lib.k1_last_error.restype = ctypes.c_char_p
    lib.k1_residual_rmsnorm.argtypes = [p, i64, p, i64, p, c_int, c_int, i64, i64, c_float, p, p, p, p]
    lib.k1_residual_rmsnorm_fp8.argtypes = [p, i64, p, i64, p, c_int, c_int, i64, i64, c_float, p, p, p, p]
    lib.k1_quantize_fp8_rows.argtypes = [p, i64, c_int, i64, i64, p, p, p]
    lib.k1_quantize_fp8_blocks.argtypes = [p, i64, c_int, i64, i64, p, p, p]
    lib.k1_residual_rmsnorm_backward.argtypes = [p, i64, p, i64, p, i64, p, p, c_int, c_int, i64, i64, p, p, p,
                                                 ctypes.c_size_t, p]
    lib.k1_fp8_linear.argtypes = [p, i64, p, p, i64, p, i64, i64, i64, p, i64, c_int, p]
    lib.k1_sample_tokens.argtypes = [p, c_int, i64, i64, i64, p, ctypes.POINTER(Sampling), p, p, p, p]
    return lib


def err(lib):
    return lib.k1_last_error().decode()


def norm(lib, x=1024, r=2048, w=4096, wd=BF16, d=BF16, n=4, h=64, eps=1e-6, s=8192, y=16384):
    return lib.k1_residual_rmsnorm(x, h, r, h, w, wd, d, n, h, eps, s, y, None, None)


def test_norm_refuses(lib):
    assert norm(lib, d=7, wd=7) == DTYPE and "bf16, fp16, or fp32" in err(lib)
    assert norm(lib, wd=F16) == DTYPE and "weight" in err(lib)
    assert norm(lib, n=-1) == INVALID
    assert norm(lib, h=0) == INVALID and "hidden" in err(lib)
    assert norm(lib, h=16385) == INVALID
    for eps in (0.0, -1.0, float("nan"), float("inf")):
        assert norm(lib, eps=eps) == INVALID and "eps" in err(lib)
    assert norm(lib, x=0) == INVALID and "NULL" in err(lib)
    assert norm(lib, s=0) == INVALID            # a residual needs somewhere to store the stream
    assert norm(lib, x=1025) == INVALID and "aligned" in err(lib)
    assert norm(lib, n=0, x=0, r=0, w=0, s=0, y=0) == OK


def test_norm_backward_and_quantisers_refuse(lib):
    b = lib.k1_residual_rmsnorm_backward
    assert b(1024, 64, None, 0, 0, 64, 2048, 4096, BF16, BF16, 4, 64, 8192, None, None, 0, None) == INVALID
    assert b(1024, 64, None, 0, 2048, 64, 2048, 4096, BF16, 9, 4, 64, 8192, None, None, 0, None) == DTYPE
    q = lib.k1_quantize_fp8_rows
    assert q(1024, 64, BF16, 4, 64, 2048, None, None) == INVALID and "NULL" in err(lib)
    assert q(1024, 64, 5, 4, 64, 2048, 4096, None) == DTYPE
    assert q(0, 64, BF16, 0, 64, 0, 0, None) == OK
    w = lib.k1_quantize_fp8_blocks
    assert w(1024, 64, BF16, 4, 0, 2048, 4096, None) == INVALID
    assert w(1025, 64, BF16, 4, 64, 2048, 4096, None) == INVALID and "aligned" in err(lib)


def linear(lib, x=1024, ldx=256, xs=2048, w=4096, ldw=256, ws=8192, m=4, k=256, n=100, y=16384, ldy=100,
           d=BF16):
    return lib.k1_fp8_linear(x, ldx, xs, w, ldw, ws, m, k, n, y, ldy, d, None)


def test_linear_refuses(lib):
    assert linear(lib, d=3) == DTYPE
    assert linear(lib, m=-1) == INVALID
    for k in (0, 8, 250, 32784):
        assert linear(lib, k=k, ldx=32784, ldw=32784) == INVALID and "inner" in err(lib)
    assert linear(lib, x=1032) == INVALID and "16 bytes" in err(lib)
    assert linear(lib, ldw=264) == INVALID
    assert linear(lib, ldx=128) == INVALID      # rows that overlap
    assert linear(lib, ldy=99) == INVALID and "y_stride" in err(lib)
    assert linear(lib, xs=0) == INVALID and "NULL" in err(lib)
    assert linear(lib, m=0, x=0) == OK and linear(lib, n=0, y=0) == OK


def sample(lib, logits=1024, d=BF16, n=4, v=100, u=2048, out=4096, **kw):
    s = Sampling(temperature=1.0, top_p=1.0)
    for k, val in kw.items():
        setattr(s, k, val)
    return lib.k1_sample_tokens(logits, d, n, v, v, u, ctypes.byref(s), out, out, out, None)


def test_sampling_refuses(lib):
    assert sample(lib, d=4) == DTYPE
    assert sample(lib, v=0) == INVALID and "vocab" in err(lib)
    assert sample(lib, n=-1) == INVALID
    for t in (-1.0, float("nan"), float("inf")):
        assert sample(lib, temperature=t) == INVALID and "temperature" in err(lib)
    for q in (-0.1, 1.1, float("nan")):
        assert sample(lib, min_p=q) == INVALID and "min_p" in err(lib)
    assert sample(lib, top_p=-0.5) == INVALID and "top_p" in err(lib)
    assert sample(lib, u=0) == INVALID and "NULL" in err(lib)
    assert sample(lib, logits=1025) == INVALID and "aligned" in err(lib)
    assert lib.k1_sample_tokens(1024, BF16, 4, 100, 100, 2048, None, 4096, 4096, 4096, None) == INVALID
    assert sample(lib, n=0, logits=0, u=0, out=0) == OK


def test_public_surface_and_cpu_tensors():
    x = torch.zeros(2, 8)
    with pytest.raises(ValueError, match="CUDA"):
        kernel_opt.fused_residual_rmsnorm(x, x, torch.ones(8))
    with pytest.raises(ValueError, match="CUDA"):
        kernel_opt.fused_residual_rmsnorm_fp8(x, None, torch.ones(8))
    with pytest.raises(ValueError, match="CUDA"):
        kernel_opt.quantize_fp8_rows(x)
    with pytest.raises(ValueError, match="CUDA"):
        kernel_opt.quantize_fp8_blocks(x)
    with pytest.raises(ValueError, match="CUDA"):
        kernel_opt.sample_tokens(x, torch.zeros(2))
    q = x.to(torch.float8_e4m3fn)
    with pytest.raises(ValueError, match="CUDA"):
        kernel_opt.fp8_linear(q, x[:, :1], q, x[:1, :1])
    assert callable(kernel_opt.RolloutHead)
