"""The stream written over x or over the residual (C ABI), in every width of piece: the same values
as into a buffer of its own.  Each element is read and written by one thread, and the kernel reads
with loads that allow for writes; a check of the sources holds it to them."""
import ctypes
import os
import re

import pytest
import torch

from _helpers import CAPI_LIB
from conftest import PKG_ROOT

F32, F16, BF16 = 0, 1, 2
CODE = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}
i64, p, c_int, c_float = ctypes.c_int64, ctypes.c_void_p, ctypes.c_int, ctypes.c_float


def test_the_norms_loads_allow_for_writes():
    text = open(os.path.join(PKG_ROOT, "csrc", "k1_norm.cuh")).read()
    loads = re.findall(r"void load\(const T\* p\) \{([^}]*)\}", text)
    assert len(loads) == 3 and not any("ldg" in body for body in loads), loads


def library():
    lib = ctypes.CDLL(CAPI_LIB)
    lib.k1_last_error.restype = ctypes.c_char_p
    lib.k1_residual_rmsnorm.argtypes = [p, i64, p, i64, p, c_int, c_int, i64, i64, c_float, p, p, p, p]
    lib.k1_residual_rmsnorm_fp8.argtypes = [p, i64, p, i64, p, c_int, c_int, i64, i64, c_float, p, p, p, p]
    return lib


def call(lib, fp8, x, r, w, stream, out, aux):
    n, h = x.shape
    f = lib.k1_residual_rmsnorm_fp8 if fp8 else lib.k1_residual_rmsnorm
    rc = f(x.data_ptr(), h, r.data_ptr(), h, w.data_ptr(), CODE[w.dtype], CODE[x.dtype], n, h, 1e-5, stream.data_ptr(),
           out.data_ptr(), aux.data_ptr(), torch.cuda.current_stream().cuda_stream)
    assert rc == 0, lib.k1_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n,h", [(700, 3584), (900, 1026), (600, 2051), (3, 16384), (1, 64)])
def test_stream_over_an_input(n, h, dtype, fp8):
    lib = library()
    g = torch.Generator(device="cuda").manual_seed(h)
    x, r = (torch.randn(n, h, generator=g, device="cuda").to(dtype) for _ in range(2))
    w = torch.randn(h, generator=g, device="cuda").to(dtype)
    results = []
    for over in ("own", "x", "residual"):
        a, b = x.clone(), r.clone()
        stream = {"own": torch.empty_like(x), "x": a, "residual": b}[over]
        out = torch.empty(n, h, dtype=torch.uint8 if fp8 else dtype, device="cuda")
        aux = torch.empty(n, -(-h // 128) if fp8 else 1, device="cuda")
        call(lib, fp8, a, b, w, stream, out, aux)
        assert torch.equal(a, stream if over == "x" else x) and torch.equal(b, stream if over == "residual" else r)
        results.append((stream.clone(), out, aux))
    assert torch.equal(results[0][0], (x.float() + r.float()).to(dtype))
    for other in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], other))
