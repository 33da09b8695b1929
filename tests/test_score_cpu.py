"""The entry points of the log-probabilities of lists of tokens reject bad arguments before any
device call (so this runs without a GPU)."""
import ctypes

import pytest
import torch

import kernel_opt
from _helpers import CAPI_LIB

OK, INVALID, DTYPE = 0, 1, 2
BF16 = 2
i64, p, c_int, c_double = ctypes.c_int64, ctypes.c_void_p, ctypes.c_int, ctypes.c_double


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(CAPI_LIB)
    lib.k1_last_error.restype = ctypes.c_char_p
    rows = [p, c_int, i64, i64, i64, i64, i64, c_double]
    lib.k1_token_logprobs.argtypes = rows + [p, i64, p, i64, p, p, p, p, p, p]
    lib.k1_token_logprobs_backward.argtypes = rows + [p, i64, p, p, i64, p, p, p, p, p, p, p, i64, p]
    return lib


def forward(lib, x=1024, d=BF16, n=4, v=1000, inner=4, t=1.0, ids=2048, n_ids=1, lp=4096, k=5, top=8192, tl=8192,
            out=16384):
    return lib.k1_token_logprobs(x, d, n, v, inner, v, 0, t, ids, n_ids, lp, k, top, tl, out, out, None, None)


def backward(lib, x=1024, d=BF16, n=4, v=1000, t=1.0, ids=2048, n_ids=1, g=4096, top=8192, k=5, gt=4096, saved=16384,
             dx=65536, stride=1000):
    return lib.k1_token_logprobs_backward(x, d, n, v, 4, v, 0, t, ids, n_ids, g, top, k, gt, saved, None, saved, None,
                                          None, dx, stride, None)


def test_refuses(lib):
    err = lambda: lib.k1_last_error().decode()
    for call in (forward, backward):
        assert call(lib, d=7) == DTYPE and "bf16, fp16, or fp32" in err()
        assert call(lib, n=-1) == INVALID and "n_rows" in err()
        assert call(lib, n=(1 << 27) + 4) == INVALID and "n_rows" in err()
        for v in (0, -5, 1 << 30):
            assert call(lib, v=v) == INVALID and "vocab" in err()
        for t in (0.0, -1.0, float("nan"), float("inf"), 1e31, 1e-31):
            assert call(lib, t=t) == INVALID and "temperature" in err()
        for n_ids in (-1, 1025):
            assert call(lib, n_ids=n_ids) == INVALID and "tokens per row" in err()
        for k in (-1, 129):
            assert call(lib, k=k) == INVALID and "k must be" in err()
        assert call(lib, v=4, k=5) == INVALID and "k must be" in err()
        assert call(lib, x=0) == INVALID and "NULL" in err()
        assert call(lib, x=1025) == INVALID and "aligned" in err()
        assert call(lib, n=0, x=0) == OK
    assert forward(lib, inner=3) == INVALID and "inner_rows" in err()
    assert forward(lib, ids=0) == INVALID and "NULL" in err()
    assert forward(lib, top=0) == INVALID and "NULL" in err()
    assert forward(lib, out=0) == INVALID and "NULL" in err()
    assert backward(lib, ids=0) == INVALID and "NULL" in err()
    assert backward(lib, saved=0) == INVALID and "NULL" in err()
    assert backward(lib, stride=999) == INVALID and "d_stride" in err()
    assert backward(lib, dx=1024) == INVALID and "d_logits" in err()


def test_cpu_tensors():
    x = torch.zeros(2, 8)
    with pytest.raises(ValueError, match="CUDA"):
        kernel_opt.fused_top_logprobs(x, None, 2)
    with pytest.raises(ValueError, match="CUDA"):
        kernel_opt.fused_token_logprobs(x, torch.zeros(2, 1, dtype=torch.int64))
