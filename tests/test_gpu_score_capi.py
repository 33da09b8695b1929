"""The C ABI of the lists' gradient in forms that the torch binding does not use: gradient rows farther apart
than the vocabulary, no lse_rest, and no gradient for some outputs."""
import ctypes

import pytest
import torch

import kernel_opt
from _helpers import CAPI_LIB
from test_gpu_score import DTYPES, check_gradient, logits_of

i64, p, c_int, c_double = ctypes.c_int64, ctypes.c_void_p, ctypes.c_int, ctypes.c_double
CODE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def library():
    lib = ctypes.CDLL(CAPI_LIB)
    lib.k1_last_error.restype = ctypes.c_char_p
    lib.k1_token_logprobs_backward.argtypes = [p, c_int, i64, i64, i64, i64, i64, c_double, p, i64, p, p, i64, p, p, p, p,
                                               p, p, p, i64, p]
    return lib


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("n,v,wide", [(1, 1000, 0), (5, 1000, 8), (5, 1003, 13), (400, 50257, 7)])
def test_wide_gradient_rows_without_rest(dtype, n, v, wide):
    # at temperature 1 an lse of about 15 errs by 2^-21 where its rest is left out: inside the 2e-5
    lib = library()
    x = logits_of(n, v, dtype)
    ids = torch.randint(0, v, (n, 6), device="cuda")
    lp, entropy, lse = kernel_opt.fused_token_logprobs(x, ids)
    g, ge = torch.randn(n, 6, device="cuda"), torch.randn(n, device="cuda")
    buf = torch.full((n, v + wide), 7.0, device="cuda").to(dtype)
    for entropy_too in (True, False):
        buf.fill_(7.0)
        rc = lib.k1_token_logprobs_backward(x.data_ptr(), CODE[dtype], n, v, n, v, 0, 1.0, ids.data_ptr(), 6, g.data_ptr(), None,
                                            0, None, lse.data_ptr(), None, entropy.data_ptr(),
                                            ge.data_ptr() if entropy_too else None, None, buf.data_ptr(), v + wide,
                                            torch.cuda.current_stream().cuda_stream)
        assert rc == 0, lib.k1_last_error()
        assert (buf[:, v:] == 7).all()
        check_gradient(x, buf[:, :v], ids, g, ge if entropy_too else None, None, 1.0)
