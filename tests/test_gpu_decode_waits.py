"""Bounded waits of the 8-bit product that run out, with the wait-timeout test library (short
limits, and a knob that makes block 0 issue no more tile copies): the kernel returns, sets its
bit of the status word, leaves NaN in what it could not finish and nothing else, and a
following call is clean.  Nothing faults or hangs: every wait gives up after some
milliseconds, and the copies that were issued have landed by then."""
import ctypes

import pytest
import torch

import kernel_opt
from _helpers import WAIT_TEST_LIB

pytestmark = pytest.mark.gpu

BF16, WAIT_BIT = 2, 16
i64, p, c_int = ctypes.c_int64, ctypes.c_void_p, ctypes.c_int


def wait_lib():
    lib = ctypes.CDLL(WAIT_TEST_LIB)
    lib.k1_test_set_knobs.argtypes = [ctypes.c_longlong, ctypes.c_longlong]
    lib.k1_ring_status.argtypes = [ctypes.POINTER(ctypes.c_uint)]
    lib.k1_fp8_linear.argtypes = [p, i64, p, p, i64, p, i64, i64, i64, p, i64, c_int, p]
    lib.k1_last_error.restype = ctypes.c_char_p
    return lib


def status(lib):
    v = ctypes.c_uint(0)
    assert lib.k1_ring_status(ctypes.byref(v)) == 0
    return v.value


def run(lib, xq, xs, wq, ws):
    (m, k), n = xq.shape, wq.shape[0]
    y = torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
    rc = lib.k1_fp8_linear(xq.data_ptr(), k, xs.data_ptr(), wq.data_ptr(), k, ws.data_ptr(), m, k, n,
                           y.data_ptr(), n, BF16, torch.cuda.current_stream().cuda_stream)
    assert rc == 0, lib.k1_last_error()
    torch.cuda.synchronize()
    return y


# few tokens alone, few tokens with K split over a cluster, many tokens (a CTA pair)
@pytest.mark.parametrize("m,k,n", [(8, 512, 64000), (8, 2048, 512), (300, 512, 20000)])
def test_withheld_copies(m, k, n):
    lib = wait_lib()
    g = torch.Generator(device="cuda").manual_seed(m + n)
    xq, xs = kernel_opt.quantize_fp8_rows(torch.randn(m, k, generator=g, device="cuda"))
    wq, ws = kernel_opt.quantize_fp8_blocks(torch.randn(n, k, generator=g, device="cuda"))
    want = kernel_opt.fp8_linear(xq, xs, wq, ws)
    assert status(lib) == 0
    assert lib.k1_test_set_knobs(1, -1) == 0
    try:
        y = run(lib, xq, xs, wq, ws)
        st = status(lib)
    finally:
        assert lib.k1_test_set_knobs(-1, -1) == 0
    assert st & WAIT_BIT, f"status {st}: the wait did not report"
    bad = torch.isnan(y)
    assert bad.any() and not bad.all()
    assert torch.equal(y[~bad], want[~bad])
    assert torch.equal(run(lib, xq, xs, wq, ws), want) and status(lib) == 0
