"""Bounded waits of the sandwich norm's ring kernels that run out, with the wait-timeout test library
(short limits, and a knob that makes block 0 order no more rows): the kernels return, set their bit of
the status word, leave NaN in the rows that they could not finish and in the sums that hold them, and a
following call is clean.  Nothing faults or hangs: every wait gives up after some milliseconds, and the
copies that were ordered have landed by then."""
import ctypes

import pytest
import torch

import kernel_opt
from _helpers import WAIT_TEST_LIB

pytestmark = pytest.mark.gpu

BF16, WAIT_BIT = 2, 1
i64, p, c_int, c_float = ctypes.c_int64, ctypes.c_void_p, ctypes.c_int, ctypes.c_float


def wait_lib():
    lib = ctypes.CDLL(WAIT_TEST_LIB)
    lib.k1_test_set_knobs.argtypes = [ctypes.c_longlong, ctypes.c_longlong]
    lib.k1_ring_status.argtypes = [ctypes.POINTER(ctypes.c_uint)]
    lib.k1_sandwich_rmsnorm.argtypes = [p, i64, p, i64, p, p, c_int, i64, p, c_int, c_int, i64, i64, c_float, c_float,
                                        c_float, p, p, p, p, p]
    lib.k1_sandwich_rmsnorm_backward.argtypes = [p, i64, p, i64, p, i64, p, i64, p, p, c_int, i64, p, c_int, c_int, p, p,
                                                 i64, i64, c_float, c_float, p, p, p, p, p, p, ctypes.c_size_t, p]
    lib.k1_sandwich_rmsnorm_workspace_bytes.argtypes = [i64, i64, c_int]
    lib.k1_sandwich_rmsnorm_workspace_bytes.restype = ctypes.c_size_t
    lib.k1_last_error.restype = ctypes.c_char_p
    return lib


def status(lib):
    v = ctypes.c_uint(0)
    assert lib.k1_ring_status(ctypes.byref(v)) == 0
    return v.value


def run(lib, t):
    n, h = t["x"].shape
    st = torch.cuda.current_stream().cuda_stream
    new = lambda *s, d=torch.bfloat16: torch.empty(*s, dtype=d, device="cuda")
    out = {"stream": new(n, h), "y": new(n, h), "dx": new(n, h), "dr": new(n, h), "dwp": new(h), "dw": new(h)}
    r1, r2 = new(n, d=torch.float32), new(n, d=torch.float32)
    ptr = lambda k: t[k].data_ptr()
    rc = lib.k1_sandwich_rmsnorm(ptr("x"), h, ptr("r"), h, ptr("wp"), None, 0, 0, ptr("w"), BF16, BF16, n, h, 1.0, 1.0,
                                 1e-6, out["stream"].data_ptr(), out["y"].data_ptr(), r1.data_ptr(), r2.data_ptr(), st)
    assert rc == 0, lib.k1_last_error()
    size = lib.k1_sandwich_rmsnorm_workspace_bytes(n, h, 0)
    ws = new(size, d=torch.uint8)
    # from the clean forward's outputs, so that only this kernel's waits count
    rc = lib.k1_sandwich_rmsnorm_backward(ptr("gy"), h, ptr("gs"), h, ptr("stream"), h, ptr("x"), h, ptr("wp"), None, 0, 0,
                                          ptr("w"), BF16, BF16, ptr("r1"), ptr("r2"), n, h, 1.0, 1.0, out["dx"].data_ptr(),
                                          out["dr"].data_ptr(), out["dwp"].data_ptr(), None, out["dw"].data_ptr(),
                                          ws.data_ptr(), size, st)
    assert rc == 0, lib.k1_last_error()
    torch.cuda.synchronize()
    return out, r1, r2


@pytest.mark.parametrize("n,h", [(2000, 1024), (3000, 3584), (1500, 8192)])
@pytest.mark.parametrize("withhold", [0, 1])
def test_withheld_rows(n, h, withhold):
    lib = wait_lib()
    g = torch.Generator(device="cuda").manual_seed(n)
    r = lambda *s: torch.randn(s, generator=g, device="cuda").bfloat16()
    t = {"x": r(n, h), "r": r(n, h), "wp": r(h), "w": r(h), "gy": r(n, h), "gs": r(n, h), "stream": r(n, h)}
    t["r1"] = t["r2"] = torch.ones(n, device="cuda")
    want, t["r1"], t["r2"] = run(lib, t)
    t["stream"] = want["stream"]
    want, _, _ = run(lib, t)
    assert status(lib) == 0
    assert lib.k1_test_set_knobs(withhold, -1) == 0
    try:
        out, _, _ = run(lib, t)
        st = status(lib)
    finally:
        assert lib.k1_test_set_knobs(-1, -1) == 0
    assert st & WAIT_BIT, f"status {st}: the wait did not report"
    for k in ("stream", "y", "dx", "dr"):
        bad = out[k].isnan()
        assert torch.equal(bad.any(1), bad.all(1)) and bad.any() and not bad.all(), k
        assert torch.equal(out[k][~bad], want[k][~bad]), k
    assert out["dw"].isnan().all() and out["dwp"].isnan().all()
    again, _, _ = run(lib, t)
    assert all(torch.equal(again[k], want[k]) for k in want) and status(lib) == 0
