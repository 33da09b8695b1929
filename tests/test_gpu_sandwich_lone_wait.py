"""A bounded wait of the sandwich norm's ring that runs out for one thread of a group only (a knob of the
wait-timeout library; the other threads see the rows land): the group's rows from there on are NaN in every
output that is computed from the whole row, what the thread itself writes is NaN, and nothing else changes.
Nothing faults or hangs: every row has been ordered and lands."""
import ctypes

import pytest
import torch

import test_gpu_sandwich_waits as waits
from test_gpu_sandwich_waits import BF16, WAIT_BIT, c_float, c_int, i64, p, status

pytestmark = pytest.mark.gpu


def library():
    lib = waits.wait_lib()
    lib.k1_test_set_lone.argtypes = [ctypes.c_longlong]
    lib.k1_sandwich_rmsnorm_fp8.argtypes = [p, i64, p, i64, p, p, c_int, i64, p, c_int, c_int, i64, i64, c_float, c_float,
                                            c_float, p, p, p, p]
    return lib


def eight_bits(lib, t):
    n, h = t["x"].shape
    st = torch.cuda.current_stream().cuda_stream
    new = lambda *s, d: torch.empty(*s, dtype=d, device="cuda")
    stream, q, scales = new(n, h, d=torch.bfloat16), new(n, h, d=torch.float8_e4m3fn), new(n, -(-h // 128), d=torch.float32)
    ptr = lambda k: t[k].data_ptr()
    rc = lib.k1_sandwich_rmsnorm_fp8(ptr("x"), h, ptr("r"), h, ptr("wp"), None, 0, 0, ptr("w"), BF16, BF16, n, h, 1.0, 1.0,
                                     1e-6, stream.data_ptr(), q.data_ptr(), scales.data_ptr(), st)
    assert rc == 0, lib.k1_last_error()
    torch.cuda.synchronize()
    return {"stream": stream, "q": q.float(), "scales": scales}


@pytest.mark.parametrize("n,h", [(2000, 1024), (3000, 3584), (1500, 8192)])
@pytest.mark.parametrize("row", [0, 1])
def test_one_thread(n, h, row):
    lib = library()
    g = torch.Generator(device="cuda").manual_seed(n)
    r = lambda *s: torch.randn(s, generator=g, device="cuda").bfloat16()
    t = {"x": r(n, h), "r": r(n, h), "wp": r(h), "w": r(h), "gy": r(n, h), "gs": r(n, h), "stream": r(n, h)}
    t["r1"] = t["r2"] = torch.ones(n, device="cuda")
    want, t["r1"], t["r2"] = waits.run(lib, t)
    t["stream"] = want["stream"]
    want, r1, r2 = waits.run(lib, t)
    want.update(r1=r1[:, None], r2=r2[:, None])
    want8 = eight_bits(lib, t)
    assert status(lib) == 0
    assert lib.k1_test_set_lone(row) == 0
    try:
        got, r1, r2 = waits.run(lib, t)
        got.update(r1=r1[:, None], r2=r2[:, None])
        st = status(lib)
        got8 = eight_bits(lib, t)
        st8 = status(lib)
    finally:
        assert lib.k1_test_set_lone(-1) == 0
    assert st & WAIT_BIT and st8 & WAIT_BIT

    def lost_rows(values):
        """Rows of one group of block 0: one per round of the grid, all from the given one on."""
        lost = values.isnan().any(1)
        at = lost.nonzero()[:, 0]
        assert 0 < len(at) < n // 2 and len(set(at.diff().tolist())) <= 1
        assert row > 0 or at[0] == 0
        return lost

    # forward and backward give a group other rows
    for names in (("r2", "stream", "y", "r1"), ("dx", "dr")):
        lost = lost_rows(got[names[0]])
        for k in names:
            assert got[k][lost].isnan().all() and torch.equal(got[k][~lost], want[k][~lost]), k
    # a column of dw takes one product from a row: of rows that the column's own thread saw land
    bad = got["dw"].isnan()
    assert got["dwp"].isnan().all() and bad.any() and torch.equal(got["dw"][~bad], want["dw"][~bad])
    lost = lost_rows(got8["stream"])
    for k in ("stream", "q", "scales"):
        assert got8[k][lost].isnan().all() and torch.equal(got8[k][~lost], want8[k][~lost]), k
    again, _, _ = waits.run(lib, t)
    assert all(torch.equal(again[k], want[k]) for k in again) and status(lib) == 0
