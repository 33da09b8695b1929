"""The bounded waits of the many-token kernel's CTA pair, as test_gpu_decode_waits has them for the
few-token kernel: block 0 of a pair withholds its tile copies, the pair's waits give up after some
milliseconds, what it could not finish is NaN, the other pairs' tiles are right, and a following
call is clean.  Nothing faults or hangs."""
import pytest
import torch

import kernel_opt
from _linear import MANY, kernel_of
from test_gpu_decode_waits import WAIT_BIT, run, status, wait_lib

pytestmark = pytest.mark.gpu

# one tile per pair; several tiles per pair
SHAPES = [(300, 512, 8192), (600, 2048, 16384)]


@pytest.mark.parametrize("withhold", [0, 1, 3])
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_withheld_copies(m, k, n, withhold):
    assert kernel_of(m, k, n, torch.cuda.get_device_properties(0).multi_processor_count) == MANY
    lib = wait_lib()
    g = torch.Generator(device="cuda").manual_seed(m + n)
    xq, xs = kernel_opt.quantize_fp8_rows(torch.randn(m, k, generator=g, device="cuda"))
    wq, ws = kernel_opt.quantize_fp8_blocks(torch.randn(n, k, generator=g, device="cuda"))
    want = kernel_opt.fp8_linear(xq, xs, wq, ws)
    assert torch.equal(run(lib, xq, xs, wq, ws), want) and status(lib) == 0
    assert lib.k1_test_set_knobs(withhold, -1) == 0
    try:
        y = run(lib, xq, xs, wq, ws)
        st = status(lib)
    finally:
        assert lib.k1_test_set_knobs(-1, -1) == 0
    assert st & WAIT_BIT, f"status {st}: the wait did not report"
    bad = torch.isnan(y)
    assert bad[:256, :256].all() and not bad.all()   # the pair's first tile
    assert torch.equal(y[~bad], want[~bad])
    assert torch.equal(run(lib, xq, xs, wq, ws), want) and status(lib) == 0
