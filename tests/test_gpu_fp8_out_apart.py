"""fp8_linear: an output and a residual that lie in one buffer without sharing an element are taken, whatever
their rows' distances; what shares one is refused."""
import pytest
import torch

import kernel_opt
from test_gpu_fp8_epilogue import extras, small

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("m,k,n", [(1, 272, 64), (5, 272, 333), (300, 4176, 8200)])
def test_halves_of_one_buffer(m, k, n, out):
    ops = small(m, k, n, out)
    _, residual = extras(m, n, out)
    want = kernel_opt.fp8_linear(*ops, out, residual=residual)
    for a, b in ((0, n), (n, 0)):
        both = torch.full((m, 2 * n), 7.0, device="cuda").to(out)
        both[:, b:b + n] = residual
        kernel_opt.fp8_linear(*ops, out=both[:, a:a + n], residual=both[:, b:b + n])
        assert torch.equal(both[:, a:a + n], want) and torch.equal(both[:, b:b + n], residual)


def test_rows_of_other_distances():
    m, n = 4, 64
    ops = small(m, 272, n, torch.bfloat16)
    _, residual = extras(m, n, torch.bfloat16)
    want = kernel_opt.fp8_linear(*ops, residual=residual)
    # rows of 64 at 0, 200, 400, 600 and at 64, 264 (64 + 200), ...; at 64, 164, 264, 364: 164 reaches into 200
    flat = torch.zeros(1000, device="cuda", dtype=torch.bfloat16)
    rows = lambda at, step: flat.as_strided((m, n), (step, 1), at)
    rows(64, 200).copy_(residual)
    kernel_opt.fp8_linear(*ops, out=rows(0, 200), residual=rows(64, 200))
    assert torch.equal(rows(0, 200), want) and torch.equal(rows(64, 200), residual)
    # twice as far apart: 0, 400, 800 (out of 3 rows) between 100, 300, 500
    flat.zero_()
    few = (ops[0][:3], ops[1][:3], *ops[2:])
    at = lambda start, step: flat.as_strided((3, n), (step, 1), start)
    at(100, 200).copy_(residual[:3])
    kernel_opt.fp8_linear(*few, out=at(0, 400), residual=at(100, 200))
    assert torch.equal(at(0, 400), want[:3]) and torch.equal(at(100, 200), residual[:3])
    for out, res in ((rows(0, 200), rows(64, 100)), (rows(0, 200), rows(63, 200)), (rows(0, 64), rows(256 - 1, 64)),
                     (rows(100, 100), rows(36 + 1, 164)), (rows(0, 100), rows(0, 101))):
        with pytest.raises(ValueError, match="lie apart"):
            kernel_opt.fp8_linear(*ops, out=out, residual=res)
