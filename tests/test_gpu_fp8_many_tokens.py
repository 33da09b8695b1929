"""The many-token kernel of the 8-bit product (a pair of SMs per tile) against the same sum in 64
bits, with the tolerance derived in test_gpu_fp8_linear: shapes that do take it (asserted on the
CPU for a B200, and here for the device at hand)."""
import pytest
import torch

import kernel_opt
from _linear import MANY, kernel_of
from test_gpu_fp8_linear import check, operands

pytestmark = pytest.mark.gpu

SHAPES = [
    (300, 4176, 8200),    # 33 blocks of K (a second chunk of scales), the last one ragged; columns past the last tile
    (300, 4176, 8201),    # rows that start anywhere
    (300, 8208, 8200),    # a third chunk of scales
    (257, 3584, 8192),    # one token in the last tile
    (600, 1040, 16640),   # several tiles per pair
    (2300, 2064, 4100),   # a second group of token tiles, several tiles per pair
    (2048, 3584, 4097),
]
LAYOUT = (300, 4176, 8201)


@pytest.fixture(autouse=True)
def takes_the_many_token_kernel():
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert all(kernel_of(*s, sms) == MANY for s in SHAPES + [LAYOUT])


def scaled(ops, out):
    # inside fp16's range
    return (ops[0], ops[1] * 0.02, ops[2], ops[3] * 0.02) if out == torch.float16 else ops


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_product(m, k, n, out):
    ops = scaled(operands(m, k, n), out)
    y = kernel_opt.fp8_linear(*ops, out)
    assert y.shape == (m, n) and y.dtype == out
    check(y, *ops)
    assert torch.equal(y, kernel_opt.fp8_linear(*ops, out))


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
def test_layouts(out):
    """Operands inside wider rows, outputs inside wider rows at any start; nothing else is written."""
    m, k, n = LAYOUT
    xq, xs, wq, ws = operands(m, k, n)
    want = kernel_opt.fp8_linear(xq, xs, wq, ws, out)
    xw = torch.zeros(m, k + 48, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    ww = torch.zeros(n, k + 32, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    xw.view(torch.uint8)[:, 16:16 + k] = xq.view(torch.uint8)
    ww.view(torch.uint8)[:, :k] = wq.view(torch.uint8)
    for off, pitch in ((0, n + 7), (1, n + 7), (3, n + 8), (0, 8216), (8, 8224)):
        big = torch.full((m, pitch), 123.0, dtype=out, device="cuda")
        y = kernel_opt.fp8_linear(xw[:, 16:16 + k], xs, ww[:, :k], ws, out=big[:, off:off + n])
        assert torch.equal(y, want)
        assert (big[:, :off] == 123).all() and (big[:, off + n:] == 123).all()


def test_zeros_and_nan():
    m, k, n = SHAPES[0]
    xq, xs, wq, ws = operands(m, k, n)
    z = torch.zeros_like(xq.view(torch.uint8)).view(torch.float8_e4m3fn)
    assert not kernel_opt.fp8_linear(z, xs, wq, ws).float().any()
    bad_x, bad_w = xs.clone(), ws.clone()
    bad_x[270, 32] = float("nan")
    bad_w[64, 1] = float("nan")        # the last 8 columns
    y = kernel_opt.fp8_linear(xq, bad_x, wq, bad_w)
    nan = torch.isnan(y)
    assert nan[270].all() and nan[:, 8192:].all()
    nan[270], nan[:, 8192:] = False, False
    assert not nan.any()
