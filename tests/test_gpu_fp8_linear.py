"""8-bit product with block scales against the same sum in 64 bits.

Tolerance: products of two e4m3 numbers are exact in fp32.  A block's 128 additions on the
tensor cores lose at most 2^-23 of the sum of magnitudes each, its scaling and the addition of
the ceil(K / 128) blocks (and up to 8 parts of K) half of that each, and the result is rounded
once: |dy| <= u |y| + (128 + ceil(K / 128) + 12) 2^-23 * sum |terms|, and half the spacing of
fp16's subnormal numbers for an fp16 result.
"""
import math

import pytest
import torch

import kernel_opt

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}


def operands(m, k, n, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + m + 3 * k + 7 * n)
    kb, nb = math.ceil(k / 128), math.ceil(n / 128)
    xq = torch.randn(m, k, generator=g, device="cuda").mul_(60).to(torch.float8_e4m3fn)
    wq = torch.randn(n, k, generator=g, device="cuda").mul_(60).to(torch.float8_e4m3fn)
    # scales over several powers of two, none of them one
    xs = torch.rand(m, kb, generator=g, device="cuda").mul_(4).exp_().mul_(1e-3)
    ws = torch.rand(nb, kb, generator=g, device="cuda").mul_(4).exp_().mul_(1e-3)
    return xq, xs, wq, ws


def reference(xq, xs, wq, ws):
    k, n = xq.shape[1], wq.shape[0]
    x = xq.double() * xs.double().repeat_interleave(128, 1)[:, :k]
    w = wq.double() * ws.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    return x @ w.t(), x.abs() @ w.abs().t()


def check(y, xq, xs, wq, ws):
    want, size = reference(xq, xs, wq, ws)
    kb = xs.shape[1]
    err = (y.double() - want).abs()
    tol = U[y.dtype] * want.abs() + (128 + kb + 12) * 2.0 ** -23 * size + TINY[y.dtype]
    assert (err <= tol).all(), (float((err - tol).max()), float(err.max()))


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m,k,n", [
    (1, 16, 1), (1, 128, 128), (3, 144, 130), (16, 1040, 1000), (17, 3584, 256), (32, 256, 300),
    (33, 512, 129), (64, 3584, 1000), (65, 128, 40000), (130, 272, 30001), (257, 384, 20000),
    (1, 8192, 77), (128, 1040, 38000), (300, 3584, 5000), (100, 2048, 100)])
def test_product(m, k, n, out):
    ops = operands(m, k, n)
    if out == torch.float16:  # stay inside fp16's range
        ops = (ops[0], ops[1] * 0.02, ops[2], ops[3] * 0.02)
    y = kernel_opt.fp8_linear(*ops, out)
    assert y.shape == (m, n) and y.dtype == out
    check(y, *ops)


def test_head_sized():
    for m in (1, 40, 200):
        ops = operands(m, 3584, 32000)
        check(kernel_opt.fp8_linear(*ops), *ops)


@pytest.mark.parametrize("m", [5, 300])
def test_layouts(m):
    """Operands inside wider rows, outputs inside wider rows and off 16-byte boundaries;
    nothing outside the output is written."""
    k, n = 272, 20000 if m > 64 else 333
    xq, xs, wq, ws = operands(m, k, n)
    want = kernel_opt.fp8_linear(xq, xs, wq, ws)
    xw = torch.zeros(m, k + 48, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    ww = torch.zeros(n, k + 32, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    xw.view(torch.uint8)[:, 16:16 + k] = xq.view(torch.uint8)
    ww.view(torch.uint8)[:, :k] = wq.view(torch.uint8)
    for off in (0, 1, 3):
        big = torch.full((m, n + 7), 123.0, dtype=torch.bfloat16, device="cuda")
        y = kernel_opt.fp8_linear(xw[:, 16:16 + k], xs, ww[:, :k], ws, out=big[:, off:off + n])
        assert torch.equal(y, want)
        assert (big[:, :off] == 123).all() and (big[:, off + n:] == 123).all()
    y = kernel_opt.fp8_linear(xq.view(1, m, k), xs.view(1, m, -1), wq, ws)
    assert y.shape == (1, m, n) and torch.equal(y[0], want)


def test_repeatable_and_independent_of_the_batch():
    xq, xs, wq, ws = operands(16, 3584, 4096)
    y = kernel_opt.fp8_linear(xq, xs, wq, ws)
    assert torch.equal(y, kernel_opt.fp8_linear(xq, xs, wq, ws))
    assert torch.equal(y[3:4], kernel_opt.fp8_linear(xq[3:4], xs[3:4], wq, ws))


def test_zeros_and_nan():
    xq, xs, wq, ws = operands(4, 256, 200)
    z = torch.zeros_like(xq.view(torch.uint8)).view(torch.float8_e4m3fn)
    assert torch.equal(kernel_opt.fp8_linear(z, xs, wq, ws), torch.zeros(4, 200, dtype=torch.bfloat16, device="cuda"))
    bad = xs.clone()
    bad[2, 1] = float("nan")
    y = kernel_opt.fp8_linear(xq, bad, wq, ws)
    assert torch.isnan(y[2]).all() and torch.isfinite(y[[0, 1, 3]]).all()


def test_empty():
    xq, xs, wq, ws = operands(4, 256, 200)
    assert kernel_opt.fp8_linear(xq[:0], xs[:0], wq, ws).shape == (0, 200)
    assert kernel_opt.fp8_linear(xq, xs, wq[:0], ws[:0]).shape == (4, 0)


def test_quantised_operands_end_to_end():
    """A product of quantised matrices is near the product of the matrices: each operand errs
    by at most 2^-4 of an element (and 2^-10 of its block's scale)."""
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(24, 3584, generator=g, device="cuda").bfloat16()
    w = torch.randn(1000, 3584, generator=g, device="cuda").mul_(0.02).bfloat16()
    xq, xs = kernel_opt.quantize_fp8_rows(x)
    wq, ws = kernel_opt.quantize_fp8_blocks(w)
    y = kernel_opt.fp8_linear(xq, xs, wq, ws, torch.float32)
    want = x.double() @ w.double().t()
    size = (x.double().abs() + 4 * 2 ** -10) @ (w.double().abs() + 0.1 * 2 ** -10).t()
    assert ((y.double() - want).abs() <= (2 * 2 ** -4 + 2 ** -8) * size).all()


def test_other_stream_and_graph():
    ops = operands(8, 3584, 2048)
    want = kernel_opt.fp8_linear(*ops)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = kernel_opt.fp8_linear(*ops)
    torch.cuda.current_stream().wait_stream(st)
    assert torch.equal(want, got)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = kernel_opt.fp8_linear(*ops)
    y.zero_()
    g.replay()
    assert torch.equal(y, want)


def test_refusals():
    xq, xs, wq, ws = operands(4, 256, 200)
    f = kernel_opt.fp8_linear
    with pytest.raises(RuntimeError, match="float8_e4m3fn"):
        f(xq.bfloat16(), xs, wq, ws)
    with pytest.raises(RuntimeError, match="x_scales must be"):
        f(xq, xs[:, :1], wq, ws)
    with pytest.raises(RuntimeError, match="weight_scales must be"):
        f(xq, xs, wq, ws[:1])
    with pytest.raises(RuntimeError, match=r"x \[N, H\] and weight \[O, H\]"):
        f(xq[:, :128], xs, wq, ws)
    with pytest.raises(RuntimeError, match="multiple of 16"):
        f(xq[:, :250].contiguous(), xs, wq[:, :250].contiguous(), ws)
    with pytest.raises(RuntimeError, match="multiples of 16 bytes"):
        f(xq[:, 8:136], xs[:, :1], wq[:, :128], ws[:, :1])
    with pytest.raises(ValueError, match="out_dtype"):
        f(xq, xs, wq, ws, torch.float64)
    with pytest.raises(RuntimeError, match="output must be"):
        f(xq, xs, wq, ws, out=torch.empty(4, 100, device="cuda"))
    with pytest.raises(ValueError, match="leading dimensions"):
        f(xq, xs[:2], wq, ws)
