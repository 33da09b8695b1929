"""The 8-bit product with bias, activation and residual against the same in 64 bits.

Tolerance: the product errs by d = (128 + ceil(K / 128) + 12) 2^-23 * sum |terms| (derived in
test_gpu_fp8_linear), the bias' addition by 2^-24 of the result.  An activation's slope is at most
1.13; its evaluation errs relative to its value by an exponential's argument u (a relative 2^-22) and
value (2 + 1.17 |u| units), a complementary error function's argument (z^2 2^-23) and value (4 units) and a
quotient (2 units): below 2^-22 (4 + 2 |u| + z^2).  The residual's addition rounds by 2^-24, and the
result is rounded once to its type.  Where an exponential overflows the quotient is 0 for less than
1e-36.
"""
import math

import pytest
import torch

import kernel_opt
from _linear import MANY, kernel_of
from test_gpu_fp8_linear import TINY, U, operands, reference

pytestmark = pytest.mark.gpu

ACTS = [None, "relu", "silu", "gelu", "gelu_tanh"]


def exact(act, v):
    """(activation in 64 bits, |u| + z^2 terms of its error)"""
    zero = torch.zeros_like(v)
    if act == "relu":
        return v.clamp(min=0), zero
    if act == "silu":
        return torch.nn.functional.silu(v), 2 * v.abs()
    if act == "gelu":
        return 0.5 * v * torch.erfc(-v * math.sqrt(0.5)), v * v
    if act == "gelu_tanh":
        u = 2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)
        return v * torch.sigmoid(u), 2 * u.abs()
    return v, zero


def check(y, ops, bias, act, residual):
    want, size = reference(*ops)
    d = (128 + ops[1].shape[1] + 12) * 2.0 ** -23 * size
    if bias is not None:
        want = want + bias.double()
        d = d + 2.0 ** -23 * want.abs()
    want, terms = exact(act, want)
    tol = 1.13 * d + 2.0 ** -22 * (4 + terms) * want.abs() + 1e-36
    if residual is not None:
        want = want + residual.double()
        tol = tol + 2.0 ** -23 * want.abs()
    err = (y.double() - want).abs()
    tol = U[y.dtype] * (want.abs() + tol) + tol + TINY[y.dtype]
    assert (err <= tol).all(), (float((err - tol).max()), float(err.max()))


def small(m, k, n, out):
    """Operands whose products are of the size activations are made for."""
    xq, xs, wq, ws = operands(m, k, n)
    f = (0.4 / (60 * 60 * 0.02 ** 2 * math.sqrt(k))) ** 0.5
    return xq, xs * f * 0.1, wq, ws * f


def extras(m, n, out, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed + m + n)
    r = lambda *s: torch.randn(s, generator=g, device="cuda")
    return (2 * r(n)).to(out), (3 * r(m, n)).to(out)


# one block's columns, K split over a cluster, whole and ragged tiles, odd columns, many tokens
SHAPES = [(1, 16, 1), (3, 144, 130), (16, 3584, 1000), (17, 1040, 257), (33, 512, 129), (64, 3584, 333),
          (65, 128, 20001), (300, 4176, 8200), (300, 4176, 8201), (257, 3584, 8192)]


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_against_64_bits(m, k, n, out):
    ops = small(m, k, n, out)
    bias, residual = extras(m, n, out)
    for act in ACTS:
        for b, r in ((bias, residual), (bias, None), (None, residual), (None, None)):
            y = kernel_opt.fp8_linear(*ops, out, bias=b, activation=act, residual=r)
            assert y.shape == (m, n) and y.dtype == out
            check(y, ops, b, act, r)
    y = kernel_opt.fp8_linear(*ops, out, bias=bias.float(), activation="silu")
    check(y, ops, bias.float(), "silu", None)
    # without an epilogue the product's own bits, and an addition of nothing changes none
    plain = kernel_opt.fp8_linear(*ops, out)
    assert torch.equal(plain, kernel_opt.fp8_linear(*ops, out, bias=torch.zeros_like(bias)))
    assert torch.equal(plain, kernel_opt.fp8_linear(*ops, out, residual=torch.zeros_like(residual)))


def test_shapes_take_both_kernels():
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert {kernel_of(*s, sms) for s in SHAPES} == {16, 32, 64, MANY}


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("m,k,n", [(5, 272, 333), (40, 272, 3334), (300, 4176, 8200)])
def test_layouts_and_in_place(m, k, n, out):
    ops = small(m, k, n, out)
    bias, residual = extras(m, n, out)
    want = kernel_opt.fp8_linear(*ops, out, bias=bias, activation="gelu", residual=residual)
    check(want, ops, bias, "gelu", residual)
    for off in (0, 1, 3):
        big = torch.full((m, n + 7), 7.0, device="cuda").to(out)
        at = big[:, off:off + n]
        wide = torch.zeros(m, n + 5, device="cuda").to(out)
        wide[:, off:off + n] = residual
        y = kernel_opt.fp8_linear(*ops, out=at, bias=torch.cat([bias[:1], bias])[1:], activation="gelu",
                                  residual=wide[:, off:off + n])
        assert torch.equal(y, want)
        assert (big[:, :off] == 7).all() and (big[:, off + n:] == 7).all()
        at.copy_(residual)  # updated in place
        kernel_opt.fp8_linear(*ops, out=at, bias=bias, activation="gelu", residual=at)
        assert torch.equal(at, want) and (big[:, :off] == 7).all() and (big[:, off + n:] == 7).all()
    row = residual[:1].expand(m, n)  # broadcast and transposed residuals, more dimensions
    y = kernel_opt.fp8_linear(*ops, out, residual=row)
    check(y, ops, None, None, row)
    turned = residual.t().contiguous().t()
    y = kernel_opt.fp8_linear(*ops, out, bias=bias, activation="gelu", residual=turned)
    assert torch.equal(y, want)
    xq, xs, wq, ws = ops
    y = kernel_opt.fp8_linear(xq.view(1, m, k), xs.view(1, m, -1), wq, ws, out, bias=bias, activation="gelu",
                              residual=residual.view(1, m, n))
    assert y.shape == (1, m, n) and torch.equal(y[0], want)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("m", [2, 300])
def test_far_values_and_nan(act, out, m):
    # the bias alone decides: far tails, both infinities, NaN
    k, n = 4176 if m > 64 else 128, 8200 if m > 64 else 130
    xq, xs, wq, ws = operands(m, k, n)
    xq = torch.zeros(m, k, device="cuda").to(torch.float8_e4m3fn)
    bias = torch.linspace(-130, 130, n, device="cuda").to(out)
    y = kernel_opt.fp8_linear(xq, xs, wq, ws, out, bias=bias, activation=act)
    check(y, (xq, xs, wq, ws), bias, act, None)
    bias[0], bias[1] = torch.nan, torch.inf
    y = kernel_opt.fp8_linear(xq, xs, wq, ws, out, bias=bias, activation=act)
    assert y[:, 0].isnan().all() and (y[:, 1] == torch.inf).all() and y[:, 2:].isfinite().all()


def test_refusals():
    ops = operands(4, 256, 100)
    bias, residual = extras(4, 100, torch.bfloat16)
    with pytest.raises(ValueError, match="activation must be"):
        kernel_opt.fp8_linear(*ops, activation="tanh")
    with pytest.raises(ValueError, match="activation must be"):
        kernel_opt.fp8_linear(*ops, activation="none")
    with pytest.raises(ValueError, match="bias must be"):
        kernel_opt.fp8_linear(*ops, bias=bias[:50])
    with pytest.raises(ValueError, match="bias must be"):
        kernel_opt.fp8_linear(*ops, bias=bias.cpu())
    with pytest.raises(RuntimeError, match="output's dtype"):
        kernel_opt.fp8_linear(*ops, bias=bias.half())
    with pytest.raises(RuntimeError, match="output's dtype"):
        kernel_opt.fp8_linear(*ops, residual=residual.float())
    with pytest.raises(ValueError, match="shaped like the product"):
        kernel_opt.fp8_linear(*ops, residual=residual[:2])
    big = torch.zeros(4, 104, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="lie apart"):
        kernel_opt.fp8_linear(*ops, out=big[:, :100], residual=big[:, 2:102])
    with pytest.raises(ValueError, match="lie apart"):
        kernel_opt.fp8_linear(*ops, out=big[:, :100], residual=big.view(-1)[:400].view(4, 100))


def test_captured():
    ops = small(16, 1040, 4100, torch.bfloat16)
    bias, residual = extras(16, 4100, torch.bfloat16)
    step = lambda: kernel_opt.fp8_linear(*ops, bias=bias, activation="silu", residual=residual)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step()
    bias.mul_(0.5)
    graph.replay()
    assert torch.equal(y, step())


def test_nothing_to_do():
    xq, xs, wq, ws = operands(4, 256, 100)
    y = kernel_opt.fp8_linear(xq[:0], xs[:0], wq, ws, bias=torch.zeros(100, device="cuda"), activation="relu",
                              residual=torch.zeros(0, 100, device="cuda", dtype=torch.bfloat16))
    assert y.shape == (0, 100)
