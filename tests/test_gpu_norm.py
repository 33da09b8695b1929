"""Residual RMS norm (forward, backward, 8-bit output) against the same formulas in 64 bits.

Tolerances, from the arithmetic (u = half a unit in the last place of the output's type, e =
2^-24): a row's sum of squares adds at most 32 values per thread and then 5 + 16 more levels,
so the mean errs by less than 64 e and rstd by less than 32 e + 2 e (rsqrtf); y adds two
products: |dy| <= (u + 40 e) |y|.  ds errs by u |ds| and by 64 e times the size of its terms;
dw by N + 32 additions of e times the sum of its terms' magnitudes, and u |dw|.
"""
import math

import pytest
import torch

import kernel_opt

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: E}
# half the spacing of the smallest numbers a type holds
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
EPS = 1e-5


def inputs(n, h, dtype, wdtype=None, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed + 7 * n + h)
    r = lambda *s: torch.randn(s, generator=g, device="cuda")
    return ((scale * r(n, h)).to(dtype), (2 * scale * r(n, h)).to(dtype),
            (1 + 0.2 * r(h)).to(wdtype or dtype), r(n, h).to(dtype), r(n, h).to(dtype))


def reference(s, w, eps=EPS):
    s, w = s.double(), w.double()
    rstd = 1 / (s.square().mean(-1, keepdim=True) + eps).sqrt()
    return s * rstd * w, rstd


def check_y(y, s, w, eps=EPS):
    want, _ = reference(s, w, eps)
    err = (y.double() - want).abs()
    tol = (U[y.dtype] + 40 * E) * want.abs() + TINY[y.dtype]
    assert (err <= tol).all(), float((err - tol).max())


def check_grads(gy, gs, s, w, dx, dw, eps=EPS):
    n, h = s.shape
    _, rstd = reference(s, w, eps)
    norm, t = s.double() * rstd, gy.double() * w.double()
    c = (t * norm).mean(-1, keepdim=True)
    gs64 = torch.zeros_like(norm) if gs is None else gs.double()
    if dx is not None:
        want = rstd * (t - norm * c) + gs64
        size = rstd * (t.abs() + norm.abs() * (t * norm).abs().mean(-1, keepdim=True)) + gs64.abs()
        err = (dx.double() - want).abs()
        tol = U[dx.dtype] * want.abs() + 64 * E * size + TINY[dx.dtype]
        assert (err <= tol).all(), float((err - tol).max())
    if dw is not None:
        want = (gy.double() * norm).sum(0)
        size = (gy.double() * norm).abs().sum(0)
        err = (dw.double() - want).abs()
        tol = U[dw.dtype] * want.abs() + (n + 64) * E * size + TINY[dw.dtype]
        assert (err <= tol).all(), float((err - tol).max())


def train(x, r, w, gy, gs, eps=EPS):
    x = x.detach().requires_grad_(True)
    r = None if r is None else r.detach().requires_grad_(True)
    w = w.detach().requires_grad_(True)
    y, s = kernel_opt.fused_residual_rmsnorm(x, r, w, eps)
    ins = [x, w] if r is None else [x, r, w]
    outs, grads = ([y], [gy]) if gs is None else ([y, s], [gy, gs])
    got = torch.autograd.grad(outs, ins, grads)
    return y.detach(), s.detach(), got


SHAPES = [(1, 1), (3, 2), (5, 7), (2, 8), (9, 100), (4, 129), (1, 3584), (700, 3584), (333, 2051), (6, 8192),
          (3, 16384), (3, 16383), (2, 4104), (1300, 64), (3, 16382), (5, 5002), (2, 8198)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,h", SHAPES)
def test_forward_and_gradients(n, h, dtype):
    x, r, w, gy, gs = inputs(n, h, dtype)
    y, s, (dx, dr, dw) = train(x, r, w, gy, gs)
    assert torch.equal(s, (x.float() + r.float()).to(dtype))
    check_y(y, s, w)
    assert torch.equal(dx, dr)
    assert dx.dtype == dtype and dw.dtype == w.dtype and dw.shape == w.shape
    check_grads(gy, gs, s, w, dx, dw)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,h", [(7, 3584), (5, 77)])
def test_fp32_weight(n, h, dtype):
    x, r, w, gy, gs = inputs(n, h, dtype, torch.float32)
    y, s, (dx, _, dw) = train(x, r, w, gy, gs)
    check_y(y, s, w)
    assert dw.dtype == torch.float32
    check_grads(gy, gs, s, w, dx, dw)


def test_without_residual_and_without_the_streams_gradient():
    x, r, w, gy, gs = inputs(11, 520, torch.bfloat16)
    y, s, (dx, dw) = train(x, None, w, gy, None)
    assert s.data_ptr() == x.data_ptr()
    check_y(y, x, w)
    check_grads(gy, None, x, w, dx, dw)
    y, s, (dx, dr, dw) = train(x, r, w, gy, None)
    check_grads(gy, None, s, w, dx, dw)


def test_only_the_stream_is_used():
    x, r, w, _, gs = inputs(4, 96, torch.float32)
    x, r, w = (t.requires_grad_(True) for t in (x, r, w))
    _, s = kernel_opt.fused_residual_rmsnorm(x, r, w, EPS)
    dx, dr, dw = torch.autograd.grad(s, (x, r, w), gs, allow_unused=True)
    assert torch.equal(dx, gs) and torch.equal(dr, gs) and dw is None


@pytest.mark.parametrize("need", ["x", "weight", "residual"])
def test_gradients_that_are_not_wanted(need):
    x, r, w, gy, _ = inputs(17, 264, torch.bfloat16)
    ins = {"x": x, "residual": r, "weight": w}
    ins[need].requires_grad_(True)
    y, s = kernel_opt.fused_residual_rmsnorm(x, r, w, EPS)
    (d,) = torch.autograd.grad(y, ins[need], gy)
    check_grads(gy, None, s.detach(), w.detach(), None if need == "weight" else d, d if need == "weight" else None)


def test_gradient_matches_differences():
    """The kernel's gradient along a direction against central differences of the formula in
    64 bits: their error is h^2 f''' / 6 + 2^-52 |f| / h, far below the 1e-4 asked for; the
    kernel's own is below 64 e times the size of the terms."""
    x, r, w, gy, gs = inputs(3, 40, torch.float32)
    y, s, (dx, dr, dw) = train(x, r, w, gy, gs)
    g = torch.Generator(device="cuda").manual_seed(5)
    vx, vw = (torch.randn(t.shape, generator=g, device="cuda").double() for t in (x, w))

    def f(a):
        st = x.double() + r.double() + a * vx
        yy, _ = reference(st, w.double() + a * vw)
        return float((yy * gy.double()).sum() + (st * gs.double()).sum())
    h = 1e-4
    diff = (f(h) - f(-h)) / (2 * h)
    got = float((dx.double() * vx).sum() + (dw.double() * vw).sum())
    assert abs(got - diff) <= 1e-4 * max(1.0, abs(diff))


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts(dtype):
    """Padded rows, rows that start off a 16-byte boundary, 3-D inputs, expanded gradients."""
    n, h = 6, 384
    x, r, w, gy, _ = inputs(n, h, dtype)
    want = kernel_opt.fused_residual_rmsnorm(x, r, w, EPS)
    wide = torch.zeros(n, h + 24, dtype=dtype, device="cuda")
    for off in (0, 1, 8):
        xs = wide[:, off:off + h]
        xs.copy_(x)
        y, s = kernel_opt.fused_residual_rmsnorm(xs, r, w, EPS)
        assert torch.equal(s, want[1])
        check_y(y, s, w)
    y, s = kernel_opt.fused_residual_rmsnorm(x.view(2, 3, h), r.view(2, 3, h), w, EPS)
    assert y.shape == (2, 3, h) and torch.equal(y.view(n, h), want[0])
    xt = x.view(2, 3, h).transpose(0, 1)  # leading dimensions that do not collapse
    y, _ = kernel_opt.fused_residual_rmsnorm(xt, r.view(2, 3, h).transpose(0, 1), w, EPS)
    assert torch.equal(y, want[0].view(2, 3, h).transpose(0, 1))
    xr = x.clone().requires_grad_(True)
    y, s = kernel_opt.fused_residual_rmsnorm(xr, r, w, EPS)
    y.sum().backward()  # the gradient arrives with strides of zero
    check_grads(torch.ones_like(x), None, s.detach(), w, xr.grad, None)


@pytest.mark.parametrize("dtype", DTYPES)
def test_no_rows(dtype):
    x = torch.empty(0, 64, dtype=dtype, device="cuda", requires_grad=True)
    w = torch.ones(64, dtype=dtype, device="cuda", requires_grad=True)
    y, s = kernel_opt.fused_residual_rmsnorm(x, x.detach(), w, EPS)
    assert y.shape == s.shape == (0, 64)
    dx, dw = torch.autograd.grad(y, (x, w), torch.empty_like(y))
    assert dx.shape == (0, 64) and torch.equal(dw, torch.zeros_like(w))
    q, sc, _ = kernel_opt.fused_residual_rmsnorm_fp8(x.detach(), None, w.detach())
    assert q.shape == (0, 64) and sc.shape == (0, 1)


def test_zero_rows_of_values_and_non_finite():
    x = torch.zeros(4, 256, device="cuda")
    x[1, 3] = float("inf")
    x[2, 5] = float("nan")
    x[3] = 1e-3
    w = torch.ones(256, device="cuda")
    y, _ = kernel_opt.fused_residual_rmsnorm(x, torch.zeros_like(x), w, EPS)
    assert torch.equal(y[0], torch.zeros(256, device="cuda"))
    assert torch.isnan(y[1, 3]) and torch.isnan(y[2]).all()
    check_y(y[3:], x[3:], w)


def check_q(q, scale, y, slack):
    """q is y / scale rounded to e4m3: off by at most 2^-4 of itself, or 2^-10 below e4m3's
    normal numbers, and what `slack` (relative) allows y and the scale."""
    n, h = y.shape
    pad = -h % 128
    amax = torch.nn.functional.pad(y.abs(), (0, pad)).view(n, -1, 128).amax(2)
    want = amax.clamp(min=1e-30) / 448
    assert ((scale.double() - want).abs() <= slack * want).all()
    full = scale.double().repeat_interleave(128, 1)[:, :h]
    err = (q.double() * full - y).abs()
    tol = torch.maximum(y.abs() * 2 ** -4, full * 2 ** -10) * (1 + 1e-5) + 2 * slack * y.abs()
    assert (err <= tol).all(), float((err - tol).max())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,h", SHAPES)
def test_fp8_output(n, h, dtype):
    x, r, w, _, _ = inputs(n, h, dtype)
    q, scale, s = kernel_opt.fused_residual_rmsnorm_fp8(x, r, w, EPS)
    assert q.dtype == torch.float8_e4m3fn and q.shape == (n, h)
    assert scale.shape == (n, math.ceil(h / 128)) and scale.dtype == torch.float32
    assert torch.equal(s, (x.float() + r.float()).to(dtype))
    want, _ = reference(s, w)
    check_q(q, scale, want, 44 * E)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,h", [(1, 1), (5, 130), (3, 3584), (64, 16384), (7, 1003)])
def test_quantize_rows(n, h, dtype):
    x, *_ = inputs(n, h, dtype, scale=5.0)
    x[0] = 0
    q, scale = kernel_opt.quantize_fp8_rows(x)
    check_q(q, scale, x.double(), 4 * E)
    assert torch.equal(q[0].float(), torch.zeros(h, device="cuda"))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("o,h", [(1, 1), (128, 128), (129, 257), (1000, 3584), (300, 77)])
def test_quantize_blocks(o, h, dtype):
    w, *_ = inputs(o, h, dtype, scale=0.02)
    q, scale = kernel_opt.quantize_fp8_blocks(w)
    ob, hb = math.ceil(o / 128), math.ceil(h / 128)
    assert scale.shape == (ob, hb)
    y = w.double()
    padded = torch.nn.functional.pad(y.abs(), (0, -h % 128, 0, -o % 128)).view(ob, 128, hb, 128)
    want = padded.amax((1, 3)).clamp(min=1e-30) / 448
    assert ((scale.double() - want).abs() <= 2 * E * want).all()
    full = scale.double().repeat_interleave(128, 0)[:o].repeat_interleave(128, 1)[:, :h]
    err = (q.double() * full - y).abs()
    assert (err <= torch.maximum(y.abs() * 2 ** -4, full * 2 ** -10) * (1 + 1e-5)).all()
    # a weight given as a transposed or padded view
    wide = torch.zeros(o, h + 3, dtype=dtype, device="cuda")
    wide[:, 1:h + 1] = w
    q2, scale2 = kernel_opt.quantize_fp8_blocks(wide[:, 1:h + 1])
    assert torch.equal(q2.view(torch.uint8), q.view(torch.uint8)) and torch.equal(scale2, scale)


def test_fp8_non_finite_values():
    x = torch.ones(2, 256, device="cuda")
    x[0, 7] = float("nan")
    x[1, 200] = float("inf")
    q, scale = kernel_opt.quantize_fp8_rows(x)
    back = q.float() * scale.repeat_interleave(128, 1)
    assert torch.isnan(back[0, :128]).all() and torch.equal(back[0, 128:], x[0, 128:])
    assert torch.equal(back[1, :128], x[1, :128]) and torch.isnan(back[1, 128:]).all()


def test_other_stream_and_graph():
    x, r, w, gy, gs = inputs(64, 3584, torch.bfloat16)
    want = train(x, r, w, gy, gs)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = train(x, r, w, gy, gs)
    torch.cuda.current_stream().wait_stream(st)
    assert torch.equal(want[0], got[0]) and all(torch.equal(a, b) for a, b in zip(want[2], got[2]))
    g = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(g):
        y, _ = kernel_opt.fused_residual_rmsnorm(x, r, w, EPS)
    x.copy_(2 * x)
    g.replay()
    check_y(y, (x.float() + r.float()).to(x.dtype), w)


def test_refusals():
    x, r, w, gy, _ = inputs(4, 64, torch.bfloat16)
    f = kernel_opt.fused_residual_rmsnorm
    with pytest.raises(ValueError, match="residual must match"):
        f(x, r[:, :32], w)
    with pytest.raises(ValueError, match="residual must match"):
        f(x, r.float(), w)
    with pytest.raises(ValueError, match="one value per column"):
        f(x, r, w[:32])
    with pytest.raises(ValueError, match="eps must be positive"):
        f(x, r, w, 0.0)
    with pytest.raises(RuntimeError, match="weight must have x's dtype or fp32"):
        f(x, r, w.half())
    with pytest.raises(RuntimeError, match="bf16, fp16, or fp32"):
        f(x.double(), r.double(), w.double())
    with pytest.raises(RuntimeError, match="hidden must be in"):
        f(torch.zeros(1, 16385, device="cuda"), None, torch.zeros(16385, device="cuda"))
    with pytest.raises(ValueError, match="CUDA"):
        f(x.cpu(), r.cpu(), w.cpu())


def exact_q(y, of_block):
    """The e4m3 number nearest to 448 y / amax, from 64 bits."""
    return (448 * y / of_block).to(torch.float8_e4m3fn)


@pytest.mark.parametrize("n,h", [(40, 3584), (33, 1026), (50, 1003), (5, 1024), (300, 128)])
def test_8_bit_values_of_bf16_are_exact(n, h):
    """A product of two bf16 numbers has 16 bits, so the quotient by the largest of 128 lies at
    least 2^-22 (relative) away from a midpoint of e4m3 unless it is one: computed without a
    rounding before the quotient, every value is the nearest, and midpoints go to even."""
    x, r, w, _, _ = inputs(n, h, torch.bfloat16)
    per_row = lambda a: torch.nn.functional.pad(a.double().abs(), (0, -h % 128)).view(n, -1, 128).amax(
        2).repeat_interleave(128, 1)[:, :h]
    q, _, s = kernel_opt.fused_residual_rmsnorm_fp8(x, r, w, EPS)
    y = s.double() * w.double()
    assert torch.equal(q.float(), exact_q(y, per_row(y)).float())
    q, _ = kernel_opt.quantize_fp8_rows(x)
    assert torch.equal(q.float(), exact_q(x.double(), per_row(x)).float())
    q, scale = kernel_opt.quantize_fp8_blocks(x)
    ob, hb = scale.shape
    top = torch.nn.functional.pad(x.double().abs(), (0, -h % 128, 0, -n % 128)).view(ob, 128, hb, 128).amax((1, 3))
    top = top.repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :h]
    assert torch.equal(q.float(), exact_q(x.double(), top).float())


@pytest.mark.parametrize("h", [256, 258, 259])
def test_8_bit_values_beside_an_infinity(h):
    x = torch.randn(3, h, device="cuda")
    x[1, 5] = float("-inf")
    for q, scale in (kernel_opt.quantize_fp8_rows(x), kernel_opt.quantize_fp8_blocks(x)):
        f = q.float()
        assert torch.isnan(f[1, 5]) and scale[(1, 0) if scale.shape[0] == 3 else (0, 0)] == float("inf")
        f[1, 5] = 0
        assert torch.equal(f[1, :128], torch.zeros(128, device="cuda"))
        assert not torch.isnan(f).any()


@pytest.mark.parametrize("scale", [1e-34, 1e-30, 2.0 ** -60, 1e15])
@pytest.mark.parametrize("h", [256, 258, 259])
def test_8_bit_values_of_extreme_streams(h, scale):
    """Values far from 1: eps rules the small ones (R = 1000), and squares up to 1e30 sum."""
    x = torch.randn(4, h, device="cuda") * scale
    w = 1 + 0.1 * torch.randn(h, device="cuda")
    q, s, stream = kernel_opt.fused_residual_rmsnorm_fp8(x, None, w, EPS)
    want, _ = reference(stream, w)
    check_q(q, s, want, 44 * E)
