"""The norms around a block's end (forward, 8-bit output, backward) against the formulas in 64 bits.

Tolerances, from the arithmetic (u = half a step of the output's type, e = 2^-24), as for the
residual norm: rstd errs by less than 34 e, the branch by 40 e with its products, so
|d stream| <= u |s| + 45 e (|rs r| + |branch|).  The rest is taken from the stored stream: ds errs by 64 e
of the size of its terms, D; what is made of it by a product with w adds under 40 e of it: 110 e D |w|;
sums over N rows or H columns add (N + 32) e or 96 e of the sum of magnitudes, and dx, with one such mean
in it, 250 e of its terms' size.  Each is rounded once more to its type.
"""
import pytest
import torch

import kernel_opt

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: E}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
EPS = 1e-5
GATES = ["none", "column", "token", "full"]


def inputs(n, h, dtype, gate, wdtype=None, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + 7 * n + h)
    r = lambda *s: torch.randn(s, generator=g, device="cuda")
    shape = {"column": (h,), "token": (n, 1), "full": (n, h)}.get(gate)
    w = wdtype or dtype
    return {"x": (3 * r(n, h)).to(dtype), "residual": (2 * r(n, h)).to(dtype), "post_weight": (1 + 0.2 * r(h)).to(w),
            "weight": (1 + 0.2 * r(h)).to(w), "gate": None if shape is None else
            (0.5 + 0.3 * r(*shape)).to(w if gate == "column" else dtype)}, r(n, h).to(dtype), r(n, h).to(dtype)


def within(got, want, tol, what):
    err = (got.double() - want).abs()
    bad = ~((err <= tol) | (got.isnan() & want.isnan()))
    assert not bad.any(), (what, float((err - tol)[bad].max()), int(bad.sum()))


def branch(t, bs):
    x = t["x"].double()
    r1 = 1 / (x.square().mean(-1, keepdim=True) + EPS).sqrt()
    gate = 1.0 if t["gate"] is None else t["gate"].double()
    return r1, x * r1, bs * gate * x * r1 * t["post_weight"].double()


def check_forward(t, y, stream, bs, rs):
    _, _, b = branch(t, bs)
    r = rs * t["residual"].double()
    u = U[stream.dtype]
    within(stream, r + b, u * (r + b).abs() + 45 * E * (r.abs() + b.abs()) + TINY[stream.dtype], "stream")
    s = stream.double()
    want = s / (s.square().mean(-1, keepdim=True) + EPS).sqrt() * t["weight"].double()
    within(y, want, (U[y.dtype] + 40 * E) * want.abs() + TINY[y.dtype], "y")


def check_grads(t, stream, gy, gs, got, bs, rs):
    n, h = stream.shape
    zero = torch.zeros(n, h, dtype=torch.float64, device="cuda")
    gy = zero if gy is None else gy.double()
    gs = zero if gs is None else gs.double()
    s, w, wp = stream.double(), t["weight"].double(), t["post_weight"].double()
    gate = 1.0 if t["gate"] is None else t["gate"].double()
    r1, m, _ = branch(t, bs)
    r2 = 1 / (s.square().mean(-1, keepdim=True) + EPS).sqrt()
    nn, gw = s * r2, gy * w
    ds = r2 * (gw - nn * (gw * nn).mean(-1, keepdim=True)) + gs
    size = r2 * (gw.abs() + nn.abs() * (gw * nn).abs().mean(-1, keepdim=True)) + gs.abs()
    u, tiny = U[stream.dtype], TINY[stream.dtype]
    wu = U[t["weight"].dtype]
    wtiny = TINY[t["weight"].dtype]

    def check(name, want, tol, half, small):
        if got.get(name) is not None:
            within(got[name], want, half * want.abs() + tol + small, name)

    check("residual", rs * ds, 66 * E * abs(rs) * size, u, tiny)
    check("weight", (gy * nn).sum(0), (n + 80) * E * (gy * nn).abs().sum(0), wu, wtiny)
    p = bs * ds * gate * m
    check("post_weight", p.sum(0), (n + 150) * E * (bs * size * gate * m).abs().sum(0), wu, wtiny)
    q, qs = bs * ds * m * wp, (bs * size * m * wp).abs()
    kind = None if t["gate"] is None else tuple(t["gate"].shape)
    if kind == (h,):
        check("gate", q.sum(0), (n + 150) * E * qs.sum(0), wu, wtiny)
    elif kind == (n, h):
        check("gate", q, 110 * E * qs, u, tiny)
    elif kind == (n, 1):
        check("gate", q.sum(1, keepdim=True), 210 * E * qs.sum(1, keepdim=True), u, tiny)
    a, asz = bs * ds * gate * wp, (bs * size * gate * wp).abs()
    want = r1 * (a - m * (a * m).mean(-1, keepdim=True))
    check("x", want, 250 * E * r1 * (asz + m.abs() * (asz * m.abs()).mean(-1, keepdim=True)), u, tiny)


def run(t, gy, gs, bs, rs, wanted=("x", "residual", "post_weight", "weight", "gate")):
    leaf = {k: (v.detach().requires_grad_(k in wanted) if v is not None else None) for k, v in t.items()}
    y, stream = kernel_opt.fused_sandwich_rmsnorm(**leaf, branch_scale=bs, residual_scale=rs, eps=EPS)
    names = [k for k in leaf if leaf[k] is not None and k in wanted]
    outs = [(o, g) for o, g in ((y, gy), (stream, gs)) if g is not None]
    grads = torch.autograd.grad([o for o, _ in outs], [leaf[k] for k in names], [g for _, g in outs])
    return y.detach(), stream.detach(), dict(zip(names, grads))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("n,h", [(1, 1), (3, 2), (5, 7), (1, 3584), (64, 128), (33, 2051), (600, 256), (17, 4098),
                                 (40, 8192), (9, 16384), (4, 16383), (3, 10242)])
def test_against_64_bits(dtype, gate, n, h):
    t, gy, gs = inputs(n, h, dtype, gate)
    y, stream, got = run(t, gy, gs, 0.7, 0.9)
    check_forward(t, y, stream, 0.7, 0.9)
    check_grads(t, stream, gy, gs, got, 0.7, 0.9)
    for k, v in got.items():
        assert v.shape == t[k].shape and v.dtype == t[k].dtype


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("gate", ["none", "column"])
def test_weights_in_fp32(dtype, gate):
    t, gy, gs = inputs(70, 1000, dtype, gate, torch.float32)
    y, stream, got = run(t, gy, gs, 1.0, 1.0)
    check_forward(t, y, stream, 1.0, 1.0)
    check_grads(t, stream, gy, gs, got, 1.0, 1.0)


@pytest.mark.parametrize("gate", GATES)
def test_many_rows_and_parts_of_the_gradient(gate):
    t, gy, gs = inputs(3000, 640, torch.bfloat16, gate)
    for wanted in (("x",), ("residual", "gate"), ("post_weight", "weight"), ("gate",), ("x", "residual")):
        if wanted == ("gate",) and gate == "none":
            continue
        for a, b in ((gy, gs), (gy, None), (None, gs)):
            y, stream, got = run(t, a, b, 1.0, 0.5, wanted)
            check_grads(t, stream, a, b, got, 1.0, 0.5)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("n,h", [(1, 3584), (5, 7), (33, 2051), (64, 128), (6, 16384), (500, 1026)])
def test_eight_bits(dtype, gate, n, h):
    t, _, _ = inputs(n, h, dtype, gate)
    y, stream = kernel_opt.fused_sandwich_rmsnorm(**t, branch_scale=1.3, eps=EPS)
    check_forward(t, y, stream, 1.3, 1.0)
    q, scales, s8 = kernel_opt.fused_sandwich_rmsnorm_fp8(**t, branch_scale=1.3, eps=EPS)
    assert torch.equal(s8, stream)
    # from the stored stream on it is the residual norm
    q0, scales0, _ = kernel_opt.fused_residual_rmsnorm_fp8(stream, None, t["weight"], EPS)
    assert torch.equal(q.view(torch.uint8), q0.view(torch.uint8)) and torch.equal(scales, scales0)
    y0, _ = kernel_opt.fused_residual_rmsnorm(stream, None, t["weight"], EPS)
    assert torch.equal(y, y0)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_layouts(dtype):
    # rows of any pitch and start, broadcast and transposed ones, and more than two dimensions
    def leaf(*s):
        return torch.randn(s, device="cuda").to(dtype)
    cases = [
        (leaf(6, 300)[:, 5:205], leaf(6, 400)[:, ::2], leaf(1, 200).expand(6, 200)),
        (leaf(200, 6).t(), leaf(1, 200).expand(6, 200), leaf(6, 1).expand(6, 200)),
        (leaf(2, 3, 256), leaf(3, 2, 256).transpose(0, 1), leaf(2, 3, 1)),
        (leaf(2, 3, 256), leaf(2, 3, 256), leaf(2, 1, 256).expand(2, 3, 256)),
        (leaf(256), leaf(256), leaf(256)), (leaf(257), leaf(257), leaf(1)),
    ]
    for x, residual, gate in cases:
        h = x.shape[-1]
        off = torch.randn(2 * h + 1, device="cuda").to(dtype)
        t = {"x": x, "residual": residual, "post_weight": off[1:h + 1], "weight": off[h + 1:], "gate": gate}
        t = {k: v.detach().requires_grad_(True) for k, v in t.items()}
        y, stream = kernel_opt.fused_sandwich_rmsnorm(**t, eps=EPS)
        gy = torch.randn(1, device="cuda").to(dtype).expand_as(y)
        gs = torch.randn(y.shape[::-1], device="cuda").to(dtype).permute(*range(y.dim())[::-1])
        got = dict(zip(t, torch.autograd.grad((y, stream), list(t.values()), (gy, gs))))
        flat = {k: (v.detach().reshape(-1, v.shape[-1]) if k in ("x", "residual") or
                    (k == "gate" and v.dim() == x.dim() and v.dim() > 1) else v.detach()) for k, v in t.items()}
        if x.dim() == 1 and gate.shape[-1] == 1:
            flat["gate"] = gate.reshape(1, 1)
        rows = lambda v: v.reshape(-1, h)
        check_forward(flat, rows(y.detach()), rows(stream.detach()), 1.0, 1.0)
        for k in ("x", "residual", "gate"):
            got[k] = got[k].reshape(flat[k].shape)
        check_grads(flat, rows(stream.detach()), rows(gy), rows(gs), got, 1.0, 1.0)


def test_gradient_against_differences():
    # fp32, step 2^-6: the difference errs by its third derivative (under h^2 of the terms' size) and
    # by the outputs' 64 e over h
    t, gy, gs = inputs(5, 96, torch.float32, "full")
    _, _, got = run(t, gy, gs, 0.6, 0.8)
    h = 2.0 ** -6

    def loss(t):
        y, stream = kernel_opt.fused_sandwich_rmsnorm(**t, branch_scale=0.6, residual_scale=0.8, eps=EPS)
        return (y.double() * gy.double()).sum() + (stream.double() * gs.double()).sum()

    size = float(gy.abs().sum() * 3 + gs.abs().sum() * 3)
    for k in t:
        g = torch.Generator(device="cuda").manual_seed(len(k))
        v = 0.3 * torch.randn(t[k].shape, generator=g, device="cuda")
        up, down = ({**t, k: t[k] + s * h * v} for s in (1, -1))
        slope = (loss(up) - loss(down)) / (2 * h)
        want = (got[k].double() * v.double()).sum()
        assert abs(float(slope - want)) <= size * (64 * E / h + h * h), (k, float(slope), float(want))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_zeros_infinities_and_nan_stay_in_their_rows(dtype):
    t, gy, gs = inputs(6, 520, dtype, "token")
    t["x"][0] = 0
    t["x"][1, 7] = torch.nan
    t["residual"][2, 9] = torch.inf
    t["gate"][3] = 0
    y, stream, got = run(t, gy, gs, 1.0, 1.0, ("x", "residual", "gate"))
    keep = torch.tensor([0, 3, 4, 5], device="cuda")
    part = {k: (v[keep] if k in ("x", "residual", "gate") else v) for k, v in t.items()}
    check_forward(part, y[keep], stream[keep], 1.0, 1.0)
    check_grads(part, stream[keep], gy[keep], gs[keep], {k: v[keep] for k, v in got.items()}, 1.0, 1.0)
    assert stream[1].isnan().all() and y[2].isnan().any()


def test_empty_and_no_gradient():
    t, _, _ = inputs(4, 64, torch.bfloat16, "column")
    e = {**t, "x": t["x"][:0], "residual": t["residual"][:0]}
    e = {k: v.detach().requires_grad_(True) for k, v in e.items()}
    y, stream = kernel_opt.fused_sandwich_rmsnorm(**e)
    grads = torch.autograd.grad((y.sum() + stream.sum()), list(e.values()))
    assert all((g == 0).all() for g in grads) and y.shape == (0, 64)
    y, stream = kernel_opt.fused_sandwich_rmsnorm(**t)
    assert not y.requires_grad
    t["x"].requires_grad_(True)
    with torch.no_grad():
        assert not kernel_opt.fused_sandwich_rmsnorm(**t)[0].requires_grad
    assert not any(o.requires_grad for o in kernel_opt.fused_sandwich_rmsnorm_fp8(**t))
    y, _ = kernel_opt.fused_sandwich_rmsnorm(**t)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(y.sum(), t["x"], create_graph=True)


def test_refusals():
    t, _, _ = inputs(4, 64, torch.bfloat16, "full")
    call = lambda **kw: kernel_opt.fused_sandwich_rmsnorm(**{**t, **kw})
    for f in (kernel_opt.fused_sandwich_rmsnorm, kernel_opt.fused_sandwich_rmsnorm_fp8):
        with pytest.raises(ValueError, match="residual must match"):
            f(**{**t, "residual": t["residual"][:, :32]})
        with pytest.raises(ValueError, match="post_weight must match"):
            f(**{**t, "post_weight": t["post_weight"].float()})
        with pytest.raises(ValueError, match="gate must be"):
            f(**{**t, "gate": t["gate"][:2]})
        with pytest.raises(ValueError, match="gate must be"):
            f(**{**t, "gate": t["gate"][:, :32]})
        with pytest.raises(RuntimeError, match="x's dtype"):
            f(**{**t, "gate": t["gate"].float()})
        with pytest.raises(RuntimeError, match="weights' dtype"):
            f(**{**t, "gate": t["gate"][0].float()})
        with pytest.raises(ValueError, match="on x's device"):
            f(**{**t, "gate": t["gate"].cpu()})
        for bad in (float("nan"), float("inf")):
            with pytest.raises(RuntimeError, match="finite"):
                f(**t, branch_scale=bad)
            with pytest.raises(RuntimeError, match="finite"):
                f(**t, residual_scale=bad)
        with pytest.raises(ValueError, match="eps"):
            f(**t, eps=0.0)
    with pytest.raises(RuntimeError, match="hidden"):
        w = torch.ones(16385, device="cuda")
        kernel_opt.fused_sandwich_rmsnorm(torch.ones(1, 16385, device="cuda"), torch.ones(1, 16385, device="cuda"), w, w)
    import torch.autograd.forward_ad as fw
    with fw.dual_level(), pytest.raises(RuntimeError, match="forward AD"):
        call(x=fw.make_dual(t["x"], torch.ones_like(t["x"])))


def test_captured_and_on_another_stream():
    t, gy, gs = inputs(40, 1024, torch.bfloat16, "column")
    t = {k: v.requires_grad_(True) for k, v in t.items()}

    def step():
        out = kernel_opt.fused_sandwich_rmsnorm(**t, branch_scale=0.5)
        return (*out, *torch.autograd.grad(out, list(t.values()), (gy, gs)), *kernel_opt.fused_sandwich_rmsnorm_fp8(**t))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in (1, 2):
        with torch.no_grad():
            for k, v in inputs(40, 1024, torch.bfloat16, "column", seed=seed)[0].items():
                t[k].copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, step()):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("n,h", [(700, 256), (460, 1000), (450, 2048), (501, 3584), (333, 4096), (300, 5120), (299, 8192)])
def test_more_rows_than_sms(dtype, gate, n, h):
    t, gy, gs = inputs(n, h, dtype, gate)
    y, stream, got = run(t, gy, gs, 0.7, 0.9)
    check_forward(t, y, stream, 0.7, 0.9)
    check_grads(t, stream, gy, gs, got, 0.7, 0.9)
    q, scales, s8 = kernel_opt.fused_sandwich_rmsnorm_fp8(**t, branch_scale=0.7, residual_scale=0.9, eps=EPS)
    assert torch.equal(s8, stream)
    s = stream.double()
    v = s / (s.square().mean(-1, keepdim=True) + EPS).sqrt() * t["weight"].double()
    step = scales.double().repeat_interleave(128, 1)[:, :h]
    top = torch.nn.functional.pad(v.abs(), (0, -h % 128)).unflatten(-1, (-1, 128)).amax(-1) / 448
    # the norm's own error (see check_forward) and four more roundings
    within(scales, top, 44 * E * top, "scales")
    # half a step of e4m3 (2^-4 of the value, or 2^-10 where it is subnormal), and the same
    within(q.double() * step, v, torch.maximum(v.abs() / 16, step / 1024) * (1 + 100 * E) + 100 * E * v.abs(), "q")
