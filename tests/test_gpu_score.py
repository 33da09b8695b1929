"""Log-probabilities of given and of the most likely tokens, with their gradient, in 64 bits.

Tolerances, from the arithmetic (e = 2^-24).  Log-probabilities and lse: the sum of weights has
terms right to 2^-21 (the exponent's product rounds by e times its size, at most 150; ex2 adds 2^-22)
and is added in fp32 per thread, then in fp64: under 64 e of the sum, 4e-6 in the logarithm;
the result is rounded to fp32: 1e-5 + e |value|.  Entropy: the same for both sums, against a
logarithm: 1e-5 (1 + its terms, log Z and sum w d / Z).  Gradient: half a step of its type, and 2e-5 of
the size of its terms (lse and the entropy come rounded to fp32, at most 64 e each; the exponent as
above).  Ids are exact.
"""
import pytest
import torch

import kernel_opt

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: E}
# half the spacing of the smallest numbers a type holds
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def scale_of(temperature):
    return torch.tensor(1.0 / temperature, dtype=torch.float64).float().double().item()


def logits_of(n, v, dtype, spread=3.0, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + 31 * n + v)
    return (spread * torch.randn((n, v), generator=g, device="cuda")).to(dtype)


def reference(x, temperature=1.0):
    """(y, lse, entropy) in 64 bits; values at or below -1e38 are masked."""
    y = x.double() * scale_of(temperature)
    y = torch.where(x.double() <= -9.9e37, -torch.inf, y)
    lse = torch.logsumexp(y, -1)
    logp = y - lse[..., None]
    p = logp.exp()
    return y, lse, -torch.where(p > 0, p * logp, 0.0).sum(-1)


def close(got, want, tol, what):
    err = (got.double() - want).abs()
    bad = ~((err <= tol) | (got.double() == want) | (got.isnan() & want.isnan()))
    assert not bad.any(), (what, float(err[bad].max()), int(bad.sum()))


def check_forward(x, out, k, targets, temperature=1.0):
    logprob, entropy, lse, ids, top = out
    y, lse0, h0 = reference(x, temperature)
    close(lse, lse0, 1e-5 + E * lse0.abs(), "lse")
    spread = (y.amax(-1) - lse0).abs()
    close(entropy, h0, 1e-5 * (1 + 2 * spread + h0), "entropy")
    if targets is not None:
        v = x.shape[-1]
        inside = (targets >= 0) & (targets < v)
        want = torch.where(inside, y.gather(-1, targets.clamp(0, v - 1)[..., None])[..., 0], 0.0) - lse0
        close(logprob, want, 1e-5 + E * want.abs(), "logprob")
    order = torch.sort(x.float(), dim=-1, descending=True, stable=True).indices[..., :k]
    assert ids.shape == order.shape and torch.equal(ids, order)
    want = y.gather(-1, order) - lse0[..., None]
    # below the floor the values as they are
    raw = x.double().gather(-1, order) * scale_of(temperature) - lse0[..., None]
    want = torch.where(want == -torch.inf, raw.float().double(), want)
    close(top, want, 1e-5 + E * want.abs(), "top")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("n,v,k,temperature", [
    (1, 1, 1, 1.0), (3, 2, 2, 1.0), (5, 7, 5, 0.5), (2, 100, 100, 1.0), (4, 129, 128, 2.0), (700, 33, 4, 1.0),
    (1, 4097, 1, 1.0), (1, 32000, 20, 0.7), (3, 50257, 64, 1.0), (2, 152064, 128, 1.3), (150, 16385, 20, 1.0),
    (301, 50257, 20, 1.0), (6, 151936, 5, 30.0), (37, 40001, 100, 0.05),
])
def test_top(dtype, n, v, k, temperature):
    x = logits_of(n, v, dtype)
    g = torch.Generator(device="cuda").manual_seed(n)
    targets = torch.randint(0, v, (n,), generator=g, device="cuda")
    targets[::3] = -100
    check_forward(x, kernel_opt.fused_top_logprobs(x, targets, k, temperature), k, targets, temperature)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_top_layouts(dtype):
    base = logits_of(9, 4 * 1031, dtype).view(3, 3, 4 * 1031)
    k = 11
    for x in (base[..., 1:], base[..., 3:2000], base[:, :-1, 5:], base[:, 1:], base[1].expand(2, 3, -1),
              base[:, 0], base[0, 0], base[..., 2:3]):
        kk = min(k, x.shape[-1])
        t = torch.zeros(x.shape[:-1], dtype=torch.int64, device="cuda")
        check_forward(x, kernel_opt.fused_top_logprobs(x, t, kk), kk, t)
        out = kernel_opt.fused_top_logprobs(x, None, kk, 1.0)
        assert out[0] is None
        check_forward(x, out, kk, None)


def hard_rows(v, dtype):
    """Rows whose lists the quick bound does not give."""
    g = torch.Generator(device="cuda").manual_seed(v)
    lowest = torch.finfo(dtype).min
    rows = [torch.zeros(v), torch.full((v,), -7.0), torch.randint(-2, 3, (v,)).float(), torch.arange(v) / 64.0,
            -torch.arange(v) / 64.0, -torch.zeros(v)]
    rows = [r.cuda() for r in rows]
    rows[5][::2] = 0.0                                   # -0 and 0 are equal
    one = 2 * torch.randn(v, generator=g, device="cuda")
    few = torch.full((v,), -torch.inf, device="cuda")
    few[v // 2:v // 2 + 3] = torch.tensor([1.0, 3.0, 1.0], device="cuda")[: few[v // 2:v // 2 + 3].numel()]
    rows.append(few)                                     # a mask that leaves three
    low = torch.full((v,), lowest, device="cuda")
    low[-1] = 0.5
    rows.append(low)                                     # masked with the type's lowest value
    mix = one.clone()
    mix[1::2] = -torch.inf
    rows.append(mix)
    col = one.clone()
    col[torch.arange(v, device="cuda") // (16 // dtype.itemsize) % 256 < 3] += 40.0   # all in a few threads' columns
    rows.append(col)
    spike = one.clone()
    spike[v // 3] = 60.0
    rows.append(spike)
    tail = one.clone()
    tail[-1] = tail[0] = 20.0
    rows.append(tail)
    return torch.stack(rows).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("v,k", [(97, 20), (5003, 128), (40000, 20), (152064, 100)])
def test_top_hard_rows(dtype, v, k):
    x = hard_rows(v, dtype)
    check_forward(x, kernel_opt.fused_top_logprobs(x, None, k), k, None)
    wide = x.repeat(30, 1)  # enough rows for one block each
    check_forward(wide, kernel_opt.fused_top_logprobs(wide, None, k), k, None)


def test_top_long_rows():
    # more chunks than a thread keeps maxima for; one block a row, and eight
    for n in (300, 2):
        x = logits_of(n, 700003, torch.bfloat16)
        check_forward(x, kernel_opt.fused_top_logprobs(x, None, 50), 50, None)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("n,v", [(7, 1000), (5, 152064), (400, 9001)])
def test_rows_without_a_distribution(dtype, n, v):
    x = logits_of(n, v, dtype)
    x[0] = -torch.inf
    x[1, v // 2] = torch.nan
    x[2, v - 1] = torch.inf
    x[3, 3:] = -torch.inf                    # a distribution of three
    t = torch.arange(n, device="cuda")
    logprob, entropy, lse, ids, top = kernel_opt.fused_top_logprobs(x, t, 4)
    assert (ids[:3] == -1).all() and top[:3].isnan().all() and entropy[:3].isnan().all() and logprob[:3].isnan().all()
    assert lse[0] == -torch.inf and lse[1:3].isnan().all()
    check_forward(x[3:], (logprob[3:], entropy[3:], lse[3:], ids[3:], top[3:]), 4, t[3:])
    lp, _, _ = kernel_opt.fused_token_logprobs(x, t[:, None])
    assert torch.equal(lp[3:, 0], logprob[3:]) and lp[:3].isnan().all()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("n,v,k,temperature", [(1, 50257, 3, 1.0), (4, 1000, 0, 1.0), (6, 333, 1024, 2.0),
                                               (300, 8191, 300, 0.6), (3, 152064, 32, 1.0)])
def test_tokens(dtype, n, v, k, temperature):
    x = logits_of(n, v, dtype)
    g = torch.Generator(device="cuda").manual_seed(k)
    ids = torch.randint(-3, v + 3, (n, k), generator=g, device="cuda")
    lp, entropy, lse = kernel_opt.fused_token_logprobs(x, ids, temperature)
    y, lse0, h0 = reference(x, temperature)
    inside = (ids >= 0) & (ids < v)
    want = torch.where(inside, y.gather(-1, ids.clamp(0, v - 1)), 0.0) - lse0[:, None]
    assert lp.shape == ids.shape
    close(lp, want, 1e-5 + E * want.abs(), "logprobs")
    close(lse, lse0, 1e-5 + E * lse0.abs(), "lse")
    close(entropy, h0, 1e-5 * (1 + 2 * (y.amax(-1) - lse0).abs() + h0), "entropy")


def check_gradient(x, d, ids, g_ids, g_entropy, g_lse, temperature):
    """dL/dx against its formula in 64 bits; ids [n, K] of all lists."""
    n, v = x.shape
    y, lse, h = reference(x, temperature)
    logp = y - lse[:, None]
    p = logp.exp()
    z = lambda g: torch.zeros(n, dtype=torch.float64, device="cuda") if g is None else g.double()
    ge, gl, g = z(g_entropy), z(g_lse), g_ids.double()
    inside = (ids >= 0) & (ids < v)
    at = torch.where(inside, ids, 0)
    along = torch.where(p > 0, logp, 0.0)
    want = p * (gl[:, None] - g.sum(1, keepdim=True) - ge[:, None] * (along + h[:, None]))
    factor = gl.abs()[:, None] + g.abs().sum(1, keepdim=True) + ge.abs()[:, None] * (along.abs() + h[:, None])
    size = p * factor
    want.scatter_add_(1, at, g * inside)
    size.scatter_add_(1, at, g.abs() * inside)
    s = scale_of(temperature)
    err = (d.double() - s * want).abs()
    # a probability below fp32's normal numbers (2^-126) is taken as 0: an error of 2^-126 times its factor
    tol = U[x.dtype] * (s * want).abs() + 2e-5 * s * size + TINY[x.dtype] + 2.0 ** -126 * s * factor
    bad = ~(err <= tol)
    assert not bad.any(), (float((err - tol)[bad].max()), int(bad.sum()))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("n,v,k,temperature", [(1, 1, 1, 1.0), (5, 7, 5, 0.5), (3, 4099, 20, 1.0), (2, 152064, 128, 1.0),
                                               (600, 1003, 8, 2.0), (2, 32000, 3, 0.7)])
@pytest.mark.parametrize("which", ["all", "top", "logprob", "entropy", "lse"])
def test_top_gradient(dtype, n, v, k, temperature, which):
    x = logits_of(n, v, dtype).requires_grad_(True)
    g = torch.Generator(device="cuda").manual_seed(k)
    r = lambda *s: torch.randn(s, generator=g, device="cuda")
    targets = torch.randint(0, v, (n,), generator=g, device="cuda")
    logprob, entropy, lse, ids, top = kernel_opt.fused_top_logprobs(x, targets, k, temperature)
    assert not ids.requires_grad
    gs = {"logprob": r(n), "entropy": r(n), "lse": r(n), "top": r(n, k)}
    outs = {"logprob": logprob, "entropy": entropy, "lse": lse, "top": top}
    if which != "all":
        gs = {which: gs[which]}
    d, = torch.autograd.grad([outs[q] for q in gs], x, list(gs.values()))
    zero = torch.zeros(n, 1, device="cuda")
    g_ids = torch.cat([gs["logprob"][:, None] if "logprob" in gs else zero,
                       gs["top"] if "top" in gs else zero.expand(n, k)], 1)
    check_gradient(x.detach(), d, torch.cat([targets[:, None], ids], 1), g_ids, gs.get("entropy"), gs.get("lse"), temperature)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("temperature", [1e-4, 0.01, 0.1, 50.0])
def test_gradient_at_far_temperatures(dtype, temperature):
    # lse is thousands of times the logits' spread here: its rounding to fp32 alone would put
    # probabilities off by 2^-24 |lse|, 4e-3 and more at 1e-4
    x = logits_of(4, 5001, dtype, spread=4.0)
    x[0, :40] = x[0].max()          # equal largest ones share the mass
    x[1, 7] = x[1].max()
    x = x.requires_grad_(True)
    ids = torch.arange(12, device="cuda").expand(4, 12)
    lp, entropy, lse = kernel_opt.fused_token_logprobs(x, ids, temperature)
    g = torch.Generator(device="cuda").manual_seed(5)
    gi, ge, gl = 0.3 * torch.randn(4, 12, generator=g, device="cuda"), *(0.3 * torch.randn(2, 4, generator=g, device="cuda"))
    d, = torch.autograd.grad((lp, entropy, lse), x, (gi, ge, gl))
    check_gradient(x.detach(), d, ids, gi, ge, gl, temperature)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("n,v,k", [(3, 50, 200), (4, 50257, 32), (2, 152064, 7), (500, 517, 1024)])
def test_tokens_gradient(dtype, n, v, k):
    # tokens named many times, ids outside the vocabulary, certain rows
    x = logits_of(n, v, dtype)
    x[0, v // 2] = 30.0
    g = torch.Generator(device="cuda").manual_seed(k)
    ids = torch.randint(-2, v + 2, (n, k), generator=g, device="cuda")
    ids[:, : k // 2] = ids[:, :1]
    ids[0, -1] = v // 2
    x = x.requires_grad_(True)
    lp, entropy, lse = kernel_opt.fused_token_logprobs(x, ids, 1.0)
    gi = torch.randn(n, k, generator=g, device="cuda")
    ge = torch.randn(n, generator=g, device="cuda")
    d, = torch.autograd.grad((lp, entropy), x, (gi, ge))
    check_gradient(x.detach(), d, ids, gi, ge, None, 1.0)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_gradient_of_strided_rows(dtype):
    base = logits_of(12, 2055, dtype).view(3, 4, 2055)
    for cut in (lambda b: b[:, :-1, 3:], lambda b: b[..., 1:1028], lambda b: b[1].expand(2, 4, 2055), lambda b: b[:, 0]):
        leaf = base.clone().requires_grad_(True)
        x = cut(leaf)
        ids = torch.randint(0, x.shape[-1], (*x.shape[:-1], 5), device="cuda")
        gi = torch.randn(ids.shape, device="cuda")
        lp, entropy, lse = kernel_opt.fused_token_logprobs(x, ids)
        d, = torch.autograd.grad(lp, x, gi, retain_graph=True)
        assert d.shape == x.shape
        check_gradient(x.detach().reshape(-1, x.shape[-1]), d.reshape(-1, x.shape[-1]), ids.reshape(-1, 5),
                       gi.reshape(-1, 5), None, None, 1.0)
        whole, = torch.autograd.grad(lp, leaf, gi)
        back = torch.zeros_like(leaf, dtype=torch.float32).requires_grad_(True)
        want, = torch.autograd.grad(cut(back), back, d.float())
        close(whole, want.double(), 2 * U[dtype] * want.double().abs() + TINY[dtype], "leaf")


def test_gradient_against_differences():
    # fp32: a central difference of step h errs by h^2 / 6 of the third derivative (about 1e-6 here)
    # and by the outputs' 1e-5 over 2 h
    x = logits_of(6, 501, torch.float32, spread=1.5).requires_grad_(True)
    ids = torch.randint(0, 501, (6, 4), device="cuda")
    w = [torch.randn(6, 4, device="cuda"), torch.randn(6, device="cuda"), torch.randn(6, device="cuda")]
    top = torch.randn(6, 3, device="cuda")

    def loss(x):
        a = kernel_opt.fused_token_logprobs(x, ids, 0.8)
        b = kernel_opt.fused_top_logprobs(x, None, 3, 0.8)
        return sum((o.double() * q.double()).sum() for o, q in zip(a, w)) + (b[4].double() * top.double()).sum()

    d, = torch.autograd.grad(loss(x), x)
    h = 2.0 ** -5
    with torch.no_grad():
        for seed in range(4):
            v = torch.randn(x.shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda") * 0.3
            got = (loss(x + h * v) - loss(x - h * v)) / (2 * h)
            want = (d.double() * v.double()).sum()
            size = sum(float(q.abs().sum()) for q in w) + float(top.abs().sum())
            assert abs(float(got - want)) <= size * (1e-5 / h + 4 * h * h), (float(got), float(want))


def test_rows_without_upstream_gradient():
    x = logits_of(8, 3001, torch.bfloat16)
    x[1] = torch.nan
    x[2] = -torch.inf
    x = x.requires_grad_(True)
    ids = torch.zeros(8, 2, dtype=torch.int64, device="cuda")
    lp, entropy, lse = kernel_opt.fused_token_logprobs(x, ids)
    g = torch.ones_like(lp)
    g[1:3] = 0
    d, = torch.autograd.grad(lp, x, g, retain_graph=True)
    assert (d[1:3] == 0).all() and d.isfinite().all() and (d[0] != 0).any()
    d, = torch.autograd.grad(lp, x, torch.ones_like(lp))
    assert d[1:3].isnan().all()


def test_only_what_is_asked_has_a_gradient():
    x = logits_of(4, 100, torch.float32)
    out = kernel_opt.fused_top_logprobs(x, None, 3)
    assert not any(o.requires_grad for o in out[1:])
    x.requires_grad_(True)
    with torch.no_grad():
        assert not kernel_opt.fused_top_logprobs(x, None, 3)[4].requires_grad
    out = kernel_opt.fused_top_logprobs(x, None, 3)
    d, = torch.autograd.grad(out[4].sum(), x, create_graph=False)
    with pytest.raises(RuntimeError, match="second derivative"):
        out = kernel_opt.fused_top_logprobs(x, None, 3)
        torch.autograd.grad(out[4].sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="forward AD"):
        import torch.autograd.forward_ad as fw
        with fw.dual_level():
            dual = fw.make_dual(x.detach(), torch.ones_like(x))
            kernel_opt.fused_token_logprobs(dual, torch.zeros(4, 1, dtype=torch.int64, device="cuda"))


def test_empty():
    x = torch.empty(0, 100, device="cuda", requires_grad=True)
    out = kernel_opt.fused_top_logprobs(x, torch.empty(0, dtype=torch.int64, device="cuda"), 3)
    assert out[0].shape == (0,) and out[3].shape == (0, 3)
    d, = torch.autograd.grad(out[4].sum(), x)
    assert d.shape == x.shape
    lp, _, _ = kernel_opt.fused_token_logprobs(torch.zeros(2, 9, device="cuda"), torch.empty(2, 0, dtype=torch.int64, device="cuda"))
    assert lp.shape == (2, 0)


def test_refusals():
    x = torch.zeros(2, 9, device="cuda")
    t = torch.zeros(2, dtype=torch.int64, device="cuda")
    for k in (0, 10, -1):
        with pytest.raises((ValueError, RuntimeError), match="k must be"):
            kernel_opt.fused_top_logprobs(x, t, k)
    with pytest.raises(RuntimeError, match="k must be"):
        kernel_opt.fused_top_logprobs(torch.zeros(1, 1000, device="cuda"), None, 129)
    for bad in (0.0, -1.0, float("nan"), float("inf"), 1e-31):
        with pytest.raises(RuntimeError, match="temperature"):
            kernel_opt.fused_top_logprobs(x, t, 2, bad)
    with pytest.raises(RuntimeError, match="int64"):
        kernel_opt.fused_top_logprobs(x, t.int(), 2)
    with pytest.raises(ValueError, match="shaped like"):
        kernel_opt.fused_top_logprobs(x, t[:1], 2)
    with pytest.raises(ValueError, match="device"):
        kernel_opt.fused_top_logprobs(x, t.cpu(), 2)
    with pytest.raises(ValueError, match="leading dimensions"):
        kernel_opt.fused_token_logprobs(x, t)
    with pytest.raises(RuntimeError, match="at most 1024"):
        kernel_opt.fused_token_logprobs(x, torch.zeros(2, 1025, dtype=torch.int64, device="cuda"))
    with pytest.raises(RuntimeError, match="dtype"):
        kernel_opt.fused_top_logprobs(x.double(), t, 2)
    with pytest.raises(RuntimeError, match="contiguous along the vocab"):
        kernel_opt.fused_top_logprobs(x.t().contiguous().t(), t, 2)


def test_captured_and_on_another_stream():
    x = logits_of(6, 20000, torch.bfloat16)
    t = torch.arange(6, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    leaf = x.clone().requires_grad_(True)
    ge = torch.randn(6, device="cuda")
    gt = torch.randn(6, 5, device="cuda")

    def step():
        out = kernel_opt.fused_top_logprobs(leaf, t, 5, 0.9)
        return (*out, *torch.autograd.grad((out[1], out[4]), leaf, (ge, gt)))

    with torch.cuda.stream(side):
        for _ in range(3):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in (3, 4):
        with torch.no_grad():
            leaf.copy_(logits_of(6, 20000, torch.bfloat16, seed=seed))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, step()):
            assert torch.equal(a, b)


def test_the_same_bits_every_time():
    x = logits_of(200, 50257, torch.float16).requires_grad_(True)
    t = torch.arange(200, device="cuda")

    def once():
        out = kernel_opt.fused_top_logprobs(x, t, 64, 0.7)
        return (*out, *torch.autograd.grad((out[0].sum() + out[4].sum(),), x))

    first = once()
    for _ in range(5):
        for a, b in zip(first, once()):
            assert torch.equal(a, b)
