"""Token sampling against the definition in 64 bits.

The operator defines y = x * fp32(1/T) and d = y - max y in fp32; the reference takes those and
computes weights and sums in 64 bits.  The kernel's weights are expf's, within 2 units of 2^-23
of the exact ones, and its sums err by far less, so any share of the mass is within D = 2^-21
of the reference's.  A token is right if u lies within D of its interval; where a cut (top-p,
min-p) is itself within D of an element, both sides of the cut are right.  Log-probabilities:
D, plus the rounding of the result to fp32.
"""
import math

import pytest
import torch

import kernel_opt

pytestmark = pytest.mark.gpu

D = 2.0 ** -21
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def per_row(v, n):
    return v.tolist() if isinstance(v, torch.Tensor) else [v] * n


def check(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    tok, lp, kp = kernel_opt.sample_tokens(logits, u, temperature, top_k, top_p, min_p)
    n, v = logits.shape
    assert tok.dtype == torch.int64 and lp.dtype == kp.dtype == torch.float32
    T, K, P, Q = (per_row(s, n) for s in (temperature, top_k, top_p, min_p))
    for r in range(n):
        t = T[r]
        s = torch.tensor(1.0 / t if t > 0 else 1.0).float().item()
        y = logits[r].float() * s
        m = y.max()
        d = y - m
        w = d.double().exp()
        total = w.sum()
        # order: value downwards, index upwards
        order = torch.sort(d, descending=True, stable=True).indices
        k = 1 if t == 0 else K[r] if 0 < K[r] < v else v
        ws = w[order][:k]
        cum = ws.cumsum(0)
        cuts = [len(ws), len(ws)]  # the kept counts that are right: least, most
        p = float(torch.tensor(P[r]).float()) if t else 1.0
        if p < 1:
            before = cum - ws
            for i, slack in enumerate((-D, D)):
                cuts[i] = min(cuts[i], max(1, int((before < (p + slack) * cum[-1]).sum())))
        q = min(float(torch.tensor(Q[r]).float()), 1.0) if t else 0.0
        if q > 0:
            for i, slack in enumerate((D, -D)):
                cuts[i] = min(cuts[i], max(1, int((ws >= q * (1 + slack)).sum())))
        token = int(tok[r])
        assert 0 <= token < v, (r, token)
        ok = False
        for kept in {cuts[0], cuts[1]}:
            idx = torch.sort(order[:kept]).values
            c = w[idx].cumsum(0)
            C = c[-1]
            at = int(torch.searchsorted(idx, torch.tensor(token, device=idx.device)))
            if at >= len(idx) or int(idx[at]) != token:
                continue
            lo = float(c[at] - w[token]) / float(C)
            hi = float(c[at]) / float(C)
            want_k = float(d[token].double() - C.log())
            if lo - D <= float(u[r]) <= hi + D and float(w[token]) > 0 and \
                    abs(float(kp[r]) - want_k) <= D + 2.0 ** -23 * abs(want_k):
                ok = True
        assert ok, (r, token, cuts, float(u[r]))
        want = float(d[token].double() - total.log())
        assert abs(float(lp[r]) - want) <= D + 2.0 ** -23 * abs(want), (r, float(lp[r]), want)
    return tok


def normal(n, v, dtype, sigma=3.0, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + 31 * n + v)
    return torch.randn(n, v, generator=g, device="cuda").mul_(sigma).to(dtype)


def uniform(n, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed + n)
    u = torch.rand(n, generator=g, device="cuda")
    if n > 2:
        u[0], u[1] = 0.0, 1.0 - 2.0 ** -24
    return u


SETTINGS = [dict(), dict(temperature=0.7), dict(top_k=1), dict(top_k=50), dict(top_k=5000),
            dict(top_p=0.9), dict(top_p=0.0), dict(top_p=0.999), dict(min_p=0.05), dict(min_p=1.0),
            dict(temperature=1.3, top_k=40, top_p=0.8, min_p=0.02), dict(top_k=3000, top_p=0.95),
            dict(temperature=0.0)]


@pytest.mark.parametrize("kw", SETTINGS, ids=str)
@pytest.mark.parametrize("n,v,dtype", [
    (1, 1, torch.bfloat16), (3, 2, torch.float32), (5, 7, torch.float16), (4, 8, torch.bfloat16),
    (4, 1000, torch.float32), (6, 1003, torch.bfloat16), (5, 32000, torch.bfloat16),
    (4, 50257, torch.float16), (3, 128256, torch.float32), (3, 152064, torch.bfloat16)])
def test_settings(n, v, dtype, kw):
    check(normal(n, v, dtype), uniform(n), **kw)


@pytest.mark.parametrize("sigma", [0.0, 1e-4, 0.3, 1.0, 8.0, 40.0])
@pytest.mark.parametrize("dtype", DTYPES)
def test_flat_and_peaked(dtype, sigma):
    """Flat rows need the selection (bins with more elements than a list holds, ties), peaked
    ones a single entry."""
    x = normal(4, 40000, dtype, sigma)
    u = uniform(4)
    for kw in (dict(top_p=0.9), dict(top_p=0.37), dict(top_k=3000), dict(top_k=20000, top_p=0.5),
               dict(top_k=700), dict(min_p=0.5), dict()):
        check(x, u, **kw)


def test_ties_go_to_the_lowest_index():
    v = 30000
    x = torch.zeros(4, v, device="cuda")
    u = torch.tensor([0.0, 0.25, 0.5, 0.999], device="cuda")
    for dtype in DTYPES:
        for k in (1, 7, 2500):
            tok = check(x.to(dtype), u, top_k=k)
            assert tok.tolist() == [min(int(float(a) * k), k - 1) for a in u]
        tok = check(x.to(dtype), u, top_p=0.5)
        assert (tok < v // 2).all()
    # two values: 4000 high ones at odd places, the rest one lower
    x = torch.full((2, v), -1.0, device="cuda")
    x[:, 1:8001:2] = 0.0
    tok = check(x, torch.tensor([0.9999, 0.5], device="cuda"), top_k=3000)
    assert tok.tolist() == [2 * 2999 + 1, 2 * 1500 + 1]
    check(x, torch.tensor([0.9999, 0.5], device="cuda"), top_k=9000)
    assert check(x, torch.tensor([0.3, 0.5], device="cuda"), temperature=0.0).tolist() == [1, 1]


@pytest.mark.parametrize("dtype", DTYPES)
def test_every_share_of_u_draws_its_token(dtype):
    """4096 evenly spaced numbers over one row (a view with a row stride of 0): each token
    comes up as often as its probability says, within one, and in the order of the ids."""
    n, v = 4096, 300
    row = normal(1, v, dtype, 1.5)
    u = (torch.arange(n, device="cuda") + 0.5) / n
    for kw in (dict(), dict(top_k=20), dict(top_p=0.8), dict(min_p=0.1)):
        tok, _, kp = kernel_opt.sample_tokens(row.expand(n, v), u, **kw)
        assert (tok[1:] >= tok[:-1]).all()
        count = torch.bincount(tok, minlength=v).double()
        seen = count > 0
        prob = torch.zeros(v, dtype=torch.float64, device="cuda").scatter_(0, tok, kp.double().exp())
        assert ((count - n * prob).abs()[seen] <= 1 + n * D).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_rows(dtype):
    n, v = 8, 5003
    x = normal(n, v, dtype)
    low = torch.finfo(dtype).min
    x[0, 10:] = float("-inf")
    x[1, :] = float("-inf")
    x[1, 4321] = -5.0
    x[2, :] = float("-inf")       # nothing is left
    x[3, ::2] = low               # masked by the type's lowest value
    x[4, :] = low                 # all equal, all lowest
    x[5, 77] = float("nan")
    x[6, 5002] = float("inf")
    x[7, :5000] = float("-inf")
    u = uniform(n)
    good = [0, 1, 3, 4, 7]
    for kw in (dict(), dict(top_k=30), dict(top_p=0.9), dict(top_k=4000), dict(min_p=0.1), dict(temperature=0.0),
               dict(top_k=4000, top_p=0.6)):
        tok, lp, kp = kernel_opt.sample_tokens(x, u, **kw)
        for r in (2, 5, 6):
            assert int(tok[r]) == -1 and math.isnan(float(lp[r])) and math.isnan(float(kp[r]))
        check(x[good], u[good], **kw)
        assert int(tok[1]) == 4321 and int(tok[7]) >= 5000


def test_extreme_values():
    u = uniform(4)
    x = normal(4, 9001, torch.float32)
    check(x * 1e30, u, top_p=0.9)
    check(x * 1e-38, u, top_p=0.5)         # differences below fp32's normal numbers
    check(x * 1e-38, u, top_k=4321)
    check(x + 1e6, u, top_p=0.7)           # few distinct values
    check(x * 1e-3, u, temperature=1e-3, top_k=100)
    check(x, u, temperature=100.0, top_p=0.9)
    y = x.clone()
    y[:, 123] = 300.0                      # every other weight is zero
    check(y, u)
    check(y, u, top_k=5000, top_p=0.99)
    y[:, 200:] = -3e38
    y[:, 100] = 3e38                       # the range overflows fp32
    check(y, u, top_p=0.9)
    check(y, u, top_k=3000)


def test_settings_per_row():
    n, v = 24, 32000
    x, u = normal(n, v, torch.bfloat16), uniform(n)
    g = torch.Generator(device="cuda").manual_seed(3)
    pick = lambda vals, dt: torch.tensor(vals, dtype=dt, device="cuda")[
        torch.randint(0, len(vals), (n,), generator=g, device="cuda")]
    t = pick([0.0, 0.5, 1.0, 1.2], torch.float32)
    k = pick([0, 1, 50, 900, 4000], torch.int32)
    p = pick([1.0, 0.3, 0.9, 2.0], torch.float32)
    q = pick([0.0, 0.0, 0.1], torch.float32)
    check(x, u, t, k, p, q)
    # the same row by row with numbers
    tok, lp, kp = kernel_opt.sample_tokens(x, u, t, k, p, q)
    for r in range(0, n, 5):
        one = kernel_opt.sample_tokens(x[r:r + 1], u[r:r + 1], float(t[r]), int(k[r]), float(p[r]), float(q[r]))
        assert int(one[0]) == int(tok[r])
    bad = t.clone()
    bad[3], bad[4], bad[5] = -1.0, float("nan"), float("inf")
    tok2, lp2, _ = kernel_opt.sample_tokens(x, u, bad, k, p, q)
    assert (tok2[3:6] == -1).all() and torch.isnan(lp2[3:6]).all()
    assert torch.equal(tok2[6:], tok[6:])


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts_and_batches_give_the_same_token(dtype):
    """A row's result depends on its values alone: not on its address, its row stride, the
    number of rows (which sets how many blocks share a row) or the leading dimensions."""
    n, v = 6, 50257
    x, u = normal(n, v, dtype), uniform(n)
    for kw in (dict(), dict(top_k=50, top_p=0.9), dict(top_p=0.95), dict(top_k=2500)):
        want = kernel_opt.sample_tokens(x, u, **kw)
        wide = torch.zeros(n, v + 11, dtype=dtype, device="cuda")
        for off in (0, 1, 2, 5):
            view = wide[:, off:off + v]
            view.copy_(x)
            got = kernel_opt.sample_tokens(view, u, **kw)
            assert torch.equal(got[0], want[0])
            torch.testing.assert_close(got[1], want[1], rtol=2.0 ** -22, atol=2.0 ** -22)
        many = kernel_opt.sample_tokens(x.repeat(60, 1), u.repeat(60), **kw)
        assert torch.equal(many[0].view(60, n), want[0].expand(60, n))
        got = kernel_opt.sample_tokens(x.view(2, 3, v), u.view(2, 3), **kw)
        assert got[0].shape == (2, 3) and torch.equal(got[0].view(-1), want[0])


@pytest.mark.parametrize("dtype,v", [(torch.bfloat16, 800001), (torch.float32, 400003)])
def test_rows_longer_than_shared_memory(dtype, v):
    x, u = normal(3, v, dtype, 2.0), uniform(3)
    for kw in (dict(), dict(top_k=50), dict(top_p=0.9), dict(top_k=30000, top_p=0.8)):
        check(x, u, **kw)


def test_logprob_is_k1s():
    x, u = normal(16, 32000, torch.bfloat16), uniform(16)
    tok, lp, _ = kernel_opt.sample_tokens(x, u)
    want, _, _ = kernel_opt.fused_logprob_entropy(x, tok)
    torch.testing.assert_close(lp, want, rtol=0, atol=2e-5)


def test_other_stream_and_graph():
    x, u = normal(8, 32000, torch.bfloat16), uniform(8)
    want = kernel_opt.sample_tokens(x, u, top_p=0.9)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = kernel_opt.sample_tokens(x, u, top_p=0.9)
    torch.cuda.current_stream().wait_stream(st)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = kernel_opt.sample_tokens(x, u, top_p=0.9)
    u.copy_(uniform(8, seed=9))
    g.replay()
    assert torch.equal(out[0], kernel_opt.sample_tokens(x, u, top_p=0.9)[0])


def test_no_rows():
    out = kernel_opt.sample_tokens(torch.empty(0, 100, device="cuda"), torch.empty(0, device="cuda"))
    assert all(o.shape == (0,) for o in out)


def test_refusals():
    x, u = normal(4, 100, torch.float32), uniform(4)
    f = kernel_opt.sample_tokens
    with pytest.raises(ValueError, match="u must be shaped"):
        f(x, u[:3])
    with pytest.raises(RuntimeError, match="temperature must be"):
        f(x, u, temperature=-1.0)
    with pytest.raises(RuntimeError, match="temperature must be"):
        f(x, u, temperature=float("nan"))
    with pytest.raises(RuntimeError, match="min_p must be"):
        f(x, u, min_p=1.5)
    with pytest.raises(RuntimeError, match="top_p must be"):
        f(x, u, top_p=-0.1)
    with pytest.raises(ValueError, match="top_k must be a number or a tensor"):
        f(x, u, top_k=torch.ones(3, device="cuda"))
    with pytest.raises(RuntimeError, match="bf16, fp16, or fp32"):
        f(x.double(), u)
    with pytest.raises(RuntimeError, match="vocab must be"):
        f(x[:, :0], u)
    with pytest.raises(ValueError, match="CUDA"):
        f(x.cpu(), u.cpu())


@pytest.mark.parametrize("kw", [dict(top_k=50), dict(top_p=0.9), dict(top_k=3000, min_p=0.001)], ids=str)
def test_many_rows_cut_into_any_number_of_parts(kw):
    """Rows in 3, 5, 6 or 7 parts (taken where there are many rows) give what the same rows give
    alone, in the power of two of parts that few rows take."""
    for v, dtype in ((128256, torch.bfloat16), (100001, torch.float32), (128256, torch.float32),
                     (152063, torch.float32)):
        base = (torch.randn(8, v, device="cuda") * 3).to(dtype)
        u = torch.rand(320, device="cuda")
        rows = base.repeat(40, 1)
        tok, lp, kp = kernel_opt.sample_tokens(rows, u, **kw)
        for at in (0, 7, 163, 319):
            t, l, k = kernel_opt.sample_tokens(rows[at:at + 1], u[at:at + 1], **kw)
            assert t == tok[at]
            assert (l - lp[at]).abs() <= 2 ** -22 * l.abs() and (k - kp[at]).abs() <= 2 ** -22 * k.abs() + 2 ** -24
