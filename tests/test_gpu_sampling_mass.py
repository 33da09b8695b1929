"""Sampling where light elements decide: shares of the mass far below those that the other tests
resolve, against sums in 64 bits of the same fp32 weights (torch.exp and the kernel's expf are one
function, so the weights are equal and only the sums are compared).
"""
import pytest
import torch

import kernel_opt

pytestmark = pytest.mark.gpu


def check(x, u, slack, top_k=0, top_p=1.0):
    """Every token is one that sums within `slack` (a share of the mass) of the exact ones allow:
    kept, where the nucleus may end anywhere within `slack` of its share, and at u in the order
    of ids."""
    tok = kernel_opt.sample_tokens(x, u, 1.0, top_k, top_p)[0]
    n, v = x.shape
    p = float(torch.tensor(top_p).float())
    for r in range(n):
        y = x[r].float()
        w = torch.exp(y - y.max()).double()
        order = torch.sort(y, descending=True, stable=True).indices  # by y: weights may be equal where y is not
        ws = w[order]
        kept = min(top_k, v) if top_k > 0 else v
        cum = ws[:kept].cumsum(0)
        if p < 1:
            kept = max(1, int((cum - ws[:kept] < (p + slack) * cum[-1]).sum()))
        token = int(tok[r])
        ids = torch.sort(order[:kept]).values
        c = w[ids].cumsum(0)
        at = int(torch.searchsorted(ids, torch.tensor(token, device=ids.device)))
        assert at < kept and int(ids[at]) == token, (r, token, "is not kept")
        C, share = float(c[-1]), float(u[r]) * float(c[-1])
        assert float(c[at] - w[token]) - 3 * slack * C <= share <= float(c[at]) + 3 * slack * C, (r, token)
    return tok


def light_row(n, v, dtype, lo, hi, seed=0):
    """n equal rows: all but the last element uniform in [lo, hi), the last one 0."""
    g = torch.Generator(device="cuda").manual_seed(seed + v)
    row = torch.empty(v, device="cuda").uniform_(lo, hi, generator=g)
    row[-1] = 0.0
    return row.to(dtype).expand(n, v)


@pytest.mark.parametrize("v,dtype,lo,hi,below_one", [
    (152064, torch.float32, -28.55, -28.45, 2.0 ** -24), (152064, torch.float32, -29.0, -28.0, 2.0 ** -24),
    (152064, torch.float16, -28.55, -28.4, 2.0 ** -24), (152064, torch.bfloat16, -28.7, -28.2, 2.0 ** -24),
    (400003, torch.float32, -29.0, -28.8, 2.0 ** -23), (400003, torch.float32, -28.95, -28.9, 2.0 ** -23),
    (50257, torch.float32, -27.5, -27.2, 2.0 ** -24), (4001, torch.float32, -25.0, -24.5, 2.0 ** -24)])
def test_a_nucleus_that_ends_among_the_lightest(v, dtype, lo, hi, below_one):
    """top-p next to 1: the list of the crossing bin holds only weights of about e^-28."""
    n = 24
    x = light_row(n, v, dtype, lo, hi)
    light = float(torch.exp(x[0, :-1].float()).double().sum())
    u = torch.linspace(0, 1.2 * light, n, device="cuda")
    for kw in (dict(top_p=1 - below_one), dict(top_p=1 - below_one, top_k=v // 2), dict(top_p=1 - 2 * below_one)):
        check(x, u, 1e-9, **kw)


# Rows (id: logit, the others masked) of two equal elements and a few whose weights are about half of
# 2^-52: u = 1/2 falls on a prefix that two orders of adding round to either side of it.
TIES = [{2: 0.0, 33: -36.75, 37: -36.75, 42: -38.375, 47: -36.75, 900: 0.0},
        {5: -38.5, 12: 0.0, 33: -38.5, 43: -36.875, 900: 0.0},
        {10: -38.0, 14: 0.0, 16: -36.375, 34: -35.75, 37: -35.25, 41: -38.25, 900: 0.0},
        {4: -38.75, 6: -38.375, 18: 0.0, 41: -37.0, 45: -37.0, 900: 0.0},
        {10: 0.0, 32: -38.5, 36: -37.75, 44: -37.0, 900: 0.0}]


@pytest.mark.parametrize("kw", [dict(), dict(min_p=1e-18)], ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_a_prefix_that_rounds_to_either_side_of_the_target(dtype, kw):
    x = torch.full((len(TIES), 1024), float("-inf"))
    for r, row in enumerate(TIES):
        for i, y in row.items():
            x[r, i] = y
    x = x.to(dtype).cuda()
    tok, lp, kp = kernel_opt.sample_tokens(x, torch.full((len(TIES),), 0.5, device="cuda"), **kw)
    for r, row in enumerate(TIES):
        # any element between the two heavy ones (their ends included): the masses there differ by 2^-51
        assert int(tok[r]) in row, (r, int(tok[r]))
        assert abs(float(lp[r]) - (row[int(tok[r])] - 0.6931472)) < 1e-5 and abs(float(kp[r] - lp[r])) < 1e-6


# Sums are right to a few 1e-13 of the mass (a list's to 2^-40), so a u whose share lies NEAR[0] or
# more from every prefix draws what sums in 64 bits draw; those tried lie within NEAR[1] of one.
NEAR = (4e-12, 4e-11)


def near_boundaries(w):
    """fp32 numbers u in [1/4, 1) whose distance from a prefix of the weights w (as a share of their
    sum) is in NEAR, and the tokens that they draw."""
    c = w.double().cumsum(-1)
    c = c / c[-1]
    c = c[(c >= 0.25) & (c < 1 - 1e-6)]
    u = c.float()
    d = (u.double() - c).abs()
    u = u[(d > NEAR[0]) & (d < NEAR[1])]
    full = w.double().cumsum(-1)
    share = u.double() * full[-1]
    at = torch.searchsorted(full, share, right=True)
    gap = torch.minimum((full[at] - share).abs(), (share - full[at - 1]).abs()) / full[-1]
    return u[gap > NEAR[0]], at[gap > NEAR[0]]


@pytest.mark.parametrize("v,dtype,peak,sigma", [
    (152063, torch.float32, 12.0, 0.5), (152063, torch.bfloat16, 12.0, 0.5), (128256, torch.float16, 10.0, 1.0),
    (152064, torch.float32, 0.0, 3.0), (400003, torch.float32, 14.0, 0.5)])
def test_shares_are_right_at_any_address_and_in_any_batch(v, dtype, peak, sigma):
    """One heavy element over a heavy tail of light ones, at addresses that are not all alike to a
    16-byte vector, in batches that cut rows into 8, 4 or 2 parts or none."""
    g = torch.Generator(device="cuda").manual_seed(v)
    row = torch.randn(v, generator=g, device="cuda").mul_(sigma)
    if peak:
        row[v // 7] = peak
    row = row.to(dtype)
    y = row.float()
    u, want = near_boundaries(torch.exp(y - y.max()))
    assert len(u) >= 20, len(u)
    buf = torch.empty(v + 8, dtype=dtype, device="cuda")
    for shift in (0, 1, 3):
        buf[shift:shift + v] = row
        x = buf[shift:shift + v]
        for n in (1, 20, 300):
            for at in range(0, min(len(u), 4 * n), n):
                k = len(u[at:at + n])
                tok = kernel_opt.sample_tokens(x.expand(n, v)[:k], u[at:at + n])[0]
                assert torch.equal(tok, want[at:at + n]), (shift, n, int((tok != want[at:at + n]).sum()))


@pytest.mark.parametrize("kw", [dict(top_k=1000), dict(top_k=1000, top_p=0.95), dict(top_k=5000), dict(top_p=0.9)], ids=str)
@pytest.mark.parametrize("sigma", [1.0, 3.0])
def test_shares_of_what_is_kept_are_right_in_any_batch(sigma, kw):
    """The same behind filters, whose threshold comes from a list or from the whole row."""
    n, v = 200, 50257
    g = torch.Generator(device="cuda").manual_seed(int(sigma))
    x = torch.randn(n, v, generator=g, device="cuda").mul_(sigma)
    u, want = torch.full((n,), 0.5, device="cuda"), torch.full((n,), -1, device="cuda")
    for r in range(n):
        w = torch.exp(x[r] - x[r].max())
        order = torch.sort(x[r], descending=True, stable=True).indices
        ws = w[order].double()
        kept = kw.get("top_k", v)
        if "top_p" in kw:
            cum = ws[:kept].cumsum(0)
            kept = max(1, int((cum - ws[:kept] < float(torch.tensor(kw["top_p"])) * cum[-1]).sum()))
        ids = torch.sort(order[:kept]).values
        some, at = near_boundaries(w[ids])
        if len(some):
            u[r], want[r] = some[0], ids[at[0]]
    hit = want >= 0
    assert int(hit.sum()) >= 10
    tok = kernel_opt.sample_tokens(x, u, **kw)[0]
    assert torch.equal(tok[hit], want[hit]), int((tok != want)[hit].sum())
    for r in torch.nonzero(hit)[:20, 0].tolist():
        assert int(kernel_opt.sample_tokens(x[r:r + 1], u[r:r + 1], **kw)[0]) == int(want[r])


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("temperature", [0.01, 0.3, 0.7, 1.3, 5.0])
def test_log_probabilities_are_of_the_rounded_quotients(dtype, temperature):
    """y = x * fp32(1 / T) is rounded before the maximum is taken from it: a token that is certain has
    the log-probability 0 however large y is, and every other one's is right to fp32's rounding
    (2^-24 of it, one more for the sum's logarithm) and the weights' 2^-21."""
    s = torch.tensor(1.0 / temperature).float()
    x = torch.rand(64, 1, device="cuda").mul_(100).to(dtype)
    u = torch.rand(64, device="cuda")
    for kw in (dict(), dict(top_k=5, min_p=1e-3), dict(min_p=1e-3)):
        _, lp, kp = kernel_opt.sample_tokens(x, u, temperature, **kw)
        assert not lp.any() and not kp.any()
    x = torch.randn(64, 5003, device="cuda").mul_(4).add_(60).to(dtype)
    for kw in (dict(), dict(min_p=1e-6), dict(top_k=3000), dict(top_p=0.99)):
        tok, lp, _ = kernel_opt.sample_tokens(x, u, temperature, **kw)
        y = x.float() * s.cuda()
        d = (y - y.amax(1, keepdim=True)).double()
        want = torch.log_softmax(d, 1).gather(1, tok[:, None])[:, 0]
        assert ((lp.double() - want).abs() <= 2.0 ** -23 * want.abs() + 2.0 ** -21).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("temperature", [0.37, 0.7, 1.3])
def test_shares_at_a_temperature(dtype, temperature):
    """The weights are those of the rounded y: with y rounded or not, shares differ by 1e-7 of them."""
    v = 152064
    g = torch.Generator(device="cuda").manual_seed(int(100 * temperature))
    x = torch.randn(1, v, generator=g, device="cuda").mul_(2).to(dtype)
    y = x[0].float() * torch.tensor(1.0 / temperature).float().cuda()
    u, want = near_boundaries(torch.exp(y - y.max()))
    assert len(u) >= 20
    for kw in (dict(), dict(min_p=1e-30)):
        tok = kernel_opt.sample_tokens(x.expand(len(u), v), u, temperature, **kw)[0]
        assert torch.equal(tok, want), int((tok != want).sum())
