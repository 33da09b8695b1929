"""Sampling where light elements decide: shares of the mass far below those that the other tests
resolve, against sums in 64 bits of the same fp32 weights (torch.exp and the kernel's expf are one
function, so the weights are equal and only the sums are compared).
"""
import pytest
import torch

import kernel_opt

pytestmark = pytest.mark.gpu


def check(x, u, slack, scale=1.0, top_k=0, top_p=1.0, tokens=None):
    """Every token is one that sums within `slack` (a share of the mass) of the exact ones allow:
    kept, where the nucleus may end anywhere within `slack` of its share, and at u in the order
    of ids."""
    tok = kernel_opt.sample_tokens(x, u, 1.0, top_k, top_p)[0] if tokens is None else tokens
    n, v = x.shape
    p = float(torch.tensor(top_p).float())
    for r in range(n):
        y = x[r].float()
        w = torch.exp(y - y.max()).double()
        ws, order = torch.sort(w, descending=True, stable=True)
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
