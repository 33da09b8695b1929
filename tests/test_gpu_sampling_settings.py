"""Settings of single rows that mean nothing: such a row gives token -1 and NaN, as one with a bad
temperature does, and the rows beside it are as they were."""
import pytest
import torch

import kernel_opt

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("sigma", [0.0, 0.3, 3.0])
@pytest.mark.parametrize("what,bad", [("top_p", [NAN, -0.5, -INF]), ("min_p", [NAN, -0.1, 1.5, INF, -INF]),
                                      ("temperature", [NAN, -1.0, INF])])
def test_rows_with_a_setting_that_means_nothing(what, bad, sigma):
    n, v = 2 * len(bad) + 1, 40000
    g = torch.Generator(device="cuda").manual_seed(7)
    x = torch.randn(n, v, generator=g, device="cuda").mul_(sigma)
    u = torch.rand(n, generator=g, device="cuda")
    good = {"temperature": [1.0, 0.0], "top_p": [0.9, 1.5, 0.0], "min_p": [0.05, 0.0, 1.0]}[what]
    vals = [b for i, v0 in enumerate(bad) for b in (good[i % len(good)], v0)] + [good[0]]
    rows = torch.tensor(vals, device="cuda")
    for kw in (dict(), dict(top_k=30), dict(top_k=5000)):
        tok, lp, kp = kernel_opt.sample_tokens(x, u, **{what: rows}, **kw)
        assert (tok[1::2] == -1).all() and torch.isnan(lp[1::2]).all() and torch.isnan(kp[1::2]).all(), tok.tolist()
        for r in range(0, n, 2):
            one = kernel_opt.sample_tokens(x[r:r + 1], u[r:r + 1], **{what: vals[r]}, **kw)
            assert int(one[0]) == int(tok[r]) >= 0
            assert float(one[1]) == float(lp[r]) and float(one[2]) == float(kp[r])


def test_a_greedy_row_with_a_bad_filter():
    x = torch.randn(2, 500, device="cuda")
    u = torch.rand(2, device="cuda")
    tok, lp, _ = kernel_opt.sample_tokens(x, u, temperature=0.0, min_p=torch.tensor([NAN, 0.0], device="cuda"))
    assert int(tok[0]) == -1 and torch.isnan(lp[0]) and int(tok[1]) == int(x[1].argmax())


def test_top_k_beyond_32_bits():
    """A 64-bit top_k above the vocabulary is off, not what its low 32 bits say."""
    x = torch.randn(4, 3000, device="cuda")
    u = torch.full((4,), 0.999, device="cuda")
    want = kernel_opt.sample_tokens(x, u)
    k = torch.tensor([2 ** 32 + 1, 2 ** 31, 2 ** 62, -2 ** 40 + 1], device="cuda")
    got = kernel_opt.sample_tokens(x, u, top_k=k)
    assert torch.equal(got[0], want[0]) and torch.equal(got[2], got[1])
    got = kernel_opt.sample_tokens(x, u, top_k=2 ** 32 + 1)
    assert torch.equal(got[0], want[0])


def test_a_top_k_that_is_no_number():
    x, u = torch.randn(1, 100, device="cuda"), torch.rand(1, device="cuda")
    with pytest.raises(ValueError, match="top_k must be"):
        kernel_opt.sample_tokens(x, u, top_k=NAN)
