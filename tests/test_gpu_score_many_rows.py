"""Log-probabilities of lists over as many rows as take the forward's instance for many rows (six per SM and
more, which has fewer threads a row), and over the numbers of rows around that border: the same checks as
for few rows (tolerances: test_gpu_score)."""
import ctypes

import pytest
import torch

import kernel_opt
from _helpers import WAIT_TEST_LIB
from test_gpu_score import DTYPES, check_forward, check_gradient, close, hard_rows, logits_of, reference

pytestmark = pytest.mark.gpu


def sms():
    return torch.cuda.get_device_properties(0).multi_processor_count


def threads_of(rows):
    return ctypes.CDLL(WAIT_TEST_LIB).k1_test_score_threads(ctypes.c_int64(rows), sms())


def test_border():
    assert [threads_of(6 * sms() + d) for d in (-1, 0, 5)] == [256, 128, 128]


# one chunk, a few, odd widths, and more chunks than a thread keeps maxima for (32 of 512 vectors)
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("more", [-1, 0, 5])
@pytest.mark.parametrize("v,k,temperature", [(7, 7, 1.0), (1000, 128, 0.5), (4099, 20, 1.0), (50257, 64, 0.8), (140001, 20, 1.0)])
def test_top(dtype, more, v, k, temperature):
    n = 6 * sms() + more
    if dtype == torch.float32:
        v = min(v, 70001)  # more than 32 chunks of this type
    x = logits_of(n, v, dtype)
    targets = torch.randint(0, v, (n,), device="cuda")
    targets[::3] = -100
    check_forward(x, kernel_opt.fused_top_logprobs(x, targets, k, temperature), k, targets, temperature)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("v,k", [(97, 20), (5003, 128), (40000, 20), (50257, 100)])
def test_hard_rows(dtype, v, k):
    x = hard_rows(v, dtype)
    x = x.repeat(-(-6 * sms() // len(x)), 1)
    assert threads_of(len(x)) == 128
    check_forward(x, kernel_opt.fused_top_logprobs(x, None, k), k, None)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("v", [1001, 50257])
def test_rows_without_a_distribution(dtype, v):
    n = 6 * sms() + 3
    x = logits_of(n, v, dtype)
    x[0] = -torch.inf
    x[1, v // 2] = torch.nan
    x[2, v - 1] = torch.inf
    x[3, 3:] = -torch.inf
    t = torch.arange(n, device="cuda")
    logprob, entropy, lse, ids, top = kernel_opt.fused_top_logprobs(x, t, 4)
    assert (ids[:3] == -1).all() and top[:3].isnan().all() and entropy[:3].isnan().all() and logprob[:3].isnan().all()
    assert lse[0] == -torch.inf and lse[1:3].isnan().all()
    check_forward(x[3:], (logprob[3:], entropy[3:], lse[3:], ids[3:], top[3:]), 4, t[3:])


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("v,k", [(517, 1024), (50257, 32)])
def test_tokens_with_gradient(dtype, v, k):
    n, temperature = 6 * sms() + 1, 0.7
    x = logits_of(n, v, dtype).requires_grad_(True)
    g = torch.Generator(device="cuda").manual_seed(k)
    ids = torch.randint(-3, v + 3, (n, k), generator=g, device="cuda")
    lp, entropy, lse = kernel_opt.fused_token_logprobs(x, ids, temperature)
    y, lse0, h0 = reference(x.detach(), temperature)
    inside = (ids >= 0) & (ids < v)
    want = torch.where(inside, y.gather(-1, ids.clamp(0, v - 1)), 0.0) - lse0[:, None]
    close(lp, want, 1e-5 + 2.0 ** -24 * want.abs(), "logprobs")
    gi, ge = torch.randn(n, k, generator=g, device="cuda"), torch.randn(n, generator=g, device="cuda")
    d, = torch.autograd.grad((lp, entropy), x, (gi, ge))
    check_gradient(x.detach(), d, ids, gi, ge, None, temperature)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_rows_that_start_anywhere(dtype):
    n, v, k = 6 * sms() + 2, 2000, 17
    base = logits_of(n, v + 9, dtype)
    for at in (1, 3, 8):
        x = base[:, at:at + v]
        check_forward(x, kernel_opt.fused_top_logprobs(x, None, k), k, None)
