"""Every shape that a test gives to one kernel of the 8-bit product takes that kernel, so a change of
the rule between them cannot move the tests away from what they test."""
import pytest

import test_gpu_decode_waits_pair as waits
import test_gpu_fp8_many_tokens as many
from _linear import MANY, kernel_of


@pytest.mark.parametrize("m,k,n", many.SHAPES + waits.SHAPES + [many.LAYOUT])
def test_many_tokens(m, k, n):
    assert kernel_of(m, k, n) == MANY


@pytest.mark.parametrize("m,k,n,want", [(1, 3584, 152064, 16), (16, 256, 300, 16), (17, 3584, 256, 32), (32, 256, 300, 32),
                                        (33, 512, 129, 64), (64, 3584, 128256, 64), (300, 512, 20000, 64)])
def test_few_tokens(m, k, n, want):
    assert kernel_of(m, k, n) == want
