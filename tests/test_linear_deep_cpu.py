"""Which products with an epilogue take the deeper ring: the kind that was measured faster with it, and none of
those that were measured slower (asked of the rule itself, in the test-only library)."""
import ctypes

import pytest

from _helpers import WAIT_TEST_LIB
from _linear import B200_SMS


def deep(tokens, inner, outer):
    f = ctypes.CDLL(WAIT_TEST_LIB).k1_test_linear_deep
    f.argtypes = [ctypes.c_int64, ctypes.c_int64, ctypes.c_int64, ctypes.c_int]
    return bool(f(tokens, inner, outer, B200_SMS))


@pytest.mark.parametrize("m,k,n", [(16, 3584, 14336), (1, 3584, 14336), (9, 2048, 12800), (16, 28672, 14336)])
def test_deep(m, k, n):
    assert deep(m, k, n)


@pytest.mark.parametrize("m,k,n", [(32, 3584, 14336), (64, 3584, 14336), (64, 28672, 2048), (16, 1040, 4100), (64, 1040, 4100),
                                   (37, 2048, 1000), (64, 512, 18000), (16, 512, 12800), (16, 3584, 151936), (2048, 14336, 3584)])
def test_not_deep(m, k, n):
    assert not deep(m, k, n)
