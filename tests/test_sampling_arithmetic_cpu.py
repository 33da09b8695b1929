"""The sampling kernel's arithmetic on the host (csrc/k1_sample_math.cuh, through the test-only
library): a list's weights as whole numbers, whatever their size, and the element that a lane draws."""
import ctypes
import math

import numpy as np
import pytest

from _helpers import CAPI_LIB, WAIT_TEST_LIB

CAP = 2048        # entries of a list
COUNT_BITS = 12


@pytest.fixture(scope="module")
def lib():
    assert not hasattr(ctypes.CDLL(CAPI_LIB), "k1_test_list")
    lib = ctypes.CDLL(WAIT_TEST_LIB)
    lib.k1_test_list.argtypes = [ctypes.c_void_p, ctypes.c_int, ctypes.c_double, ctypes.c_void_p, ctypes.c_void_p]
    lib.k1_test_list.restype = None
    lib.k1_test_pick.argtypes = [ctypes.c_void_p, ctypes.c_double, ctypes.c_double]
    lib.k1_test_pick.restype = ctypes.c_int
    return lib


def words(lib, w, share):
    w = np.ascontiguousarray(w, np.float32)
    out, target = np.zeros(len(w), np.uint64), np.zeros(1, np.uint64)
    lib.k1_test_list(w.ctypes.data, len(w), share, out.ctypes.data, target.ctypes.data)
    return [int(v) for v in out], int(target[0])


def lists():
    rng = np.random.default_rng(0)
    yield "one", [1.0]
    yield "flat", np.ones(CAP)
    yield "the lightest weights that fp32 holds", np.full(CAP, 2.0 ** -149)
    yield "one of them", [2.0 ** -149]
    # rows whose nucleus ends among weights of e^-28.5: a list of their own
    yield "light", np.exp(rng.uniform(-28.55, -28.45, 91))
    yield "lighter", np.exp(rng.uniform(-60, -45, CAP))
    yield "peaked", np.concatenate([[1.0], np.exp(rng.uniform(-30, -2, CAP - 1))])
    yield "spread", np.exp(rng.uniform(-103, 0, 1000))
    yield "below a power of two", [1.0 - 2.0 ** -24] * 3


@pytest.mark.parametrize("name,w", list(lists()), ids=lambda v: v if isinstance(v, str) else "")
@pytest.mark.parametrize("share", [0.0, 1e-9, 0.5, 1 - 2.0 ** -24, 1.0])
def test_a_list_keeps_its_mass(lib, name, w, share):
    w = np.asarray(w, np.float32)
    out, target = words(lib, w, share)
    total = sum(out)
    assert total < 2 ** 64
    assert total & (2 ** COUNT_BITS - 1) == len(w)
    weights = [v >> COUNT_BITS for v in out]
    all_units, mass = total >> COUNT_BITS, float(w.astype(np.float64).sum())
    assert sum(weights) == all_units
    # the unit, from the heaviest entry: 2^50 to 2^51 units in all
    assert 2 ** 50 - CAP <= all_units <= 2 ** 51 + CAP
    assert max(weights) >= 2 ** 39 - 1
    unit = 2.0 ** (51 - math.frexp(mass)[1])
    assert all(abs(v - float(x) * unit) <= 0.5 for v, x in zip(weights, w))
    # a target that some entry reaches, within the words' rounding of the share
    assert 1 <= target <= all_units
    assert abs(target - share * all_units) <= 1 + 2.0 ** -40 * all_units


def test_a_list_without_mass_asks_for_nothing(lib):
    out, target = words(lib, [0.0, 0.0], 0.9)
    assert out == [1, 1] and target == 0


def pick(lib, w, cum, target):
    w = np.array(list(w) + [0] * (8 - len(w)), np.float32)
    return lib.k1_test_pick(w.ctypes.data, cum, target)


def test_the_element_whose_prefix_exceeds_the_target(lib):
    assert pick(lib, [0.25, 0, 0.25, 0.5], 1.0, 1.0) == 0
    assert pick(lib, [0.25, 0, 0.25, 0.5], 1.0, 1.25) == 2
    assert pick(lib, [0.25, 0, 0.25, 0.5], 1.0, 1.49) == 2
    assert pick(lib, [0.25, 0, 0.25, 0.5], 1.0, 1.5) == 3
    assert pick(lib, [0.25, 0, 0.25, 0.5], 1.0, math.inf) == 3   # none exceeds: the last with a weight
    assert pick(lib, [0, 0, 0, 0.5], 0.0, 0.0) == 3
    assert pick(lib, [0] * 8, 0.0, 0.0) == -1


def test_a_lane_with_mass_always_draws(lib):
    """The prefix sums of a warp's lanes are rounded in another order than a lane's prefix less its
    own mass: here the third lane's prefix exceeds the target, which the second's does not, and its
    start (1 + 2^-52) does too."""
    t = 0.4 * 2.0 ** -52
    lane = [np.float32(t)]
    incl = 1.0 + (t + t)                 # a tree adds the two small ones first
    assert 1.0 + t == 1.0 and incl == 1.0 + 2.0 ** -52 and incl - t > 1.0
    assert pick(lib, lane, incl - float(np.float32(t)), 1.0) == 0
    rng = np.random.default_rng(2)
    for _ in range(2000):
        w = rng.random(8).astype(np.float32) * (rng.random(8) < 0.5)
        got = pick(lib, w, rng.random() * 2, rng.random() * 2)
        assert (got >= 0) == bool((w > 0).any()) and (got < 0 or w[got] > 0)
