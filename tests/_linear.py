"""Which kernel an 8-bit product takes, asked of the rule itself (in the test-only library)."""
import ctypes

from _helpers import WAIT_TEST_LIB

MANY = 0        # the many-token kernel; else the tokens per block of the few-token kernel
B200_SMS = 148


def kernel_of(tokens, inner, outer, sms=B200_SMS):
    f = ctypes.CDLL(WAIT_TEST_LIB).k1_test_linear_kernel
    f.argtypes = [ctypes.c_int64, ctypes.c_int64, ctypes.c_int64, ctypes.c_int]
    f.restype = ctypes.c_int
    return f(tokens, inner, outer, sms)
