"""The probability that the wrappers hand to the C ABI, in 32 bits, keeps the threshold of the
caller's 64-bit one (no GPU)."""
import math

import numpy as np

from teenyformers_b200 import ops


def _t(p):
    return math.floor((1.0 - p) * 65536.0 + 0.5)


def test_threshold_is_that_of_the_64_bit_probability():
    # (12 of the 4-digit ones differ where p itself is rounded to 32 bits)
    assert sum(_t(k / 10000) != _t(float(np.float32(k / 10000))) for k in range(10001)) == 12
    for p in [k / 10000 for k in range(10001)] + [2.0 ** -k for k in range(1, 60)] + [1 - 2.0 ** -17]:
        q = ops._drop_p(p)
        assert float(np.float32(q)) == q and _t(q) == _t(p), p


def test_what_is_no_probability_is_left_to_be_refused():
    assert ops._drop_p(-0.1) == -0.1 and ops._drop_p(1.5) == 1.5
    assert math.isnan(ops._drop_p(float("nan")))
