"""Rotary frequencies between the ends that YaRN keeps and stretches."""
import ctypes as C
import math
from fractions import Fraction

import pytest

import arcllm_b200 as A


def yarn(rot, theta, factor, trained):
    """The published form: pair i turns trained * f_i / 2 pi times over the trained context; the pairs at which that is
    32 and 1, rounded outwards, are the ends of a linear ramp from f_i to f_i / factor.  Ends and ramp as fractions."""
    f = [theta ** (-2.0 * i / rot) for i in range(rot // 2)]

    def pair_of(turns):  # the real number i with trained * theta^(-2 i / rot) = 2 pi turns
        return math.log(trained / (2 * math.pi * turns)) / math.log(theta) * rot / 2

    lo, hi = max(0, math.floor(pair_of(32))), min(rot - 1, math.ceil(pair_of(1)))
    assert hi > lo and all(abs(x - round(x)) > 1e-9 for x in (pair_of(32), pair_of(1)))
    ramp = [min(Fraction(1), max(Fraction(0), Fraction(i - lo, hi - lo))) for i in range(rot // 2)]
    return [x * float(1 - r) + x / factor * float(r) for x, r in zip(f, ramp)], f


@pytest.mark.parametrize("rot", [16, 32, 64, 96, 128])
@pytest.mark.parametrize("theta,factor,trained", [(1e6, 4.0, 4096.0), (1e4, 16.0, 2048.0), (5e5, 8.0, 8192.0),
                                                  (1e6, 1.0, 32768.0), (1e4, 40.0, 4096.0)])
def test_yarn_ramp(rot, theta, factor, trained):
    f, s = (C.c_double * (rot // 2))(), C.c_float()
    A.call("arcllm_cuda_rope_freqs", A.ROPE_YARN, rot, theta, factor, trained, f, C.byref(s))
    want, plain = yarn(rot, theta, factor, trained)
    # Six roundings of positive terms (power, quotients, products, sum) on either side; and the ramp, which is a difference
    # from 1, may be off by two of 1, which is factor times as many of what is left of a frequency.
    tol = (12 + 2 * factor) * 2.0 ** -53
    for g, w in zip(f, want):
        assert abs(g - w) <= tol * w
    assert abs(s.value - (0.1 * math.log(factor) + 1)) < 1e-7
    kept = [g / x for g, x in zip(f, plain)]  # from 1 down to 1 / factor, in order
    assert all(b <= a + tol for a, b in zip(kept, kept[1:]))
    if factor > 1 and rot >= 64:
        assert any(1 / factor + 1e-3 < k < 1 - 1e-3 for k in kept)
