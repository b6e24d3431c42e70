"""The roundings that the quantised, sampled decode's kernels state of themselves, computed: the series of the sampling weights and the bf16 planes of an fp32 number."""
import math
from fractions import Fraction

import numpy as np


def test_the_series_of_a_sampling_weight():
    """sample_kernels.hip: e^y, |y| <= ln 2 / 64, as 1 + y + y^2 / 2 + y^3 / 6 + y^4 / 24 is off by less than 2^-39: 21 to 22 units of 2^-44 at the largest weight, half a unit at 2^-6"""
    worst = 0.0
    for i in range(-1000, 1001):
        y = Fraction(math.log(2) / 64) * i / 1000
        series = sum(y ** k / math.factorial(k) for k in range(5))
        whole = sum(y ** k / math.factorial(k) for k in range(20))
        worst = max(worst, float(abs(series / whole - 1)))
    assert 2.0 ** -40 < worst < 2.0 ** -39
    assert 21 < worst * 2 ** 44 < 23 and worst * 2 ** 38 < 0.5


def _cut(x):
    return (x.view(np.uint32) & np.uint32(0xffff0000)).view(np.float32)


def test_bf16_planes_of_an_fp32_number():
    """nn_common.h, kv8_kernels.hip: three planes are the number; two leave up to 2^-15 of it, always of its own sign, about 2^-17 on average"""
    rng = np.random.default_rng(0)
    x = np.concatenate([rng.random(1 << 20, dtype=np.float32), np.array([0x3f80ffff, 0x3f80feff, 0x3fffffff], dtype=np.uint32).view(np.float32)])
    x = x[x > 0]
    hi = _cut(x)
    mid = _cut(x - hi)
    lo = _cut(x - hi - mid)
    assert (hi.astype(np.float64) + mid + lo == x).all()
    left = (x.astype(np.float64) - hi - mid) / x
    assert (left >= 0).all() and 2.0 ** -16 < left.max() < 2.0 ** -15 and 2.0 ** -18 < left.mean() < 2.0 ** -16
