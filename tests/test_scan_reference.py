"""The exponents that the pass over the tokens outside a list forms (csrc/row_scan.h): with c = log2(e) / T as a sum
of two fp32 numbers and r the rounded product of the largest x and the first, no x at most that large
gives an exponent x c - r that fp32 sums of powers cannot bear, while |r| is at most FAR."""

import math
import random
import re
from fractions import Fraction
from pathlib import Path

import numpy as np

HEADER = Path(__file__).resolve().parents[1] / "tiny-dsv41_amd" / "csrc" / "row_scan.h"
FAR = float.fromhex(re.search(r"constexpr float FAR = (0x1p\d+)f;", HEADER.read_text()).group(1))
MARGIN = 2.0  # powers of two that a logit may exceed the reference by before it becomes the reference


def split(T):
    """As scale_of forms it."""
    c = 1.4426950408889634 / T
    hi = np.float32(c)
    while float(hi) >= c or np.float32(c - float(hi)) == 0:
        hi = np.nextafter(hi, np.float32(0))
    return float(hi), float(np.float32(c - float(hi)))


def rounded(v: Fraction) -> float:
    """An exact value as the nearest fp32 number, ties to even."""
    if v == 0:
        return 0.0
    e = max(math.frexp(float(v))[1] - 24, -149)
    step = Fraction(2) ** e
    q = v / step
    n = q.numerator // q.denominator
    rest = q - n
    if rest > Fraction(1, 2) or (rest == Fraction(1, 2) and n % 2):
        n += 1
    return float(n * step)


def exponent(x, c, c_lo, r):
    """fma(x, c_lo, fma(x, c, -r)), each rounded to fp32."""
    X = Fraction(x)
    return rounded(X * Fraction(c_lo) + Fraction(rounded(X * Fraction(c) - Fraction(r))))


def test_no_exponent_above_what_the_sums_bear():
    rng = random.Random(1)
    worst = 0.0
    for T in (0.05, 0.3, 0.5, 0.7, 1.0, 1.3, 2.0, 20.0, 1e-6, 1e6):
        c, c_lo = split(T)
        assert c_lo > 0
        for _ in range(400):
            far = FAR * 2.0 ** -rng.uniform(0, 30)
            x = float(np.float32(rng.choice([-1, 1]) * far / c))
            r = rounded(Fraction(x) * Fraction(c))
            if abs(r) <= FAR:
                worst = max(worst, exponent(x, c, c_lo, r))
                # and the logit that is as far above it as one may be
                y = float(np.float32((r + MARGIN) / c))
                if rounded(Fraction(y) * Fraction(c)) <= r + MARGIN:
                    worst = max(worst, exponent(y, c, c_lo, r))
    assert 2.0 <= worst <= 5.0


def test_masks_below_the_first_reference_add_nothing():
    for T in (0.3, 0.5, 1.0, 2.0, 20.0):
        c, c_lo = split(T)
        for fill in (-1e9, -1e10, -1e12, -1e20, -1e30, float(np.finfo(np.float32).min)):
            x = float(np.float32(fill))
            if rounded(Fraction(x) * Fraction(c)) <= -FAR + MARGIN:
                assert exponent(x, c, c_lo, -FAR) <= (-FAR + MARGIN if x * c < -2 * FAR else MARGIN)
        # what they would add against their own rounded product, without the bound on r
    c, c_lo = split(1.0)
    x = float(np.float32(-1e10))
    assert exponent(x, c, c_lo, rounded(Fraction(x) * Fraction(c))) > 128


def test_the_split_is_the_scale():
    for T in (0.05, 0.3, 1.0, 2.0, 1e-30, 1e30):
        T = float(np.float32(T))
        c, c_lo = split(T)
        assert abs((c + c_lo) * T / 1.4426950408889634 - 1) < 2.0 ** -46 and 0 < c_lo <= c * 2.0 ** -23 * 1.01
