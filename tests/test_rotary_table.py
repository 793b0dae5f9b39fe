"""CPU tests of a rotary plan's table against exact arithmetic."""
import math
from fractions import Fraction

import pytest

from fft_amd import rotary

# 2 pi to 100 decimals
TWO_PI = Fraction("6.2831853071795864769252867665590057683943387987502116419498891846156328125724179972560696506842341360")


def word(f):
    """round(2^64 f / (2 pi)) modulo 2^64 for an fp64 frequency. With 100 decimals of 2 pi it is right for |f| below 2^200."""
    return round(Fraction(f) * 2 ** 64 / TWO_PI) % 2 ** 64


def table(frequencies):
    plan = rotary.RotaryPlan(2 * len(frequencies), frequencies=frequencies, device="cpu")
    return [int(w) % 2 ** 64 for w in plan.turns.tolist()]


@pytest.mark.parametrize("frequencies", [
    [1.0, -1.0, 0.5, -0.5, 1e-4, -1e-4], [1e-12, -1e-12, 3e-19, -3e-19, 5e-324, -5e-324, 0.0, -0.0],
    [2 * math.pi, -2 * math.pi, math.pi, -math.pi, math.pi / 2, math.nextafter(2 * math.pi, 0), math.nextafter(2 * math.pi, 9)],
    [100.0, -100.0, 1e6 + 0.1, -1e9, 2.0 ** 60 + 2.0 ** 9, 1e50, -1e50]])
def test_words(frequencies):
    assert table(frequencies) == [word(f) for f in frequencies]


def test_words_of_bases():
    for size, base in ((128, 10000.0), (64, 500000.0), (2, 7.0), (254, 1e6)):
        plan = rotary.RotaryPlan(size, base=base, device="cpu")
        assert [int(w) % 2 ** 64 for w in plan.turns.tolist()] == [word(base ** (-2.0 * i / size)) for i in range(size // 2)]
        # the way back is the negated table
        back = table([-f for f in plan.frequencies])
        assert back == [-word(f) % 2 ** 64 for f in plan.frequencies]


def test_the_largest_frequency():
    """Any finite frequency has a word; two neighbours, far more than a turn apart, have words of their own."""
    big = table([1.7976931348623157e308, -1.7976931348623157e308, math.nextafter(1.7976931348623157e308, 0)])
    assert (big[0] + big[1]) % 2 ** 64 == 0 and big[0] != big[2]
