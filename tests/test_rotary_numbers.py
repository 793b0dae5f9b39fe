"""Numbers that a rotary call cannot be made with are refused as such: a magnitude beyond fp32, frequencies and bases that leave
fp64, first positions beyond 64 bits."""
import pytest

import fft_amd
from fft_amd import rotary


@pytest.mark.parametrize("arguments", [
    dict(magnitude=1e39), dict(magnitude=-3.5e38), dict(magnitude=float("nan")), dict(base=1e-300, scaling="linear", factor=1e-300),
    dict(base=1e300, scaling="base", factor=1e100), dict(base=float("inf")), dict(factor=float("nan")), dict(frequencies=[1.0, float("inf")])])
def test_plans(arguments):
    with pytest.raises(fft_amd.ThunderFFTError):
        rotary.RotaryPlan(4, device="cpu", **arguments)


def test_the_largest_magnitude():
    assert rotary.RotaryPlan(4, device="cpu", magnitude=3.4e38).magnitude == 3.4e38


@pytest.mark.gpu
def test_first_positions():
    import torch

    plan, x = rotary.RotaryPlan(4), torch.zeros(1, 2, 1, 4, device="cuda")
    for first in (2 ** 63, -2 ** 63 - 1):
        with pytest.raises(fft_amd.ThunderFFTError):
            rotary.rotate(plan, x, first=first)
    assert not rotary.rotate(plan, x, first=2 ** 63 - 2).any() and not rotary.rotate(plan, x, first=-2 ** 63).any()
