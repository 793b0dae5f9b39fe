"""GPU tests of rotary positions at sizes where a thread shares its factors among several heads, streamed results among them,
against fp64 on the device."""
import math

import pytest

pytestmark = pytest.mark.gpu

import torch  # noqa: E402

from fft_amd import rotary  # noqa: E402
from scan_reference import UNIT, half_step, tiny  # noqa: E402

SHARED = 4 * 256 * 1024  # units of heads from which on four heads share a thread's factors


def units(B, L, heads, P, size, dtype, pairs, in_place):
    """Units of 16 bytes (tfft_rotary), of all heads"""
    run = 128 // torch.finfo(dtype).bits
    turned = -(-(size // 2 if pairs == "half" else size) // run)
    return B * L * heads * (turned + (0 if in_place else -(-(P - size) // run)))


def phases(plan, positions):
    """Radians of the plan's fixed-point frequencies in fp64. The 64-bit product wraps as the kernel's does."""
    turns = positions[..., None] * plan.turns
    return turns.double() * (2.0 * math.pi * 2.0 ** -64)


def expect(plan, y, x, positions, pairs, inverse):
    angle = phases(plan, positions)[:, :, None]
    angle = -angle if inverse else angle
    c, s = plan.magnitude * angle.cos(), plan.magnitude * angle.sin()
    r = plan.size
    first, second = (slice(0, r // 2), slice(r // 2, r)) if pairs == "half" else (slice(0, r, 2), slice(1, r, 2))
    re, im = x[..., first].double(), x[..., second].double()
    # cosine and sine 4 units of 2^-24, magnitude, products and sum one each; stored once
    off = 7 * UNIT * abs(plan.magnitude) * (re.abs() + im.abs()) + tiny(x.dtype)
    for got, want in ((y[..., first], re * c - im * s), (y[..., second], re * s + im * c)):
        over = (got.double() - want).abs() - off - half_step(x.dtype) * want.abs()
        assert torch.isfinite(got).all() and float(over.max()) <= 0, float(over.max())
    assert torch.equal(y[..., r:], x[..., r:])


# heads that divide among four and do not, the second tensor's beginning inside a thread's four; whole lines (streamed) and not;
# whole heads and parts; heads that whole units fill and do not
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("pairs", ["half", "interleaved"])
@pytest.mark.parametrize("B,L,heads,key_heads,P,size", [(2, 2400, 21, 8, 128, 128), (3, 1700, 8, 6, 256, 192), (2, 1601, 33, 0, 128, 64),
                                                        (2, 2700, 13, 3, 174, 174), (1, 5003, 9, 2, 174, 100), (2, 2100, 30, 1, 102, 102)])
def test_heads_that_share(dtype, pairs, B, L, heads, key_heads, P, size):
    g = torch.Generator(device="cuda").manual_seed(P + heads)
    plan = rotary.RotaryPlan(size, magnitude=1.25)
    q = torch.randn(B, L, heads, P, device="cuda", generator=g).to(dtype)
    k = torch.randn(B, L, key_heads, P, device="cuda", generator=g).to(dtype) if key_heads else None
    positions = torch.randint(0, 1000000, (B, L), device="cuda", generator=g)
    # repeated where needed, so that every one of these calls, in place too, is above the bound
    need = SHARED / units(B, L, heads + key_heads, P, size, dtype, pairs, True)
    if need > 1:
        again = math.ceil(need)
        q, positions = q.repeat(again, 1, 1, 1), positions.repeat(again, 1)
        k = k.repeat(again, 1, 1, 1) if key_heads else None
        B *= again
    assert units(B, L, heads + key_heads, P, size, dtype, pairs, True) >= SHARED
    for inverse in (False, True):
        y = rotary.rotate(plan, q, k, positions, pairs=pairs, inverse=inverse)
        y, z = y if key_heads else (y, None)
        expect(plan, y, q, positions, pairs, inverse)
        if key_heads:
            expect(plan, z, k, positions, pairs, inverse)
        q2, k2 = q.clone(), k.clone() if key_heads else None
        rotary.rotate(plan, q2, k2, positions, pairs=pairs, inverse=inverse, out=q2, out_k=k2)
        assert torch.equal(q2, y) and (not key_heads or torch.equal(k2, z))
    # results in frames: rows that are no whole lines, and the frame stays
    frame = torch.full((B, L, heads + 1, P + 3), 7.0, device="cuda", dtype=dtype)
    rotary.rotate(plan, q, positions=positions, pairs=pairs, inverse=True, out=frame[:, :, 1:, 3:])
    assert torch.equal(frame[:, :, 1:, 3:], y) and bool((frame[:, :, 0] == 7.0).all()) and bool((frame[..., :3] == 7.0).all())
