"""Rotary positions: pairs of a head's values times exp(i position frequency), and the inverse, which is the gradient.

The framework's twiddle product (tfft_fourstep_twiddle) for positions and frequencies of a model's. A frequency is rounded
once, to a 64-bit fraction of a turn per position; the product with a 64-bit position is exact modulo one turn, so position p is
off by p 2^-65 turns at most (2^-25 at 2^40). See tfft_rotary in include/thunderfft_c.h. No counterpart in the reference, whose
twiddles belong to one transform (thunderfft/include/thunderfft/detail/util_arith.h:75-91).

    plan = RotaryPlan(128, base=10000.0)
    q, k = rotate(plan, q, k, positions)                  # q [B, L, H, P], k [B, L, H', P], positions int [B, L] or [L]
    dq, dk = rotate(plan, dq, dk, positions, inverse=True)

Autograd does not see these calls; a tensor that requires a gradient is taken for its values, with a warning while gradients are
enabled (the gradient is the inverse rotation, in a torch.autograd.Function).
"""
import functools
import math

import torch

from . import _lib
from .api import _check
from .recurrence import _FLOATS, _out, _placed, _refuse, _same_device, _values

_PAIRS = {"half": 0, "interleaved": 1}
_POSITIONS = {torch.int64: 8, torch.int32: 4}


@functools.lru_cache(maxsize=None)
def _one_turn(bits):
    """2^bits / (2 pi) to within a few units, with pi by Machin's formula 16 atan(1/5) - 4 atan(1/239) in integers and 32 bits more"""
    def atan(n):
        term = total = (1 << bits + 32) // n
        k = 1
        while term:
            term //= -n * n
            k += 2
            total += term // k
        return total

    return (1 << 2 * bits + 31) // (16 * atan(5) - 4 * atan(239))


def _word(f):
    """round(2^64 f / (2 pi)) modulo 2^64 for any fp64 number f, as a signed 64-bit number. f is m 2^e with 53 bits of m; the
    product with so many bits of 1 / (2 pi) is right to 2^-120 before it is rounded."""
    m, e = math.frexp(f)
    bits = 256 if e <= 64 else 1216
    shift = bits - 11 - e  # at least 181
    word = (int(m * 2.0 ** 53) * _one_turn(bits) + (1 << shift - 1) >> shift) % 2 ** 64
    return word - 2 ** 64 if word >= 2 ** 63 else word


class RotaryPlan:
    """Frequencies of `size` rotated values (size / 2 pairs): pair i turns by base^(-2 i / size) radians a position.

    scaling stretches them for contexts longer than the one a model was trained on, by `factor`:
      "linear"  every frequency divided by factor;
      "base"    base grown to base * factor^(size / (size - 2)), which divides the slowest frequency by factor and
                leaves the fastest;
      "ramp"    pairs that make at least high_turns turns within original_length positions keep their frequency,
                pairs with at most low_turns have it divided by factor, those between mix the two linearly.
    frequencies: a list of size / 2 radians per position in their place. magnitude multiplies the rotated values.
    The table lies on `device` (default: the current one); a plan belongs to that device."""

    def __init__(self, size, base=10000.0, scaling=None, factor=1.0, original_length=None, low_turns=1.0,
                 high_turns=32.0, magnitude=1.0, frequencies=None, device=None):
        size = int(size)
        if size < 2 or size % 2:
            _refuse(f"RotaryPlan: an even number of values of at least 2, not {size}")
        if frequencies is None:
            if not (math.isfinite(base) and base > 0 and math.isfinite(factor) and factor > 0):
                _refuse("RotaryPlan: base and factor are positive")
            if scaling not in (None, "linear", "base", "ramp"):
                _refuse(f"RotaryPlan: unknown scaling {scaling!r} (None, 'linear', 'base' or 'ramp')")
            try:
                if scaling == "base" and size > 2:
                    base = base * factor ** (size / (size - 2.0))
                frequencies = [base ** (-2.0 * i / size) for i in range(size // 2)]
            except (OverflowError, ZeroDivisionError):
                base = math.inf
            if not math.isfinite(base):
                _refuse("RotaryPlan: base and factor leave the range of fp64")
            if scaling == "linear":
                frequencies = [f / factor for f in frequencies]
            if scaling == "ramp":
                if original_length is None or not original_length > 0 or not high_turns > low_turns:
                    _refuse("RotaryPlan: scaling 'ramp' needs original_length and low_turns < high_turns")
                mixed = []
                for f in frequencies:
                    turns = original_length * f / (2.0 * math.pi)
                    keep = min(1.0, max(0.0, (turns - low_turns) / (high_turns - low_turns)))
                    mixed.append(f * keep + f / factor * (1.0 - keep))
                frequencies = mixed
        elif scaling is not None:
            _refuse("RotaryPlan: scaling is applied to base's frequencies, not to a given list")
        frequencies = [float(f) for f in frequencies]
        if len(frequencies) != size // 2 or not all(math.isfinite(f) for f in frequencies):
            _refuse(f"RotaryPlan: {size // 2} finite frequencies")
        if not abs(magnitude) <= torch.finfo(torch.float32).max:
            _refuse("RotaryPlan: magnitude is a finite fp32 number")
        self.size, self.magnitude, self.frequencies = size, float(magnitude), frequencies
        # turns per position in units of 2^-64, modulo 1 turn
        self.turns = torch.tensor([_word(f) for f in frequencies], dtype=torch.int64).to("cuda" if device is None else device)


def rotate(plan, q, k=None, positions=None, pairs="half", inverse=False, first=0, out=None, out_k=None, stream=None):
    """q (and k, by the same positions and in the same launch) rotated: a tensor, or a pair where k is given.

    q, k: [B, L, heads, P] float32, float16 or bfloat16 with contiguous heads, heads of their own number; the first
    plan.size of the P values are rotated, the rest copied. pairs: "half" pairs value i with i + size / 2, "interleaved"
    2 i with 2 i + 1. positions: int64 or int32 [B, L] or [L] on the device (negative ones turn backwards); without
    them position t is first + t. inverse: the other way round, which is the gradient of rotate. out, out_k: tensors for the
    results, q and k themselves allowed (but no view that torch has only noted as negated). Asynchronous on `stream` (default:
    torch's current stream)."""
    device = _same_device("rotate", q, k, plan.turns, positions, out, out_k)
    return _placed(_rotate, device, stream, plan, q, k, positions, pairs, inverse, first, out, out_k)


_NO_TENSOR = (0,) * 9


def _rotate(plan, q, k, positions, pairs, inverse, first, out, out_k, stream):
    who = "rotate"
    if q.is_neg() or (k is not None and k.is_neg()) or (positions is not None and positions.is_neg()):
        q, k, positions = _values(q, k, positions)
    dtype, shape = q.dtype, q.shape
    code = _FLOATS.get(dtype)
    if code is None:
        _refuse(f"{who}: unsupported element type {dtype}", 1)
    if pairs not in _PAIRS:
        _refuse(f"{who}: pairs is 'half' or 'interleaved', not {pairs!r}")
    if len(shape) != 4:
        _refuse(f"{who}: q is [batch, time, heads, values], got {tuple(shape)}")
    B, L, H, P = shape
    if plan.size > P:
        _refuse(f"{who}: the plan rotates {plan.size} values, a head has {P}")
    at = position_bytes = position_batch = position_time = 0
    if positions is None:
        first = int(first)
        if not -2 ** 63 <= first < 2 ** 63:
            _refuse(f"{who}: first is a 64-bit number, not {first}")
    else:
        first = 0
        position_bytes = _POSITIONS.get(positions.dtype)
        if position_bytes is None:
            _refuse(f"{who}: positions are int64 or int32, not {positions.dtype}")
        if positions.shape == (B, L):
            position_batch, position_time = positions.stride()
        elif positions.shape == (L,):
            position_time = positions.stride(0)
        else:
            _refuse(f"{who}: positions {tuple(positions.shape)} are neither [{B}, {L}] nor [{L}]")
        at = positions.data_ptr()
    out = _out(who, "the result of q", out, q)
    first_view = _view(who, q, out, H, P)
    if k is None:
        if out_k is not None:
            _refuse(f"{who}: out_k without k")
        second_view = _NO_TENSOR
    else:
        k_shape = k.shape
        if k.dtype != dtype or len(k_shape) != 4 or k_shape[0] != B or k_shape[1] != L or k_shape[3] != P:
            _refuse(f"{who}: k is a {dtype} tensor [{B}, {L}, heads, {P}]")
        out_k = _out(who, "the result of k", out_k, k)
        second_view = _view(who, k, out_k, k_shape[2], P)
    rc = _lib.load().tfft_rotary(
        _lib.ROTARY_ARGS.pack(_lib.ROTARY_ARGS.size, code, _PAIRS[pairs], bool(inverse), B, L, P, plan.size, plan.magnitude,
                              position_bytes, plan.turns.data_ptr(), at, position_batch, position_time, first,
                              *first_view, *second_view), stream)
    if rc:
        _check(rc)
    return out if k is None else (out, out_k)


def _view(who, t, out, heads, values):
    a, b, c, one = t.stride()
    d, e, f, out_one = out.stride()
    if values > 1 and (one != 1 or out_one != 1):
        _refuse(f"{who}: the values of a head are contiguous")
    return t.data_ptr(), out.data_ptr(), heads, a, b, c, d, e, f
