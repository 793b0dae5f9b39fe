"""Rotary positions: pairs of a head's values times exp(i position frequency), and the inverse, which is the gradient.

The framework's twiddle product (tfft_fourstep_twiddle) for positions and frequencies of a model's: the phase is an
exact fraction of a turn in 64-bit integers, so positions of any size lose nothing. See tfft_rotary in
include/thunderfft_c.h. No counterpart in the reference, whose twiddles belong to one transform
(thunderfft/include/thunderfft/detail/util_arith.h:75-91).

    plan = RotaryPlan(128, base=10000.0)
    q, k = rotate(plan, q, k, positions)                  # q [B, L, H, P], k [B, L, H', P], positions int [B, L] or [L]
    dq, dk = rotate(plan, dq, dk, positions, inverse=True)
"""
import math

import torch

from . import _lib
from .api import _check
from .recurrence import _FLOATS, _placed, _refuse

_PAIRS = {"half": 0, "interleaved": 1}


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
            if scaling == "base" and size > 2:
                base = base * factor ** (size / (size - 2.0))
            frequencies = [base ** (-2.0 * i / size) for i in range(size // 2)]
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
        if not math.isfinite(magnitude):
            _refuse("RotaryPlan: magnitude is finite")
        self.size, self.magnitude, self.frequencies = size, float(magnitude), frequencies
        # turns per position in units of 2^-64, modulo 1 turn; the fp64 quotient is exact to 2^-53 of itself
        words = [int(f / (2.0 * math.pi) % 1.0 * 2.0 ** 64) % 2 ** 64 for f in frequencies]
        words = [w - 2 ** 64 if w >= 2 ** 63 else w for w in words]
        self.turns = torch.tensor(words, dtype=torch.int64).to("cuda" if device is None else device)


def rotate(plan, q, k=None, positions=None, pairs="half", inverse=False, first=0, out=None, out_k=None, stream=None):
    """q (and k, by the same positions and in the same launch) rotated: a tensor, or a pair where k is given.

    q, k: [B, L, heads, P] float32, float16 or bfloat16 with contiguous heads, heads of their own number; the first
    plan.size of the P values are rotated, the rest copied. pairs: "half" pairs value i with i + size / 2, "interleaved"
    2 i with 2 i + 1. positions: int64 or int32 [B, L] or [L] on the device (negative ones turn backwards); without
    them position t is first + t. inverse: the other way round, which is the gradient of rotate. out, out_k: tensors for the results,
    q and k themselves allowed. Asynchronous on `stream` (default: torch's current stream)."""
    if not q.is_cuda:
        _refuse("rotate needs device tensors")
    return _placed(_rotate, q.device, stream, plan, q, k, positions, pairs, inverse, first, out, out_k)


_NO_TENSOR = (0,) * 9


def _rotate(plan, q, k, positions, pairs, inverse, first, out, out_k, stream):
    who = "rotate"
    code = _FLOATS.get(q.dtype)
    if code is None:
        _refuse(f"{who}: unsupported element type {q.dtype}", 1)
    if pairs not in _PAIRS:
        _refuse(f"{who}: pairs is 'half' or 'interleaved', not {pairs!r}")
    if q.dim() != 4:
        _refuse(f"{who}: q is [batch, time, heads, values], got {tuple(q.shape)}")
    B, L, _, P = q.shape
    if plan.size > P:
        _refuse(f"{who}: the plan rotates {plan.size} values, a head has {P}")
    if k is None and out_k is not None:
        _refuse(f"{who}: out_k without k")
    device = q.device
    for t in (plan.turns, k, positions, out, out_k):
        if t is not None and t.device != device:
            _refuse(f"{who}: tensors on {device} and {t.device}")
    position_bytes = position_batch = position_time = 0
    if positions is not None:
        if positions.dtype not in (torch.int64, torch.int32):
            _refuse(f"{who}: positions are int64 or int32, not {positions.dtype}")
        if positions.shape != (B, L) and positions.shape != (L,):
            _refuse(f"{who}: positions {tuple(positions.shape)} are neither [{B}, {L}] nor [{L}]")
        position_bytes = positions.element_size()
        position_batch = positions.stride(0) if positions.dim() == 2 else 0
        position_time = positions.stride(-1)
    views, results = [], []
    for t, o in ((q, out), (k, out_k)):
        if t is None:
            views += _NO_TENSOR
            continue
        if t.dim() != 4 or t.dtype != q.dtype or t.shape[0] != B or t.shape[1] != L or t.shape[3] != P:
            _refuse(f"{who}: k is a {q.dtype} tensor [{B}, {L}, heads, {P}]")
        if o is None:
            o = torch.empty(t.shape, dtype=t.dtype, device=device)
        elif o.dtype != t.dtype or o.shape != t.shape:
            _refuse(f"{who}: a result is a {t.dtype} tensor {tuple(t.shape)}")
        *steps, one = t.stride()
        *out_steps, out_one = o.stride()
        if P > 1 and (one != 1 or out_one != 1):
            _refuse(f"{who}: the values of a head are contiguous")
        results.append(o)
        views += (t.data_ptr(), o.data_ptr(), t.shape[2], *steps, *out_steps)
    rc = _lib.load().tfft_rotary(
        _lib.ROTARY_ARGS.pack(_lib.ROTARY_ARGS.size, code, _PAIRS[pairs], bool(inverse), B, L, P, plan.size, plan.magnitude,
                              position_bytes, plan.turns.data_ptr(), 0 if positions is None else positions.data_ptr(),
                              position_batch, position_time, int(first), *views), stream)
    if rc:
        _check(rc)
    return results[0] if k is None else tuple(results)
