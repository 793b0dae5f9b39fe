"""GPU tests of the gated recurrence on rows of whole cache lines, which pass through the chip as streams, over several chunks:
against fp64 on the device with a bound for every element, and in place."""
import pytest

pytestmark = pytest.mark.gpu

import torch  # noqa: E402

from fft_amd import recurrence  # noqa: E402
from scan_reference import UNIT, half_step, tiny  # noqa: E402

TYPES = [(torch.float32, torch.float32), (torch.float16, torch.float32), (torch.float16, torch.float16),
         (torch.bfloat16, torch.float32), (torch.bfloat16, torch.bfloat16)]
M = 64


def walk(a, v, start):
    """h[t] = a[t] h[t-1] + v[t] along dim 1 in fp64: stretches of M steps side by side, then joined."""
    B, L, D = v.shape
    pad = (0, 0, 0, -L % M)
    a = torch.nn.functional.pad(a, pad, value=1.0).view(B, -1, M, D)
    v = torch.nn.functional.pad(v, pad).view(B, -1, M, D)
    h, product = torch.empty_like(v), torch.cumprod(a, 2)
    z = torch.zeros_like(v[:, :, 0])
    for t in range(M):
        z = a[:, :, t] * z + v[:, :, t]
        h[:, :, t] = z
    for j in range(h.shape[1]):
        h[:, j] += product[:, j] * start[:, None]
        start = h[:, j, M - 1].clone()
    return h.view(B, -1, D)[:, :L]


def sums(a, w, v, start):
    """The three sums of the bound in scan_reference: H, of the terms' magnitudes, N, each counted once for every step it
    travelled, and K, as often as the |log decays| it met add up to; each a recurrence with the decays `a`."""
    H = walk(a, v.abs(), start.abs())
    before = torch.cat([start.abs()[:, None], H[:, :-1]], 1)
    zero = torch.zeros_like(start)
    return H, walk(a, a * before, zero), walk(a, a * w * before, zero)


def within(got, want, bound, what):
    assert torch.isfinite(got).all(), what
    over = float(((got.double() - want).abs() - bound).max())
    assert over <= 0, (what, over)


@pytest.mark.parametrize("dtype,gate_dtype", TYPES)
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("B,L,D", [(3, 700, 4096), (1, 6000, 128), (2, 1031, 256)])
def test_lines(dtype, gate_dtype, ragged, B, L, D):
    g = torch.Generator(device="cuda").manual_seed(L)
    x, dy = (torch.randn(B, L, D, device="cuda", generator=g).to(dtype) for _ in range(2))
    gate = (-torch.exp(-6.9 * torch.rand(B, L, D, device="cuda", generator=g))).to(gate_dtype)
    initial, dlast = torch.randn(B, D, device="cuda", generator=g), torch.randn(B, D, device="cuda", generator=g)
    lengths = torch.tensor([L - 130, 3, 400][:B], dtype=torch.int32, device="cuda") if ragged else None
    assert all(t.data_ptr() % 128 == 0 and D * t.element_size() % 128 == 0 for t in (x, dy, gate))
    kw = dict(log_gate=True, lengths=lengths, initial=initial)
    y, last = recurrence.gated_scan(x, gate, **kw)
    dx, dgate, dinitial = recurrence.gated_scan_backward(dy, y, gate, dlast=dlast, **kw)

    inside = torch.ones(B, L, 1, dtype=torch.bool, device="cuda")
    if ragged:
        inside = (torch.arange(L, device="cuda") < lengths[:, None])[:, :, None]
    a = torch.where(inside, gate.double().exp(), 1.0)
    w = torch.where(inside, gate.double().abs(), 0.0)
    zero = torch.zeros((), dtype=torch.float64, device="cuda")
    v, d = torch.where(inside, x.double(), zero), torch.where(inside, dy.double(), zero)
    # steps behind a sequence (a decay of 1) count as travelled here, which only widens the bound by nothing that is compared:
    # y is 0 there, and last is taken from the last step inside
    h = walk(a, v, initial.double())
    H, N, K = sums(a, w, v, initial.double())
    off = UNIT * (4 * N + 1.5 * K + 24 * H)
    within(y, torch.where(inside, h, zero), torch.where(inside, off + half_step(dtype) * h.abs() + tiny(dtype), zero), "y")
    at = (lengths.long() if ragged else torch.full((B,), L, device="cuda")) - 1
    rows = torch.arange(B, device="cuda")
    within(last, h[rows, at], off[rows, at] + 1e-38, "last")
    # e[t] = dy[t] + a[t+1] e[t+1]; the last state's gradient in front of the first step back
    one = torch.ones_like(a[:, :1])
    later = torch.cat([a[:, 1:], one], 1).flip(1)
    later_w = torch.cat([w[:, 1:], torch.zeros_like(one)], 1).flip(1)
    e = walk(later, d.flip(1), dlast.double()).flip(1)
    H, N, K = (s.flip(1) for s in sums(later, later_w, d.flip(1), dlast.double()))
    off = UNIT * (4 * N + 1.5 * K + 24 * H)
    within(dx, torch.where(inside, e, zero), torch.where(inside, off + half_step(dtype) * e.abs() + tiny(dtype), zero), "dx")
    before = torch.cat([initial.double()[:, None], y.double()[:, :-1]], 1)
    da = e * before * a
    bound = (before * a).abs() * (off + UNIT * (7 + 1.5 * w) * H) + half_step(gate_dtype) * da.abs() + tiny(gate_dtype)
    within(dgate, torch.where(inside, da, zero), torch.where(inside, bound, zero), "dgate")
    # one product and decay more than e[0]
    within(dinitial, a[:, 0] * e[:, 0], a[:, 0] * (off[:, 0] + UNIT * (6 + 1.5 * w[:, 0]) * H[:, 0]) + 1e-38, "dinitial")

    # in place: the same bits
    x2, dy2 = x.clone(), dy.clone()
    assert torch.equal(recurrence.gated_scan(x2, gate, out=x2, **kw)[0], y)
    got = recurrence.gated_scan_backward(dy2, y, gate, dlast=dlast, dx=dy2, **kw)
    assert torch.equal(dy2, dx) and torch.equal(got[1], dgate) and torch.equal(got[2], dinitial)
