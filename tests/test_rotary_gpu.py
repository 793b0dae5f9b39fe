"""GPU tests of rotary positions (fft_amd.rotary, tfft_rotary) against exact phases and fp64 rotations."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

import torch  # noqa: E402

import fft_amd  # noqa: E402
from fft_amd import rotary  # noqa: E402
from scan_reference import UNIT, close, half_step, tiny  # noqa: E402


def phases(plan, positions):
    """Radians of the plan's fixed-point frequencies, exact modulo one turn, in fp64."""
    words = [int(w) % 2 ** 64 for w in plan.turns.cpu().tolist()]
    flat = [int(p) for p in positions.cpu().flatten().tolist()]
    turns = [[((p * w + 2 ** 63) % 2 ** 64 - 2 ** 63) / 2.0 ** 64 for w in words] for p in flat]
    return 2.0 * math.pi * np.array(turns).reshape(tuple(positions.shape) + (len(words),))


def reference(plan, x, positions, pairs, inverse):
    """The rotated tensor in fp64 and the bound: cosine and sine are off by at most 4 units of 2^-24 (2 for the rounded
    argument, 2 for the functions), the magnitude's and the two products and the sum round once each, the result is stored once."""
    B, L = x.shape[:2]
    angle = phases(plan, positions.expand(B, L))[:, :, None, :]
    angle = torch.from_numpy(-angle if inverse else angle)
    c, s = plan.magnitude * angle.cos(), plan.magnitude * angle.sin()
    v, r = x.double().cpu(), plan.size
    first, second = (slice(0, r // 2), slice(r // 2, r)) if pairs == "half" else (slice(0, r, 2), slice(1, r, 2))
    re, im = v[..., first], v[..., second]
    want, off = v.clone(), torch.zeros_like(v)
    want[..., first], want[..., second] = re * c - im * s, re * s + im * c
    off[..., first] = off[..., second] = 7 * UNIT * abs(plan.magnitude) * (re.abs() + im.abs()) + tiny(x.dtype)
    off[..., :r] += half_step(x.dtype) * want[..., :r].abs()
    return want, off


def check(plan, x, positions, pairs="half", inverse=False, **kw):
    y = rotary.rotate(plan, x, positions=positions, pairs=pairs, inverse=inverse, **kw)
    close(y, *reference(plan, x, positions, pairs, inverse))
    return y


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("pairs", ["half", "interleaved"])
@pytest.mark.parametrize("B,L,H,P,size", [(1, 1, 1, 2, 2), (2, 3, 5, 64, 64), (1, 130, 3, 128, 128), (3, 1, 8, 128, 64), (2, 7, 1, 17, 6),
                                          (1, 9, 2, 80, 80), (2, 33, 4, 96, 48), (1, 5, 3, 256, 254), (1, 2, 70, 36, 34),
                                          (5, 1, 40, 128, 128), (1, 3, 2, 1001, 1000)])
def test_sizes(dtype, pairs, B, L, H, P, size):
    g = torch.Generator(device="cuda").manual_seed(P + L)
    plan = rotary.RotaryPlan(size)
    x = torch.randn(B, L, H, P, device="cuda", generator=g).to(dtype)
    positions = torch.randint(0, 100000, (B, L), device="cuda", generator=g)
    for inverse in (False, True):
        y = check(plan, x, positions, pairs, inverse)
        assert torch.equal(y[..., size:], x[..., size:])
    # the keys of the same tokens, with heads of their own number, give the same as on their own
    k = torch.randn(B, L, 3, P, device="cuda", generator=g).to(dtype)
    a, b = rotary.rotate(plan, x, k, positions, pairs=pairs)
    assert torch.equal(a, rotary.rotate(plan, x, positions=positions, pairs=pairs))
    assert torch.equal(b, rotary.rotate(plan, k, positions=positions, pairs=pairs))


def test_positions():
    plan = rotary.RotaryPlan(32)
    x = torch.randn(2, 50, 3, 32, device="cuda")
    row = torch.arange(50, device="cuda")
    y = check(plan, x, row.expand(2, 50))
    assert torch.equal(y, rotary.rotate(plan, x))
    assert torch.equal(y, rotary.rotate(plan, x, positions=row)) and torch.equal(y, rotary.rotate(plan, x, positions=row.int()))
    assert torch.equal(rotary.rotate(plan, x, first=77), rotary.rotate(plan, x, positions=row + 77))
    assert torch.equal(rotary.rotate(plan, x, positions=row.expand(2, 50).int()), y)
    wide = torch.zeros(50, 7, dtype=torch.int64, device="cuda")
    wide[:, 2] = row
    wide[:, 5] = row + 9
    check(plan, x, wide[:, 2::3].t())
    for far in (2 ** 20, 2 ** 31 - 30, 2 ** 40 + 12345, 2 ** 62):
        check(plan, x, row + far)
    check(plan, x, -row)
    # turning back by negative positions is the inverse
    assert torch.equal(rotary.rotate(plan, x, positions=-row), rotary.rotate(plan, x, positions=row, inverse=True))


def test_quarter_turns_are_exact():
    plan = rotary.RotaryPlan(8, frequencies=[math.pi / 2, math.pi, 2 * math.pi, 0.0])
    plan.turns.copy_(torch.tensor([2 ** 62, -2 ** 63, 0, 0]))
    x = torch.randn(1, 4, 1, 8, device="cuda")
    y = rotary.rotate(plan, x, pairs="interleaved")[0, :, 0]
    z = torch.view_as_complex(x[0, :, 0].reshape(4, 4, 2))
    for t in range(4):
        want = torch.stack([z[t, 0] * 1j ** t, z[t, 1] * (-1) ** t, z[t, 2], z[t, 3]])
        assert torch.equal(torch.view_as_complex(y[t].reshape(4, 2)), want)


def test_scalings():
    base, size, factor, context = 10000.0, 64, 4.0, 2048
    plain = np.array([base ** (-2 * i / size) for i in range(size // 2)])
    plans = {None: rotary.RotaryPlan(size), "linear": rotary.RotaryPlan(size, scaling="linear", factor=factor),
             "base": rotary.RotaryPlan(size, scaling="base", factor=factor),
             "ramp": rotary.RotaryPlan(size, scaling="ramp", factor=factor, original_length=context, magnitude=1.25),
             "given": rotary.RotaryPlan(size, frequencies=list(plain))}
    f = {name: np.array(p.frequencies) for name, p in plans.items()}
    assert np.array_equal(f[None], plain) and np.array_equal(f["given"], plain) and np.allclose(f["linear"] * factor, plain, rtol=1e-14)
    assert f["base"][0] == 1.0 and math.isclose(f["base"][-1] * factor, plain[-1], rel_tol=1e-12)
    turns = context * plain / (2 * math.pi)
    assert np.array_equal(f["ramp"][turns >= 32], plain[turns >= 32]) and np.allclose(f["ramp"][turns <= 1] * factor, plain[turns <= 1], rtol=1e-14)
    assert (np.diff(f["ramp"]) < 0).all()
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(2, 20, 3, 80, device="cuda", generator=g)
    positions = torch.randint(0, 50000, (2, 20), device="cuda", generator=g)
    for name, plan in plans.items():
        words = np.array([int(w) % 2 ** 64 for w in plan.turns.tolist()], dtype=np.float64) / 2.0 ** 64
        assert np.allclose(words, f[name] / (2 * math.pi), rtol=1e-15)
        for pairs in ("half", "interleaved"):
            check(plan, x, positions, pairs)


@pytest.mark.parametrize("pairs", ["half", "interleaved"])
def test_strides_and_places(pairs):
    """Heads before tokens, slices of a packed projection at odd offsets, in place, and framed results."""
    for dtype in (torch.float32, torch.bfloat16):
        g = torch.Generator(device="cuda").manual_seed(4)
        plan = rotary.RotaryPlan(24)
        positions = torch.randint(0, 9000, (2, 31), device="cuda", generator=g)
        packed = torch.randn(2, 31, 8 * 40 + 3, device="cuda", generator=g).to(dtype)
        q = packed[..., 1:1 + 5 * 40].unflatten(-1, (5, 40))
        k = packed[..., 1 + 5 * 40:1 + 8 * 40].unflatten(-1, (3, 40))
        y = check(plan, q, positions, pairs)
        heads_first = q.transpose(1, 2).contiguous().transpose(1, 2)
        assert torch.equal(check(plan, heads_first, positions, pairs), y)
        assert torch.equal(check(plan, q.expand(2, 31, 5, 40)[:, :, :1].expand(2, 31, 4, 40), positions, pairs)[:, :, 2], y[:, :, 0])
        frame = torch.full((2, 33, 7, 45), 7.0, device="cuda", dtype=dtype)
        rotary.rotate(plan, q, positions=positions, pairs=pairs, out=frame[:, 1:-1, 1:-1, 3:-2])
        assert torch.equal(frame[:, 1:-1, 1:-1, 3:-2], y) and int((frame == 7.0).sum()) == frame.numel() - y.numel()
        yk = check(plan, k, positions, pairs)
        before = packed.clone()
        rotary.rotate(plan, q, k, positions, pairs=pairs, out=q, out_k=k)
        assert torch.equal(q, y) and torch.equal(k, yk)
        assert torch.equal(packed[..., 0], before[..., 0]) and torch.equal(packed[..., 321:], before[..., 321:])


def test_there_and_back_and_gradient():
    """The inverse is the transpose of the rotation: <rotate(x), w> = <x, inverse(w)>, and a rotation keeps lengths."""
    g = torch.Generator(device="cuda").manual_seed(6)
    plan = rotary.RotaryPlan(48, magnitude=1.5)
    x, w = torch.randn(2, 40, 4, 64, device="cuda", generator=g), torch.randn(2, 40, 4, 64, device="cuda", generator=g)
    for pairs in ("half", "interleaved"):
        y, dx = rotary.rotate(plan, x, first=1000, pairs=pairs), rotary.rotate(plan, w, first=1000, pairs=pairs, inverse=True)
        a, b = (y.double() * w.double()), (x.double() * dx.double())
        # each side's terms are off by 8 units of at most 1.5 (|re| + |im|) |w|
        scale = 2 * 1.5 * float((x.double().abs().sum() * w.double().abs().max()))
        assert abs(float(a.sum() - b.sum())) <= 2 * 8 * UNIT * scale
        back = rotary.rotate(rotary.RotaryPlan(48), rotary.rotate(rotary.RotaryPlan(48), x, pairs=pairs), pairs=pairs, inverse=True)
        assert float((back - x).abs().max()) <= 32 * UNIT * float(x.abs().max())
        # differences: the rotation is linear, so a difference is the rotation of the difference
        step = torch.zeros_like(x)
        step[1, 7, 2, 5] = 1.0
        slope = rotary.rotate(plan, step, first=1000, pairs=pairs).double()
        assert abs(float((slope * w).sum()) - float(dx[1, 7, 2, 5])) <= 32 * UNIT * 1.5 * float(w.abs().max())


def test_empty():
    plan = rotary.RotaryPlan(8)
    for shape in ((0, 3, 2, 8), (2, 0, 2, 8), (2, 3, 0, 8)):
        x = torch.empty(shape, device="cuda")
        assert rotary.rotate(plan, x).shape == x.shape
    x = torch.randn(2, 3, 0, 8, device="cuda")
    k = torch.randn(2, 3, 2, 8, device="cuda")
    assert torch.equal(rotary.rotate(plan, x, k)[1], rotary.rotate(plan, k))


def test_streams_and_graphs():
    plan = rotary.RotaryPlan(64)
    q, k = torch.randn(3, 100, 8, 64, device="cuda").half(), torch.randn(3, 100, 2, 64, device="cuda").half()
    positions = torch.arange(100, device="cuda").expand(3, 100).clone()
    want = rotary.rotate(plan, q, k, positions)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [rotary.rotate(plan, q, k, positions, stream=s) for _ in range(4) for s in streams]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(want, g))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rotary.rotate(plan, q, k, positions)
    for step in range(4):
        positions += 17
        graph.replay()
        eager = rotary.rotate(plan, q, k, positions)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager))


def test_far_offsets():
    wide = torch.zeros(3, 2, 2 ** 30 + 64, device="cuda", dtype=torch.bfloat16)  # 12 GiB, rows past 2^32 elements
    plan = rotary.RotaryPlan(16)
    x = wide[:, :, 40:72].unflatten(-1, (2, 16))
    x.copy_(torch.randn(3, 2, 2, 16, device="cuda"))
    y = check(plan, x, torch.arange(6, device="cuda").view(3, 2))
    rotary.rotate(plan, x, positions=torch.arange(6, device="cuda").view(3, 2), out=x)
    assert torch.equal(x, y)


def test_refusals():
    plan = rotary.RotaryPlan(8)
    x = torch.zeros(2, 3, 2, 8, device="cuda")
    p = torch.zeros(2, 3, dtype=torch.int64, device="cuda")
    bad = [lambda: rotary.RotaryPlan(7), lambda: rotary.RotaryPlan(0), lambda: rotary.RotaryPlan(8, base=-1.0),
           lambda: rotary.RotaryPlan(8, scaling="other"), lambda: rotary.RotaryPlan(8, scaling="ramp"), lambda: rotary.RotaryPlan(8, factor=0.0),
           lambda: rotary.RotaryPlan(8, frequencies=[1.0]), lambda: rotary.RotaryPlan(8, frequencies=[1.0] * 4, scaling="linear"),
           lambda: rotary.RotaryPlan(8, frequencies=[float("nan")] * 4), lambda: rotary.RotaryPlan(8, magnitude=float("inf")),
           lambda: rotary.rotate(plan, x.cpu()), lambda: rotary.rotate(plan, x.double()), lambda: rotary.rotate(plan, x[0]),
           lambda: rotary.rotate(plan, x[..., :6]), lambda: rotary.rotate(plan, x, pairs="third"),
           lambda: rotary.rotate(plan, x, x.half()), lambda: rotary.rotate(plan, x, x[:1]), lambda: rotary.rotate(plan, x, x[..., :7]),
           lambda: rotary.rotate(plan, x, positions=p.float()), lambda: rotary.rotate(plan, x, positions=p[:, :2]),
           lambda: rotary.rotate(plan, x, positions=p.cpu()), lambda: rotary.rotate(plan, x, out=x.half()),
           lambda: rotary.rotate(plan, x, out=x[:1]), lambda: rotary.rotate(plan, x, out_k=x),
           lambda: rotary.rotate(plan, x, out=torch.zeros(2, 3, 8, 2, device="cuda").transpose(2, 3)),
           lambda: rotary.rotate(plan, torch.zeros(2, 3, 8, 2, device="cuda").transpose(2, 3)),
           lambda: rotary.rotate(plan, x, out=x[:, :, :1].expand(2, 3, 2, 8))]
    for i, call in enumerate(bad):
        with pytest.raises(fft_amd.ThunderFFTError):
            call()
            print("not refused:", i)
