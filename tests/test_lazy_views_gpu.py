"""GPU tests of tensors whose values torch has only noted: the imaginary part of a conjugated tensor is its negation, but
lies at the same address. The sequence operators take such inputs by their values and refuse to write into them; the
transforms, which take contiguous data as it lies, refuse them."""
import pytest

pytestmark = pytest.mark.gpu

import torch  # noqa: E402

import fft_amd  # noqa: E402
from fft_amd import recurrence, rotary  # noqa: E402


def negated(t):
    """A view with the values of t, which torch has noted as the negation of what lies there."""
    lies = torch.stack([torch.randn_like(t), -t], -1)
    if t.dtype == torch.bfloat16:  # no complex type has it: the view that conj().imag makes
        return torch._neg_view(lies[..., 1])
    view = torch.view_as_complex(lies).conj().imag
    assert view.is_neg() and torch.equal(view, t) and view.data_ptr() == lies[..., 1].data_ptr()
    return view


def dense(t):
    """The same with rows that are contiguous."""
    view = torch._neg_view(-t)
    assert view.is_neg() and torch.equal(view, t)
    return view


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [1, 2])
def test_recurrence(dtype, dim):
    g = torch.Generator(device="cuda").manual_seed(dim)
    shape = (2, 70, 6) if dim == 1 else (2, 6, 70)
    x, dy = torch.randn(shape, device="cuda", generator=g).to(dtype), torch.randn(shape, device="cuda", generator=g).to(dtype)
    gate = -torch.rand(shape, device="cuda", generator=g).to(dtype)
    initial, dlast = torch.randn(2, 6, device="cuda", generator=g), torch.randn(2, 6, device="cuda", generator=g)
    kw = dict(dim=dim, log_gate=True, initial=initial)
    y, last = recurrence.gated_scan(x, gate, **kw)
    want = recurrence.gated_scan_backward(dy, y, gate, dlast=dlast, **kw)
    for a, b in ((negated(x), gate), (x, negated(gate)), (negated(x), negated(gate)), (dense(x), dense(gate))):
        got = recurrence.gated_scan(a, b, **kw)
        assert torch.equal(got[0], y) and torch.equal(got[1], last)
    assert torch.equal(recurrence.gated_scan(x, gate, dim=dim, log_gate=True, initial=dense(initial))[0], y)
    for a, b, c in ((negated(dy), y, gate), (dy, negated(y), gate), (dy, y, negated(gate)), (negated(dy), negated(y), negated(gate))):
        assert all(torch.equal(u, v) for u, v in zip(recurrence.gated_scan_backward(a, b, c, dlast=dlast, **kw), want))
    kw["initial"] = dense(initial)
    assert all(torch.equal(u, v) for u, v in zip(recurrence.gated_scan_backward(dy, y, gate, dlast=dense(dlast), **kw), want))
    lengths = torch.tensor([-70, -3], dtype=torch.int32, device="cuda")
    padded = recurrence.gated_scan(x, gate, dim=dim, log_gate=True, lengths=-lengths)
    assert torch.equal(recurrence.gated_scan(x, gate, dim=dim, log_gate=True, lengths=torch._neg_view(lengths))[0], padded[0])


def test_step():
    g = torch.Generator(device="cuda").manual_seed(3)
    x, gate, state = (torch.randn(5, 12, device="cuda", generator=g) for _ in range(3))
    fresh, again = torch.empty_like(state), torch.empty_like(state)
    y = recurrence.gated_scan_step(x, gate, state, new_state=fresh)
    for a, b, c in ((dense(x), gate, state), (x, dense(gate), state), (x, gate, dense(state)), (negated(x), negated(gate), negated(state))):
        assert torch.equal(recurrence.gated_scan_step(a, b, c, new_state=again), y) and torch.equal(again, fresh)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_rotary(dtype):
    g = torch.Generator(device="cuda").manual_seed(4)
    plan = rotary.RotaryPlan(16)
    q, k = torch.randn(2, 9, 3, 24, device="cuda", generator=g).to(dtype), torch.randn(2, 9, 1, 24, device="cuda", generator=g).to(dtype)
    positions = torch.randint(0, 1000, (2, 9), device="cuda", generator=g)
    want = rotary.rotate(plan, q, k, positions)
    for a, b in ((dense(q), k), (q, dense(k)), (negated(q), negated(k))):
        assert all(torch.equal(u, v) for u, v in zip(rotary.rotate(plan, a, b, positions), want))
    assert torch.equal(rotary.rotate(plan, q, positions=torch._neg_view(-positions)), want[0])


def test_on_another_stream():
    """The values are settled on the stream of the call."""
    x, gate = torch.randn(4, 3000, 64, device="cuda"), -torch.rand(4, 3000, 64, device="cuda")
    view, want = negated(x), recurrence.gated_scan(x, gate, log_gate=True)[0]
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(4):
        y = recurrence.gated_scan(view, gate, log_gate=True, stream=stream)[0]
        stream.synchronize()
        assert torch.equal(y, want)


def test_nothing_is_written_into_them():
    x, gate, s = torch.randn(2, 30, 4, device="cuda"), torch.rand(2, 30, 4, device="cuda"), torch.randn(2, 4, device="cuda")
    plan, q = rotary.RotaryPlan(4), torch.randn(2, 30, 1, 4, device="cuda")
    y = recurrence.gated_scan(x, gate)[0]
    bad = [lambda: recurrence.gated_scan(x, gate, out=dense(x)), lambda: recurrence.gated_scan_backward(x, y, gate, dx=dense(x)),
           lambda: recurrence.gated_scan_backward(x, y, gate, dgate=dense(x)), lambda: recurrence.gated_scan_step(s, s, dense(s)),
           lambda: recurrence.gated_scan_step(s, s, s.clone(), out=dense(s)), lambda: recurrence.gated_scan_step(s, s, s, new_state=dense(s)),
           lambda: rotary.rotate(plan, q, out=dense(q)), lambda: rotary.rotate(plan, q, q, out_k=dense(q))]
    for i, call in enumerate(bad):
        with pytest.raises(fft_amd.ThunderFFTError):
            call()
            print("not refused:", i)
