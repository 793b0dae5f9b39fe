"""GPU tests of the sequence operators beside autograd, which does not see them: a call that cuts a graph off says so, and goes on."""
import warnings

import pytest

pytestmark = pytest.mark.gpu

import torch  # noqa: E402

from fft_amd import recurrence, rotary  # noqa: E402


def test_a_graph_that_is_cut_off_is_said():
    x, gate, s = torch.randn(2, 30, 4, device="cuda"), torch.rand(2, 30, 4, device="cuda"), torch.randn(2, 4, device="cuda")
    q, plan = torch.randn(2, 30, 1, 4, device="cuda"), rotary.RotaryPlan(4)
    leaf = lambda t: t.clone().requires_grad_()  # noqa: E731
    calls = [lambda f: recurrence.gated_scan(f(x), gate), lambda f: recurrence.gated_scan(x, f(gate)),
             lambda f: recurrence.gated_scan(x, gate, initial=f(s)), lambda f: recurrence.gated_scan_backward(f(x), x, gate),
             lambda f: recurrence.gated_scan_step(f(s), s, s.clone()), lambda f: rotary.rotate(plan, q, f(q))]
    for call in calls:
        with pytest.warns(UserWarning, match="autograd"):
            cut = call(leaf)
        with warnings.catch_warnings():
            warnings.simplefilter("error")
            plain = call(lambda t: t)
            with torch.no_grad():
                silent = call(leaf)
            with torch.inference_mode():
                call(leaf)
        for other in (cut, silent):  # and goes on as before
            pairs = zip(plain, other) if isinstance(plain, tuple) else [(plain, other)]
            assert all(torch.equal(a, b) for a, b in pairs)


def test_inside_a_function():
    """The way to a gradient: a torch.autograd.Function, where nothing is cut off."""

    class Scan(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, gate):
            y, last = recurrence.gated_scan(x, gate, log_gate=True)
            ctx.save_for_backward(y, gate)
            return y, last

        @staticmethod
        def backward(ctx, dy, dlast):
            y, gate = ctx.saved_tensors
            return recurrence.gated_scan_backward(dy, y, gate, log_gate=True, dlast=dlast.contiguous())[:2]

    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(1, 20, 3, device="cuda", generator=g).requires_grad_()
    gate = (-torch.rand(1, 20, 3, device="cuda", generator=g)).requires_grad_()
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        y, last = Scan.apply(x, gate)
        (y.square().sum() + last.sum()).backward()
    xr, gr = x.detach().double().cpu().requires_grad_(), gate.detach().double().cpu().requires_grad_()
    h, out = torch.zeros(1, 3, dtype=torch.float64), []
    for t in range(20):
        h = torch.exp(gr[:, t]) * h + xr[:, t]
        out.append(h)
    (torch.stack(out, 1).square().sum() + h.sum()).backward()
    # at most 20 steps of 8 roundings each way, of sums of at most 40 terms that are at most 10 times the gradients' norm
    for got, want in ((x.grad, xr.grad), (gate.grad, gr.grad)):
        assert float((got.double().cpu() - want).norm() / want.norm()) <= 2 * 20 * 8 * 2.0 ** -24 * 10
