"""The sequence operators as they are used together: a recurrence whose decay turns, h[t] = a[t] e^{i w} h[t-1] + x[t], is
the inputs turned back by their positions, the recurrence with the real decays, and the result turned forth. With a constant
decay it is the long convolution with the taps (a e^{i w})^k."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

import torch  # noqa: E402

from fft_amd import conv, recurrence, rotary  # noqa: E402
from scan_reference import UNIT  # noqa: E402


def turning_scan(plan, x, gate, first=0, **kw):
    """x [B, L, 2 D] (interleaved complex), gate [B, L, D] log decays."""
    B, L, P = x.shape
    back = rotary.rotate(plan, x.view(B, L, 1, P), pairs="interleaved", inverse=True, first=first).view(B, L, P)
    z, last = recurrence.gated_scan(back, gate, log_gate=True, **kw)
    return rotary.rotate(plan, z.view(B, L, 1, P), pairs="interleaved", first=first).view(B, L, P), last, z


def reference(x, gate, w):
    """The definition in complex128, with torch's gradients."""
    h, out = torch.zeros_like(x[:, 0]), []
    for t in range(x.shape[1]):
        h = torch.exp(gate[:, t] + 1j * w) * h + x[:, t]
        out.append(h)
    return torch.stack(out, 1)


def make(B, L, D, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(B, L, 2 * D, device="cuda", generator=g)
    gate = -torch.exp(-5.0 * torch.rand(B, L, D, device="cuda", generator=g))
    w = [float(v) for v in torch.linspace(0.01, 2.5, D)]
    return x, gate, w, rotary.RotaryPlan(2 * D, frequencies=w)


def test_constant_decays_are_the_long_convolution():
    N, L, B, D = 4096, 2048, 3, 6
    x, _, w, plan = make(B, L, D)
    decay = -torch.linspace(0.002, 0.5, D, device="cuda")
    h, _, _ = turning_scan(plan, x, decay.expand(B, L, D))
    k = np.arange(L)[None]
    taps = np.exp((decay.double().cpu().numpy()[:, None] + 1j * np.array(w)[:, None]) * k) / N
    taps = torch.from_numpy(np.stack([taps.real, taps.imag], -1)).float().cuda()
    signal = torch.zeros(B, D, N, 2, device="cuda")
    signal[:, :, :L] = x.view(B, L, D, 2).transpose(1, 2)
    y = conv.fft_conv(signal, conv.filter_spectra(taps, N), N, conv.CONV_COMPLEX)[:, :, :L].transpose(1, 2).reshape(B, L, 2 * D)
    # the convolution is within 1e-5 (its own tests), the recurrence's fp32 roundings of a memory of 500 steps within 4e-6
    assert float((h - y).double().norm() / y.double().norm()) <= 1.5e-5


def test_a_training_step():
    B, L, D = 2, 300, 5
    x, gate, w, plan = make(B, L, D, 1)
    weight = torch.randn_like(x)
    h, _, z = turning_scan(plan, x, gate)
    # backwards through the three calls
    dz = rotary.rotate(plan, weight.view(B, L, 1, 2 * D), pairs="interleaved", inverse=True).view(B, L, 2 * D)
    dback, dgate, _ = recurrence.gated_scan_backward(dz, z, gate, log_gate=True)
    dx = rotary.rotate(plan, dback.view(B, L, 1, 2 * D), pairs="interleaved").view(B, L, 2 * D)
    xr = x.double().cpu().view(B, L, D, 2).requires_grad_()
    gr = gate.double().cpu().requires_grad_()
    want = reference(torch.view_as_complex(xr), gr, torch.tensor(w, dtype=torch.float64))
    flat = torch.view_as_real(want).reshape(B, L, 2 * D)
    (flat * weight.double().cpu()).sum().backward()
    # a term of h meets two rotations (7 roundings each) and the recurrence's 4 a step over a memory of at most 150
    # steps: 614 roundings of 2^-24, or 4e-5, of the sums of magnitudes, which are within a factor of ten of the values' norm
    for got, exact in ((h, flat), (dx, xr.grad.reshape(B, L, 2 * D)), (dgate, gr.grad)):
        assert float((got.double().cpu() - exact.detach()).norm() / exact.detach().norm()) <= 614 * UNIT * 10


def test_prefill_and_tokens():
    """A padded prompt, then one token at a time at the positions that follow: the recurrence over the whole."""
    B, L, D, more = 3, 120, 4, 8
    x, gate, w, plan = make(B, L + more, D, 2)
    lengths = torch.tensor([120, 1, 77], dtype=torch.int32, device="cuda")
    prompt_h, state, _ = turning_scan(plan, x[:, :L].contiguous(), gate[:, :L], lengths=lengths)
    want = [torch.view_as_real(reference(torch.view_as_complex(x[b:b + 1].double().cpu().view(1, -1, D, 2)), gate[b:b + 1].double().cpu(),
                                         torch.tensor(w, dtype=torch.float64))).reshape(-1, 2 * D) for b in range(B)]
    rows = torch.arange(B, device="cuda")
    for b in range(B):
        n = int(lengths[b])
        assert float((prompt_h[b, :n].double().cpu() - want[b][:n]).norm() / want[b][:n].norm()) <= 614 * UNIT * 10
        assert not prompt_h[b, n:].any()
    for i in range(more):
        at = lengths.long() + i
        token, positions = x[rows, at].view(B, 1, 1, 2 * D), at.view(B, 1)
        back = rotary.rotate(plan, token, positions=positions, pairs="interleaved", inverse=True).view(B, 2 * D)
        z = recurrence.gated_scan_step(back, gate[rows, at], state, log_gate=True)
        h = rotary.rotate(plan, z.view(B, 1, 1, 2 * D), positions=positions, pairs="interleaved").view(B, 2 * D).double().cpu()
        exact = torch.stack([want[b][int(at[b])] for b in range(B)])
        assert float((h - exact).norm() / exact.norm()) <= 614 * UNIT * 10
