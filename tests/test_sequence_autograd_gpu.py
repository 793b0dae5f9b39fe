"""GPU tests of the sequence operators beside autograd, which does not see them: tensors that a call writes into count as
changed."""
import pytest

pytestmark = pytest.mark.gpu

import torch  # noqa: E402

from fft_amd import recurrence, rotary  # noqa: E402


def changed(*tensors):
    return [t._version for t in tensors]


def test_written_tensors_count_as_changed():
    x, gate, s = torch.randn(2, 30, 4, device="cuda"), torch.rand(2, 30, 4, device="cuda"), torch.randn(2, 4, device="cuda")
    out, dx, dgate = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)
    y, _ = recurrence.gated_scan(x, gate)
    plan, q, k = rotary.RotaryPlan(4), torch.randn(2, 30, 2, 4, device="cuda"), torch.randn(2, 30, 1, 4, device="cuda")
    token, fresh, place = torch.randn(2, 4, device="cuda"), torch.empty(2, 4, device="cuda"), torch.empty(2, 4, device="cuda")
    cases = [(lambda: recurrence.gated_scan(x, gate), [], [x, gate]), (lambda: recurrence.gated_scan(x, gate, out=out), [out], [x, gate]),
             (lambda: recurrence.gated_scan_backward(x, y, gate, dx=dx, dgate=dgate), [dx, dgate], [x, y, gate]),
             (lambda: recurrence.gated_scan_step(token, token, s), [s], [token]),
             (lambda: recurrence.gated_scan_step(token, token, s, new_state=fresh, out=place), [fresh, place], [s, token]),
             (lambda: rotary.rotate(plan, q, k), [], [q, k]), (lambda: rotary.rotate(plan, q, k, out=q, out_k=k), [q, k], [plan.turns])]
    for call, written, read in cases:
        before = changed(*written, *read)
        call()
        after = changed(*written, *read)
        assert all(a > b for a, b in zip(after[:len(written)], before)), call
        assert after[len(written):] == before[len(written):], call


def test_a_saved_tensor_that_was_overwritten_is_noticed():
    leaf = torch.randn(2, 30, 4, device="cuda", requires_grad=True)
    x = leaf * 2.0
    loss = (x * x).sum()  # saves x
    recurrence.gated_scan(x.detach(), torch.rand(2, 30, 4, device="cuda"), out=x.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_inference_tensors():
    """They have no version; a state from a prefill in inference mode goes on outside it."""
    x, gate = torch.randn(2, 30, 4, device="cuda"), torch.rand(2, 30, 4, device="cuda")
    with torch.inference_mode():
        _, state = recurrence.gated_scan(x, gate)
        want = recurrence.gated_scan_step(x[:, 0], gate[:, 0], state.clone())
    assert state.is_inference() and torch.equal(recurrence.gated_scan_step(x[:, 0], gate[:, 0], state), want)
