"""GPU tests of the gated recurrence with decays above 1: right as long as every stretch's product and states stay finite in fp32,
over restarts too."""
import pytest

pytestmark = pytest.mark.gpu

import torch  # noqa: E402

from fft_amd import recurrence  # noqa: E402
from scan_reference import close, scan, scan_grad  # noqa: E402


@pytest.mark.parametrize("dim", [1, 2])
@pytest.mark.parametrize("L", [60, 1000, 9000])
@pytest.mark.parametrize("share", [1, 2])
def test_growth_between_restarts(dim, L, share):
    g = torch.Generator(device="cuda").manual_seed(L)
    shape = (lambda n: (2, L, n)) if dim == 1 else (lambda n: (2, n, L))
    x, dy = torch.randn(shape(6), device="cuda", generator=g), torch.randn(shape(6), device="cuda", generator=g)
    initial, dlast = torch.randn(2, 6, device="cuda", generator=g), torch.randn(2, 6, device="cuda", generator=g)
    starts = torch.arange(L, device="cuda") % 60 == 0
    starts = starts[None, :, None] if dim == 1 else starts[None, None]
    # 4^59 = 3e35 in a stretch between restarts, and states of a few times as much
    gate = torch.where(starts, 0.0, 4.0).expand(shape(6 // share)).contiguous()
    y, last = recurrence.gated_scan(x, gate, dim=dim, initial=initial)
    want, bound, want_last, last_bound = scan(x, gate, dim, False, None, initial)
    close(y, want, bound, "y")
    close(last, want_last, last_bound, "last")
    # 2^59 each way, whose product is a gradient
    gate = torch.where(starts, 0.0, 2.0).expand(shape(6 // share)).contiguous()
    y, last = recurrence.gated_scan(x, gate, dim=dim, initial=initial)
    got = recurrence.gated_scan_backward(dy, y, gate, dim=dim, initial=initial, dlast=dlast)
    for name, a, (b, c) in zip(("dx", "dgate", "dinitial"), got, scan_grad(dy, y, gate, dim, False, None, initial, dlast)):
        close(a, b, c, name)
