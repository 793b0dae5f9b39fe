"""Signals of few steps in numbers that fill a launch: a wave holds several rows, and a launch counts what it really starts."""
import ctypes

import pytest

from fft_amd import _lib


def packed(B, D, L, share=1, backward=False):
    A, G = 1 << 20, D // share
    wide, narrow = (A, D * L, 1, L), (A, G * L, 1, L)
    pack = (_lib.SCAN_GRAD_ARGS, (wide, wide, narrow, wide, narrow), 4) if backward else (_lib.SCAN_ARGS, (wide, narrow, wide), 3)
    form, views, states = pack
    return form.pack(form.size, 1, 0, 1, B, L, D, share, *[v for view in views for v in view], *(0,) * states, 0, 0)


def limit(B, D, L, share=1):
    """Return codes for the workspaces of the two calls."""
    lib, need = _lib.load(), ctypes.c_ulonglong()
    return (lib.tfft_scan_workspace_bytes(packed(B, D, L, share), None, need),
            lib.tfft_scan_workspace_bytes(None, packed(B, D, L, share, True), need))


# fp16: a thread has 16 steps, a row of up to 512 has a power of two of threads, and a launch takes 2^32 - 2^16 of them
@pytest.mark.parametrize("L,lanes", [(2, 1), (16, 1), (17, 2), (100, 8), (257, 32), (512, 32)])
def test_rows_of_a_launch(L, lanes):
    for D in (4095, 4096):
        assert limit(4096, D, L) == (0, 0)
    most = 0xffff0000 // lanes
    rows = min(most // 4096 * 4096, (1 << 31) - (1 << 22))  # batch * (channels + 3) stays below 2^31 as well
    assert limit(rows // 4096, 4096, L) == (0, 0)
    if lanes >= 4:
        assert limit(rows // 4096 + 1, 4096, L) == (3, 3)


def test_rows_of_their_own_workgroups():
    """From 513 steps on in fp16 a row has a workgroup of 64 threads and more."""
    assert limit(4096, 4096, 513) == (0, 0) and limit(4096 * 16, 4096, 513) == (3, 3)


def test_shared_gates():
    """Backward a workgroup takes eight rows of a gate one after the other."""
    assert limit(4096, 4096, 100, 64) == (0, 0) and limit(4096, 4096, 2, 4) == (0, 0)


@pytest.mark.gpu
def test_results():
    import torch

    from fft_amd import recurrence

    g = torch.Generator(device="cuda").manual_seed(1)
    for share in (1, 8):
        B, D, L = 4096, 4104, 2
        x, dy = (torch.randn(B, D, L, device="cuda", generator=g).half() for _ in range(2))
        gate = torch.rand(B, D // share, L, device="cuda", generator=g)
        y, last = recurrence.gated_scan(x, gate, dim=2)
        dx, dgate, dinitial = recurrence.gated_scan_backward(dy, y, gate, dim=2)
        a = gate.repeat_interleave(share, 1)
        h = a[..., 1] * x[..., 0].float() + x[..., 1].float()
        e = dy[..., 0].float() + a[..., 1] * dy[..., 1].float()
        da = (dy[..., 1].float() * y[..., 0].float()).view(B, D // share, share)
        # h, e and each term of da are a product and a sum, 2^-24 of the terms' magnitudes each, here and in the kernel; stored once
        size, half = 2.0 ** -24, 2.0 ** -11
        assert torch.equal(y[..., 0], x[..., 0]) and torch.equal(dx[..., 1], dy[..., 1]) and not dgate[..., 0].any()
        wide = (a[..., 1] * x[..., 0].float()).abs() + x[..., 1].float().abs()
        assert ((last - h).abs() <= 4 * size * wide).all()
        assert ((y[..., 1].float() - h).abs() <= 4 * size * wide + half * h.abs() + 2.0 ** -25).all()
        wide = (a[..., 1] * dy[..., 1].float()).abs() + dy[..., 0].float().abs()
        assert ((dx[..., 0].float() - e).abs() <= 4 * size * wide + half * e.abs() + 2.0 ** -25).all()
        assert ((dinitial - a[..., 0] * e).abs() <= 6 * size * wide).all()
        assert ((dgate[..., 1] - da.sum(-1)).abs() <= 4 * share * size * da.abs().sum(-1)).all()
