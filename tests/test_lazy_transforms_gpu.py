"""GPU tests of conjugated and negated views as operands of the transforms and convolutions: torch only notes them, the
data at their address is something else, so they are refused."""
import pytest

pytestmark = pytest.mark.gpu

import torch  # noqa: E402

import fft_amd  # noqa: E402
from fft_amd import conv  # noqa: E402


def test_transforms():
    z = torch.randn(3, 256, dtype=torch.complex64, device="cuda")
    want = fft_amd.fft(z.conj().resolve_conj())
    assert torch.equal(want, fft_amd.fft(z.conj().clone().resolve_conj()))
    pairs = torch.view_as_real(z).clone()
    bad = [lambda: fft_amd.fft(z.conj()), lambda: fft_amd.fft(torch._neg_view(z)), lambda: fft_amd.fft(torch._neg_view(pairs)),
           lambda: fft_amd.ThunderFFT_global(z, z.conj(), 3, 256), lambda: fft_amd.ThunderFFT_global(z.conj(), z, 3, 256),
           lambda: fft_amd.ThunderFFT_global(pairs, torch._neg_view(pairs), 3, 256)]
    before = z.clone()
    for i, call in enumerate(bad):
        with pytest.raises(fft_amd.ThunderFFTError):
            call()
            print("not refused:", i)
    assert torch.equal(z, before)


def test_convolutions():
    N, D = 4096, 2
    lazy = torch._neg_view
    h = torch.randn(D, N, 2, device="cuda") / N
    x = torch.randn(1, D, N, 2, device="cuda")
    perm = conv.filter_layout(h, N)
    half = h.half()
    signal, taps = torch.randn(500, 2, device="cuda"), torch.randn(9, 2, device="cuda")
    spectrum = conv.tiled_filter_spectrum(taps)
    bad = [lambda: conv.filter_layout(lazy(h), N), lambda: conv.filter_spectra_fused(lazy(half), N),
           lambda: conv.fft_conv(lazy(x), perm, N), lambda: conv.fft_conv(x, lazy(perm), N),
           lambda: conv.fft_conv(x, perm, N, out=lazy(x.clone())), lambda: conv.conv1d_tiled(lazy(signal), spectrum, 9),
           lambda: conv.conv1d_tiled(signal, lazy(spectrum), 9),
           lambda: conv.conv1d_tiled(signal, spectrum, 9, out=lazy(torch.zeros(492, 2, device="cuda")))]
    for i, call in enumerate(bad):
        with pytest.raises(fft_amd.ThunderFFTError):
            call()
            print("not refused:", i)
    # taps go through torch, which carries a noted negation out
    assert torch.equal(conv.filter_spectra(lazy(h), N), conv.filter_spectra(-h, N))
    assert torch.equal(conv.tiled_filter_spectrum(lazy(taps)), conv.tiled_filter_spectrum(-taps))


def test_distributed_shards():
    """The shard counts by its values, and no result is written into such a view."""
    from fft_amd import distributed

    plan = distributed.DistributedFFT(1 << 14, rank=0, world=1)
    x = torch.randn(1 << 14, 2, device="cuda")
    want = distributed.run_virtual([plan], [x])[0].clone()
    assert torch.equal(distributed.run_virtual([plan], [torch._neg_view(-x)])[0], want)
    with pytest.raises(ValueError):
        plan.transform(x, out=torch._neg_view(x.clone()))
