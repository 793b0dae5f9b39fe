"""CPU tests of the sequence operators' C entry points: argument structures, workspaces, refusals. Every call here is
refused before a launch, or has nothing to launch."""
import ctypes

import pytest

from fft_amd import _lib

F32, F16, BF16 = 0, 1, 2
OK, UNSUPPORTED, INVALID = 0, 1, 3
A = 1 << 20  # addresses that are looked at, never followed


def scan(dtype=BF16, gate_dtype=F32, form=1, B=2, L=100, D=64, share=1, x=None, gate=None, y=None, lengths=0, initial=0, last=A,
         workspace=A, workspace_bytes=1 << 40, size=_lib.SCAN_ARGS.size):
    G = D // share if share > 0 else D
    x = x or (A, L * D, D, 1)
    gate = gate or (2 * A, L * G, G, 1)
    y = y or (3 * A, L * D, D, 1)
    return _lib.SCAN_ARGS.pack(size, dtype, gate_dtype, form, B, L, D, share, *x, *gate, *y, lengths, initial, last, workspace, workspace_bytes)


def grad(dtype=BF16, gate_dtype=F32, form=1, B=2, L=100, D=64, share=1, views=None, size=_lib.SCAN_GRAD_ARGS.size, workspace=A,
         workspace_bytes=1 << 40, lengths=0):
    G = D // share
    wide, narrow = (L * D, D, 1), (L * G, G, 1)
    views = views or [(A, *wide), (2 * A, *wide), (3 * A, *narrow), (4 * A, *wide), (5 * A, *narrow)]
    flat = [v for view in views for v in view]
    return _lib.SCAN_GRAD_ARGS.pack(size, dtype, gate_dtype, form, B, L, D, share, *flat, lengths, 0, 0, A, workspace, workspace_bytes)


def step(dtype=BF16, gate_dtype=F32, form=1, B=2, D=64, share=1, places=(A, 2 * A, 3 * A, 3 * A, 4 * A), strides=None,
         size=_lib.SCAN_STEP_ARGS.size):
    return _lib.SCAN_STEP_ARGS.pack(size, dtype, gate_dtype, form, B, D, share, *places, *(strides or (D, D // share, D, D, D)))


def rotary(dtype=BF16, pairs=0, B=2, L=5, head=64, size_rotated=32, magnitude=1.0, position_bytes=8, turns=A, positions=2 * A,
           views=((3 * A, 4 * A, 4, 1280, 256, 64, 1280, 256, 64), (0,) * 9), size=_lib.ROTARY_ARGS.size):
    return _lib.ROTARY_ARGS.pack(size, dtype, pairs, 0, B, L, head, size_rotated, magnitude, position_bytes, turns, positions, L, 1, 0,
                                 *views[0], *views[1])


def workspace(forward=None, backward=None):
    need = ctypes.c_ulonglong(77)
    rc = _lib.load().tfft_scan_workspace_bytes(forward, backward, need)
    return rc, need.value


def refused(rc, code=INVALID):
    assert rc == code, (rc, _lib.load().tfft_last_error())
    assert len(_lib.load().tfft_last_error()) > 10


@pytest.mark.parametrize("changes,code", [
    (dict(size=8), INVALID), (dict(dtype=7), UNSUPPORTED), (dict(dtype=-1), UNSUPPORTED), (dict(dtype=F32, gate_dtype=BF16), UNSUPPORTED),
    (dict(gate_dtype=F16), UNSUPPORTED), (dict(form=2), INVALID), (dict(B=-1), INVALID), (dict(L=-1), INVALID), (dict(D=-4), INVALID),
    (dict(share=0), INVALID), (dict(share=3), INVALID), (dict(L=1 << 31), INVALID), (dict(B=1 << 20, D=1 << 20), INVALID),
    (dict(B=1 << 24, L=4096, D=64), INVALID), (dict(x=(0, 6400, 64, 1)), INVALID), (dict(x=(A + 1, 6400, 64, 1)), INVALID),
    (dict(gate=(A + 2, 6400, 64, 1)), INVALID), (dict(x=(A, -6400, 64, 1)), INVALID), (dict(x=(A, 1 << 61, 64, 1)), INVALID),
    (dict(y=(0, 6400, 64, 1)), INVALID), (dict(y=(A, 0, 64, 1)), INVALID), (dict(y=(3 * A, 6400, 0, 1)), INVALID),
    (dict(y=(3 * A, 6400, 63, 1)), INVALID), (dict(y=(3 * A, 64, 64, 1)), INVALID), (dict(y=(2 * A, 6400, 64, 1)), INVALID),
    (dict(y=(A, 1, 128, 2)), INVALID), (dict(last=A + 2), INVALID), (dict(initial=A + 1), INVALID), (dict(lengths=A + 2), INVALID),
    (dict(L=9000, workspace=0), INVALID), (dict(L=9000, workspace_bytes=8), INVALID), (dict(L=9000, workspace=A + 4), INVALID),
])
def test_forward_refusals(changes, code):
    refused(_lib.load().tfft_scan_forward(scan(**changes), None), code)


def test_null_arguments():
    lib = _lib.load()
    for call in (lib.tfft_scan_forward, lib.tfft_scan_backward, lib.tfft_scan_step, lib.tfft_rotary):
        refused(call(None, None))
    refused(workspace()[0])
    refused(workspace(scan(), grad())[0])
    refused(lib.tfft_scan_workspace_bytes(scan(), None, None))


@pytest.mark.parametrize("changes,code", [
    (dict(size=8), INVALID), (dict(dtype=9), UNSUPPORTED), (dict(gate_dtype=F16), UNSUPPORTED), (dict(form=-1), INVALID),
    (dict(L=9000, workspace=0), INVALID), (dict(share=200, D=400, workspace_bytes=8), INVALID)])
def test_backward_refusals(changes, code):
    refused(_lib.load().tfft_scan_backward(grad(**changes), None), code)


@pytest.mark.parametrize("place,with_place", [(4, 0), (4, 1), (4, 2), (4, 3), (3, 1), (3, 2)])
def test_backward_places(place, with_place):
    """An output at another tensor's address, but for dx at dy's."""
    views = [((i + 1) * A, 6400, 64, 1) for i in range(5)]
    views[place] = views[with_place]
    refused(_lib.load().tfft_scan_backward(grad(views=views), None))
    views = [((i + 1) * A, 6400, 64, 1) for i in range(5)]
    views[3] = (A, 64, 128, 1)
    refused(_lib.load().tfft_scan_backward(grad(views=views), None))


@pytest.mark.parametrize("changes,code", [
    (dict(size=8), INVALID), (dict(dtype=3), UNSUPPORTED), (dict(share=5), INVALID), (dict(B=-2), INVALID), (dict(B=1 << 20, D=1 << 20), INVALID),
    (dict(places=(0, 2 * A, 3 * A, 3 * A, 4 * A)), INVALID), (dict(places=(A, 0, 3 * A, 3 * A, 4 * A)), INVALID),
    (dict(places=(A, 2 * A, 3 * A + 2, 3 * A, 4 * A)), INVALID), (dict(places=(A, 2 * A, 3 * A, 0, 4 * A)), INVALID),
    (dict(places=(A, 2 * A, 3 * A, 3 * A, 2 * A)), INVALID), (dict(places=(A, 2 * A, 3 * A, A, 4 * A)), INVALID),
    (dict(places=(A, 2 * A, 3 * A, 3 * A, 3 * A)), INVALID), (dict(strides=(64, 64, 64, 32, 64)), INVALID),
    (dict(strides=(64, 64, 64, 128, 64)), INVALID), (dict(strides=(64, 64, 0, 0, 64)), INVALID), (dict(strides=(64, 64, 64, 64, 0)), INVALID)])
def test_step_refusals(changes, code):
    refused(_lib.load().tfft_scan_step(step(**changes), None), code)


VIEW = (3 * A, 4 * A, 4, 1280, 256, 64, 1280, 256, 64)
KEYS = (5 * A, 6 * A, 2, 640, 128, 64, 640, 128, 64)


@pytest.mark.parametrize("changes,code", [
    (dict(size=8), INVALID), (dict(dtype=4), UNSUPPORTED), (dict(pairs=2), INVALID), (dict(B=-1), INVALID), (dict(L=-1), INVALID),
    (dict(size_rotated=0), INVALID), (dict(size_rotated=31), INVALID), (dict(size_rotated=66), INVALID), (dict(position_bytes=2), INVALID),
    (dict(turns=0), INVALID), (dict(views=((0,) + VIEW[1:], KEYS)), INVALID), (dict(views=((3 * A + 1,) + VIEW[1:], KEYS)), INVALID),
    (dict(views=(VIEW[:1] + (0,) + VIEW[2:], KEYS)), INVALID), (dict(views=(VIEW[:2] + (-4,) + VIEW[3:], KEYS)), INVALID),
    (dict(views=(VIEW[:6] + (1280, 256, 0), KEYS)), INVALID), (dict(views=(VIEW[:6] + (1280, 64, 64), KEYS)), INVALID),
    (dict(views=((3 * A, 3 * A, 4, 1280, 256, 64, 320, 640, 64), KEYS)), INVALID),
    (dict(views=(VIEW, (5 * A, 4 * A) + KEYS[2:])), INVALID), (dict(views=(VIEW, (4 * A, 5 * A) + KEYS[2:])), INVALID),
    (dict(L=1 << 31), INVALID), (dict(B=1 << 20, L=1 << 20, views=((3 * A, 4 * A, 1, 1 << 26, 64, 64, 1 << 26, 64, 64), (0,) * 9)), INVALID)])
def test_rotary_refusals(changes, code):
    refused(_lib.load().tfft_rotary(rotary(**changes), None), code)


def test_nothing_to_do():
    lib = _lib.load()
    assert lib.tfft_scan_forward(scan(B=0), None) == OK and lib.tfft_scan_forward(scan(D=0, share=1), None) == OK
    assert lib.tfft_scan_backward(grad(B=0), None) == OK
    assert lib.tfft_scan_step(step(B=0), None) == OK
    assert lib.tfft_rotary(rotary(B=0), None) == OK and lib.tfft_rotary(rotary(L=0), None) == OK
    assert lib.tfft_rotary(rotary(views=((0, 0, 0) + VIEW[3:], (0,) * 9)), None) == OK


@pytest.mark.parametrize("empty", [dict(B=0), dict(B=0, L=0), dict(B=0, L=9000), dict(D=0)])
def test_an_empty_padded_batch(empty):
    lib = _lib.load()
    assert workspace(scan(lengths=A, **empty)) == (OK, 0) and lib.tfft_scan_forward(scan(lengths=A, **empty), None) == OK
    back = grad(lengths=A, **empty)
    assert workspace(backward=back) == (OK, 0) and lib.tfft_scan_backward(back, None) == OK


def test_workspaces():
    """None where a workgroup holds or walks the whole time axis; else counters, and 12 bytes a channel and chunk at most."""
    signals = dict(x=(A, 64 * 4096, 1, 4096), gate=(2 * A, 64 * 4096, 1, 4096), y=(3 * A, 64 * 4096, 1, 4096))
    assert workspace(scan(L=128)) == (OK, 0) and workspace(scan(L=0)) == (OK, 0) and workspace(scan(B=0, L=9000)) == (OK, 0)
    assert workspace(scan(L=4096, **signals)) == (OK, 0)
    many = dict(x=(A, 768 * 9000, 1, 9000), gate=(2 * A, 768 * 9000, 1, 9000), y=(3 * A, 768 * 9000, 1, 9000))
    assert workspace(scan(B=64, D=768, L=9000, **many)) == (OK, 0)
    rc, need = workspace(scan(B=8, L=4096, D=2048))
    assert rc == OK and 0 < need <= 12 * 8 * 2048 * 32 + 8 * 128
    rc, need = workspace(backward=grad(B=2, L=100, D=400, share=200))
    assert rc == OK and need == 4 * 2 * 100 * 4  # of gates whose channels a wave does not hold, the sums of halves
    assert workspace(backward=grad(B=2, L=100, D=96, share=48)) == (OK, 0)
    assert workspace(backward=grad(B=2, L=100, D=64, share=64)) == (OK, 0)
