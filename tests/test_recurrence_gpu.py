"""GPU tests of the gated linear recurrence (fft_amd.recurrence, tfft_scan_*) against the fp64 recurrence."""
import pytest

pytestmark = pytest.mark.gpu

import torch  # noqa: E402

import fft_amd  # noqa: E402
from fft_amd import recurrence  # noqa: E402
from scan_reference import close, scan, scan_grad  # noqa: E402

TYPES = [(torch.float32, torch.float32), (torch.float16, torch.float32), (torch.float16, torch.float16),
         (torch.bfloat16, torch.float32), (torch.bfloat16, torch.bfloat16)]


def make(B, L, D, share=1, dtype=torch.float32, gate_dtype=torch.float32, dim=1, log=True, seed=0, ragged=False, states=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    shape = (lambda n: (B, L, n)) if dim == 1 else (lambda n: (B, n, L))
    x = torch.randn(shape(D), device="cuda", generator=g).to(dtype)
    gate = -torch.exp(-6.9 * torch.rand(shape(D // share), device="cuda", generator=g))
    gate = (gate if log else gate.exp()).to(gate_dtype)
    lengths = torch.randint(0, L + 1, (B,), device="cuda", generator=g).int() if ragged else None
    initial = torch.randn(B, D, device="cuda", generator=g) if states else None
    dlast = torch.randn(B, D, device="cuda", generator=g) if states else None
    dy = torch.randn(shape(D), device="cuda", generator=g).to(dtype)
    return x, gate, lengths, initial, dlast, dy


def check_both(x, gate, lengths, initial, dlast, dy, dim, log):
    y, last = recurrence.gated_scan(x, gate, dim=dim, log_gate=log, lengths=lengths, initial=initial)
    want, bound, want_last, last_bound = scan(x, gate, dim, log, lengths, initial)
    close(y, want, bound, "y")
    close(last, want_last, last_bound, "last")
    got = recurrence.gated_scan_backward(dy, y, gate, dim=dim, log_gate=log, lengths=lengths, initial=initial, dlast=dlast)
    for name, a, (b, c) in zip(("dx", "dgate", "dinitial"), got, scan_grad(dy, y, gate, dim, log, lengths, initial, dlast)):
        assert a.dtype == {"dx": dy.dtype, "dgate": gate.dtype, "dinitial": torch.float32}[name]
        close(a, b, c, name)
    return y, last, got


# lengths of one token, around the wave's, the block's and several blocks' steps; channels below, at and beyond a tile
@pytest.mark.parametrize("dim", [1, 2])
@pytest.mark.parametrize("B,L,D", [(1, 1, 1), (2, 1, 5), (3, 2, 64), (1, 17, 257), (2, 63, 96), (5, 129, 33), (2, 1000, 70),
                                   (1, 4099, 12), (1, 9001, 3)])
def test_sizes(dim, B, L, D):
    for k, (dtype, gate_dtype) in enumerate(TYPES):
        check_both(*make(B, L, D, 1, dtype, gate_dtype, dim, log=k % 2 == 0, seed=L + k), dim, k % 2 == 0)


@pytest.mark.parametrize("dim", [1, 2])
@pytest.mark.parametrize("dtype,gate_dtype", TYPES)
@pytest.mark.parametrize("log", [False, True])
def test_padded_batch(dim, dtype, gate_dtype, log):
    for B, L, D in ((7, 301, 20), (4, 4500, 6), (9, 5, 130)):
        x, gate, lengths, initial, dlast, dy = make(B, L, D, 1, dtype, gate_dtype, dim, log, seed=L, ragged=True)
        lengths[0], lengths[1], lengths[2] = 0, L, 1
        check_both(x, gate, lengths, initial, dlast, dy, dim, log)


def test_padding_is_not_read():
    for dim in (1, 2):
        x, gate, _, initial, dlast, dy = make(4, 400, 10, dim=dim)
        lengths = torch.tensor([0, 400, 131, 1], dtype=torch.int32, device="cuda")
        y, last, grads = check_both(x, gate, lengths, initial, dlast, dy, dim, True)
        behind = torch.arange(400, device="cuda") >= lengths[:, None]
        behind = (behind[:, :, None] if dim == 1 else behind[:, None, :]).expand(x.shape)
        for value in (float("nan"), float("inf")):
            bad = [t.masked_fill(behind, value) for t in (x, gate, dy, y)]
            y2, last2 = recurrence.gated_scan(bad[0], bad[1], dim=dim, log_gate=True, lengths=lengths, initial=initial)
            grads2 = recurrence.gated_scan_backward(bad[2], bad[3], bad[1], dim=dim, log_gate=True, lengths=lengths,
                                                    initial=initial, dlast=dlast)
            assert torch.equal(y, y2) and torch.equal(last, last2)
            assert all(torch.equal(a, b) for a, b in zip(grads, grads2))
        # lengths outside 0 ... L count as the nearest of these
        wild = torch.tensor([-7, 2000000000, 131, 1], dtype=torch.int32, device="cuda")
        assert torch.equal(y, recurrence.gated_scan(x, gate, dim=dim, log_gate=True, lengths=wild, initial=initial)[0])


@pytest.mark.parametrize("share", [2, 3, 8, 48, 64, 128, 200, 512])
def test_shared_gates(share):
    for k, (dim, B, L, gates, ragged) in enumerate(((1, 2, 150, 3, False), (1, 3, 40, 1, True), (2, 2, 70, 2, False))):
        for dtype, gate_dtype in (TYPES[0], TYPES[3], TYPES[2]):
            check_both(*make(B, L, gates * share, share, dtype, gate_dtype, dim, log=k != 1, seed=share + k, ragged=ragged), dim, k != 1)


@pytest.mark.parametrize("share", [3, 6, 7, 10, 33, 48, 66, 96, 126, 130, 134, 200, 256])
@pytest.mark.parametrize("B,L,groups", [(5, 150, 1), (2, 37, 5), (40, 300, 3)])
def test_shares_that_are_no_power_of_two(share, B, L, groups):
    """Tiles that leave lanes of a wave empty, in one batch entry and over several, in one chunk and in more."""
    x, gate, lengths, initial, dlast, dy = make(B, L, groups * share, share, torch.float16, torch.float32, seed=share, ragged=True)
    check_both(x, gate, lengths, initial, dlast, dy, 1, True)


@pytest.mark.parametrize("share", [2, 3, 48, 64, 200])
def test_shared_gates_of_signals(share):
    """[batch, channel, time] with heads; lengths of every kind of chunking, and rows that lie apart."""
    for L in (1, 2, 7, 300, 517, 8193):
        x, gate, lengths, initial, dlast, dy = make(3, L, 2 * share if L < 1000 else share, share, torch.bfloat16, torch.float32, dim=2, seed=share + L,
                                                    ragged=True)
        check_both(x, gate, lengths, initial, dlast, dy, 2, True)
    x, gate, lengths, initial, dlast, dy = make(2, 203, 3 * share, share, torch.float32, torch.float32, dim=2, log=False)
    wide = torch.randn(2, 3 * share, 300, device="cuda")
    check_both(wide[:, :, 5:208], torch.nn.functional.pad(gate, (3, 9))[:, :, 3:206], None, initial, dlast, dy, 2, False)
    x, gate, lengths, initial, dlast, dy = make(3, 0, share, share, torch.bfloat16, torch.float32, dim=2)  # no steps: states pass through
    assert torch.equal(recurrence.gated_scan(x, gate, dim=2, initial=initial)[1], initial)
    assert torch.equal(recurrence.gated_scan_backward(dy, x, gate, dim=2, initial=initial, dlast=dlast)[2], dlast)


def test_no_states():
    for dim in (1, 2):
        check_both(*make(2, 300, 9, dim=dim, states=False), dim, True)


def test_length_zero():
    for dim in (1, 2):
        x, gate, _, initial, dlast, dy = make(3, 0, 6, dim=dim)
        y, last = recurrence.gated_scan(x, gate, dim=dim, initial=initial)
        assert y.shape == x.shape and torch.equal(last, initial)
        assert not recurrence.gated_scan(x, gate, dim=dim)[1].any()
        dx, dgate, dinitial = recurrence.gated_scan_backward(dy, y, gate, dim=dim, initial=initial, dlast=dlast)
        assert torch.equal(dinitial, dlast) and dx.numel() == 0 and dgate.numel() == 0
    empty = torch.empty(0, 5, 4, device="cuda")
    assert recurrence.gated_scan(empty, empty)[1].shape == (0, 4)
    empty = torch.empty(2, 5, 0, device="cuda")
    assert recurrence.gated_scan(empty, empty)[1].shape == (2, 0)


def test_strides():
    """Slices of a packed projection, transposed and stepped views, odd offsets, and gates broadcast by strides of 0."""
    for dtype in (torch.float32, torch.bfloat16):
        g = torch.Generator(device="cuda").manual_seed(1)
        B, L, D = 2, 333, 37
        packed = torch.randn(B, L, 3 * D + 1, device="cuda", generator=g).to(dtype)
        x, dy = packed[..., 1:1 + D], packed[..., 1 + D:1 + 2 * D]
        gate = -packed[..., 1 + 2 * D:].abs()
        views = [(x, gate, dy, 1), (x.transpose(1, 2), gate.transpose(1, 2), dy.transpose(1, 2), 2),
                 (x.transpose(1, 2).contiguous().transpose(1, 2), gate, dy, 1),
                 (packed[:, ::3, 0:2 * D:2], gate[:, ::3], packed[:, ::3, D:2 * D], 1),
                 (x.transpose(1, 2).contiguous()[..., 1:], gate.transpose(1, 2).contiguous()[..., 1:],
                  dy.transpose(1, 2).contiguous()[..., :-1], 2),
                 (x, gate[:1, :1].expand(B, L, D), dy, 1), (x, gate[..., :1].expand(B, L, D), dy, 1),
                 (x.transpose(1, 2).contiguous(), gate[:1, :1].transpose(1, 2).expand(B, D, L), dy.transpose(1, 2).contiguous(), 2)]
        for x, gt, dy, dim in views:
            check_both(x, gt, None, None, None, dy, dim, True)


def test_given_outputs():
    """In place, and into strided views whose surroundings stay as they were."""
    for dim in (1, 2):
        x, gate, lengths, initial, dlast, dy = make(3, 260, 18, dim=dim, ragged=True)
        y, last = recurrence.gated_scan(x, gate, dim=dim, log_gate=True, lengths=lengths, initial=initial)
        dx, dgate, _ = recurrence.gated_scan_backward(dy, y, gate, dim=dim, log_gate=True, lengths=lengths, initial=initial)
        x2 = x.clone()
        recurrence.gated_scan(x2, gate, dim=dim, log_gate=True, lengths=lengths, initial=initial, out=x2)
        assert torch.equal(x2, y)
        frame = torch.full((3, x.shape[1] + 2, x.shape[2] + 3), 7.0, device="cuda")
        recurrence.gated_scan(x, gate, dim=dim, log_gate=True, lengths=lengths, initial=initial, out=frame[:, 1:-1, 2:-1])
        assert torch.equal(frame[:, 1:-1, 2:-1], y)
        assert int((frame == 7.0).sum()) == frame.numel() - x.numel()
        dy2, frame = dy.clone(), torch.full_like(frame, 7.0)
        recurrence.gated_scan_backward(dy2, y, gate, dim=dim, log_gate=True, lengths=lengths, initial=initial, dx=dy2,
                                       dgate=frame[:, 1:-1, 2:-1])
        assert torch.equal(dy2, dx) and torch.equal(frame[:, 1:-1, 2:-1], dgate)
        assert int((frame == 7.0).sum()) == frame.numel() - x.numel()


def test_restarts():
    """A decay of zero (a log decay of minus infinity) starts a packed sequence anew: the same as its own call."""
    for dim in (1, 2):
        for log in (False, True):
            x, gate, _, _, _, dy = make(2, 700, 8, dim=dim, log=log, states=False)
            starts = [0, 1, 130, 131, 512, 699, 700]
            for s in starts[:-1]:
                gate.select(dim, s).fill_(float("-inf") if log else 0.0)
            y, _, (dx, dgate, _) = check_both(x, gate, None, None, None, dy, dim, log)
            for s, e in zip(starts, starts[1:]):
                want, bound, _, _ = scan(x.narrow(dim, s, e - s), gate.narrow(dim, s, e - s), dim, log)
                close(y.narrow(dim, s, e - s), want, bound, "part")


def test_signs_growth_and_specials():
    """Negative decays; growth that stays finite; products that underflow; a NaN stays in its channel, from its step on."""
    for dim in (1, 2):
        x, gate, _, initial, dlast, dy = make(2, 600, 6, dim=dim, log=False)
        check_both(x, -gate, None, initial, dlast, dy, dim, False)
        check_both(x, gate * 1e-20, None, initial, dlast, dy, dim, False)
        grown = torch.ones_like(gate) * 1.05
        check_both(x, grown, None, initial, dlast, dy, dim, False)
        # no state to multiply a large product with: zeros stay zeros
        big = recurrence.gated_scan(torch.zeros_like(x), torch.full_like(gate, 4.0), dim=dim)[0]
        assert not big.any()
        y, last = recurrence.gated_scan(x, gate, dim=dim)
        c = (0, 200, 3) if dim == 1 else (0, 3, 200)
        x[c] = float("nan")
        y2, last2 = recurrence.gated_scan(x, gate, dim=dim)
        a, b = (y, y2) if dim == 1 else (y.transpose(1, 2), y2.transpose(1, 2))
        assert torch.isnan(b[0, 200:, 3]).all() and torch.isnan(last2[0, 3])
        b[0, 200:, 3] = a[0, 200:, 3]
        assert torch.equal(a, b)


def test_gradient_against_differences():
    g = torch.Generator(device="cuda").manual_seed(5)
    for dim, share in ((1, 1), (1, 2), (2, 1)):
        shape = (lambda n: (2, 37, n)) if dim == 1 else (lambda n: (2, n, 37))
        x = torch.randn(shape(4), device="cuda", generator=g)
        gate = -torch.rand(shape(4 // share), device="cuda", generator=g)
        initial = torch.randn(2, 4, device="cuda", generator=g)
        dy, dlast = torch.randn(shape(4), device="cuda", generator=g), torch.randn(2, 4, device="cuda", generator=g)

        def loss(x, gate, initial):
            y, _, last, _ = scan(x, gate, dim, True, None, initial)
            return float((y * dy.double().cpu()).sum() + (last * dlast.double().cpu()).sum())

        y, _ = recurrence.gated_scan(x, gate, dim=dim, log_gate=True, initial=initial)
        grads = recurrence.gated_scan_backward(dy, y, gate, dim=dim, log_gate=True, initial=initial, dlast=dlast)
        inputs = [x.double(), gate.double(), initial.double()]
        for i, grad in enumerate(grads):
            for _ in range(4):
                way = torch.randn(inputs[i].shape, device="cuda", generator=g, dtype=torch.float64)
                far = [[t + s * 1e-4 * way if j == i else t for j, t in enumerate(inputs)] for s in (1, -1)]
                slope = (loss(*far[0]) - loss(*far[1])) / 2e-4
                # the difference is off by 1e-8 of the third derivative, the fp32 gradient by its bound: both far below
                assert abs(slope - float((grad.double() * way).sum())) <= 1e-4 * float((grad.double().abs() * way.abs()).sum())


@pytest.mark.parametrize("dtype,gate_dtype", TYPES)
@pytest.mark.parametrize("B,D,share", [(1, 1, 1), (1, 768, 1), (33, 130, 1), (64, 2048, 64), (3, 90, 3), (2, 6, 6)])
def test_step(dtype, gate_dtype, B, D, share):
    for log in (False, True):
        x, gate, _, state, _, _ = make(B, 1, D, share, dtype, gate_dtype, 1, log, seed=D)
        x, gate = x[:, 0], gate[:, 0]
        want, bound, want_last, last_bound = scan(x[:, None], gate[:, None], 1, log, None, state)
        fresh = torch.empty_like(state)
        y = recurrence.gated_scan_step(x, gate, state, log_gate=log, new_state=fresh)
        close(y, want[:, 0], bound[:, 0], "y")
        close(fresh, want_last, last_bound, "state")
        old = state.clone()
        y2 = recurrence.gated_scan_step(x, gate, state, log_gate=log)
        assert torch.equal(y, y2) and torch.equal(state, fresh)
        # rows of a wider pool, and y in the place of x
        pool = torch.zeros(B, D + 3, device="cuda")
        pool[:, 1:1 + D] = old
        wide = torch.zeros(B, D + 5, device="cuda", dtype=dtype)
        wide[:, 3:3 + D] = x
        recurrence.gated_scan_step(wide[:, 3:3 + D], gate, pool[:, 1:1 + D], log_gate=log, out=wide[:, 3:3 + D])
        assert torch.equal(wide[:, 3:3 + D], y) and torch.equal(pool[:, 1:1 + D], fresh)
        assert not pool[:, 0].any() and not pool[:, 1 + D:].any() and not wide[:, :3].any() and not wide[:, 3 + D:].any()


def test_prefill_then_steps():
    """A padded prefill, then tokens one by one, is the recurrence over the whole."""
    x, gate, _, _, _, _ = make(3, 90, 64, 4, torch.float32, torch.float32)
    lengths = torch.tensor([50, 0, 80], dtype=torch.int32, device="cuda")
    y, state = recurrence.gated_scan(x, gate, log_gate=True, lengths=lengths)
    rows = torch.arange(3, device="cuda")
    got = [recurrence.gated_scan_step(x[rows, lengths.long() + i], gate[rows, lengths.long() + i], state, log_gate=True)
           for i in range(10)]
    want, bound, _, _ = scan(x, gate, 1, True)
    for i, t in enumerate(got):
        at = (rows.cpu(), lengths.cpu().long() + i)
        close(t, want[at], bound[at], i)


def test_same_bits_again():
    x, gate, _, initial, dlast, dy = make(2, 5000, 300, 1, torch.bfloat16, torch.float32)
    for dim in (1, 2):
        t = (lambda v: v) if dim == 1 else (lambda v: v.transpose(1, 2).contiguous())
        first = None
        for _ in range(6):
            y, last = recurrence.gated_scan(t(x), t(gate), dim=dim, log_gate=True, initial=initial)
            now = [y, last, *recurrence.gated_scan_backward(t(dy), y, t(gate), dim=dim, log_gate=True, initial=initial, dlast=dlast)]
            first = first or now
            assert all(torch.equal(a, b) for a, b in zip(first, now))


def test_streams_and_graphs():
    """Calls on two other streams at once, and a captured forward and backward replayed with new inputs."""
    cases = [make(2, 5000, 200, 1, torch.bfloat16, torch.float32, dim, seed=dim) for dim in (1, 2)]

    def both(dim, x, gate, initial, dlast, dy, stream=None):
        y, last = recurrence.gated_scan(x, gate, dim=dim, log_gate=True, initial=initial, stream=stream)
        return [y, last, *recurrence.gated_scan_backward(dy, y, gate, dim=dim, log_gate=True, initial=initial, dlast=dlast, stream=stream)]

    want = [both(dim, x, g, i, dl, dy) for dim, (x, g, _, i, dl, dy) in zip((1, 2), cases)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[both(dim, x, g, i, dl, dy, s) for dim, s, (x, g, _, i, dl, dy) in zip((1, 2), streams, cases)] for _ in range(4)]
    torch.cuda.synchronize()
    for one in got:
        assert all(torch.equal(a, b) for w, o in zip(want, one) for a, b in zip(w, o))
    for dim, (x, g, _, i, dl, dy) in zip((1, 2), cases):
        x, dy = x.clone(), dy.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = both(dim, x, g, i, dl, dy)
        for seed in range(4):
            fresh = make(2, 5000, 200, 1, torch.bfloat16, torch.float32, dim, seed=40 + seed)
            x.copy_(fresh[0])
            dy.copy_(fresh[5])
            graph.replay()
            eager = both(dim, x, g, i, dl, dy)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, eager))


def test_two_graphs_at_once():
    """Two captured calls replayed on two streams at the same time have workspaces of their own."""
    cases = [make(1, 40000, 128, 1, torch.bfloat16, torch.bfloat16, seed=s) for s in (1, 2)]
    want = [recurrence.gated_scan(x, g, log_gate=True, initial=i) for x, g, _, i, _, _ in cases]
    graphs, outs = [torch.cuda.CUDAGraph() for _ in cases], []
    for graph, (x, g, _, i, _, _) in zip(graphs, cases):
        with torch.cuda.graph(graph):
            outs.append(recurrence.gated_scan(x, g, log_gate=True, initial=i))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        for stream, graph, out in zip(streams, graphs, outs):
            with torch.cuda.stream(stream):
                out[0].zero_()
                graph.replay()
        torch.cuda.synchronize()
        for w, o in zip(want, outs):
            assert torch.equal(w[0], o[0]) and torch.equal(w[1], o[1])


def test_far_offsets():
    """Views whose elements lie more than 2^32 bytes and 2^31 elements apart."""
    wide = torch.zeros(2, 40, 2 ** 26, device="cuda", dtype=torch.bfloat16)  # 10 GiB; the last rows lie past 2^32 elements
    g = torch.Generator(device="cuda").manual_seed(3)
    x = wide[:, :, 5:25]
    x.copy_(torch.randn(2, 40, 20, device="cuda", generator=g))
    gate = wide[:, :, 1000:1020]
    gate.copy_(-torch.rand(2, 40, 20, device="cuda", generator=g))
    dy = torch.randn(2, 40, 20, device="cuda", generator=g).bfloat16()
    check_both(x, gate, None, None, None, dy, 1, True)
    y = wide[:, :, 2 ** 26 - 20:]
    recurrence.gated_scan(x, gate, log_gate=True, out=y)
    assert torch.equal(y, recurrence.gated_scan(x.contiguous(), gate.contiguous(), log_gate=True)[0])


def test_refusals():
    x = torch.zeros(2, 8, 6, device="cuda")
    s = torch.zeros(2, 6, device="cuda")
    n = torch.zeros(2, dtype=torch.int32, device="cuda")
    bad = [lambda: recurrence.gated_scan(x.cpu(), x), lambda: recurrence.gated_scan(x, x.cpu()),
           lambda: recurrence.gated_scan(x.double(), x), lambda: recurrence.gated_scan(x, x.half()),
           lambda: recurrence.gated_scan(x.half(), x.bfloat16()), lambda: recurrence.gated_scan(x[0], x[0]),
           lambda: recurrence.gated_scan(x, x, dim=0), lambda: recurrence.gated_scan(x, x[..., :4]),
           lambda: recurrence.gated_scan(x, x[..., :0]), lambda: recurrence.gated_scan(x, x[:, :5]),
           lambda: recurrence.gated_scan(x, x[:1]), lambda: recurrence.gated_scan(x, x, initial=s[:1]),
           lambda: recurrence.gated_scan(x, x, initial=s.half()), lambda: recurrence.gated_scan(x, x, lengths=n.long()),
           lambda: recurrence.gated_scan(x, x, lengths=n[:1]), lambda: recurrence.gated_scan(x, x, lengths=n.cpu()),
           lambda: recurrence.gated_scan(x, x, out=x.half()), lambda: recurrence.gated_scan(x, x, out=x[:, :4]),
           lambda: recurrence.gated_scan(x, x, out=x[:, :1].expand(2, 8, 6)),
           lambda: recurrence.gated_scan_backward(x, x[:, :4], x), lambda: recurrence.gated_scan_backward(x, x.half(), x),
           lambda: recurrence.gated_scan_backward(x, x, x, dlast=s.t()), lambda: recurrence.gated_scan_backward(x, x, x, dgate=x[..., :3]),
           lambda: recurrence.gated_scan_step(x, x, s), lambda: recurrence.gated_scan_step(s, s, s.half()),
           lambda: recurrence.gated_scan_step(s, s[:, :4], s), lambda: recurrence.gated_scan_step(s, s, s[:, :3]),
           lambda: recurrence.gated_scan_step(s, s, torch.zeros(6, 2, device="cuda").t()),
           lambda: recurrence.gated_scan_step(s, s, s[:1].expand(2, 6))]
    for i, call in enumerate(bad):
        with pytest.raises(fft_amd.ThunderFFTError):
            call()
            print("not refused:", i)


@pytest.mark.parametrize("dim,B,L,D,share", [(1, 40, 700, 330, 1), (1, 3, 1300, 4100, 1), (1, 2, 2000, 384, 48), (1, 3, 900, 640, 128),
                                             (2, 9, 17000, 30, 1), (2, 40, 8211, 30, 1), (2, 2, 40000, 3, 1), (2, 1, 600000, 1, 1)])
def test_larger(dim, B, L, D, share):
    """Sizes at which tiles are dealt to the XCDs, rows are walked and chunks are taken apart, against the fp64
    recurrence in torch on the device, by norms: the fp32 roundings of memories of up to 1000 steps, 4 of 2^-24 a
    step, are 2.4e-4 at the very most, and random as they are a hundredth of that; 16-bit results add half a step."""
    for dtype, gate_dtype in ((torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.float16, torch.float16)):
        x, gate, lengths, initial, dlast, dy = make(B, L, D, share, dtype, gate_dtype, dim, seed=L, ragged=True)
        lengths[0] = L
        y, last = recurrence.gated_scan(x, gate, dim=dim, log_gate=True, lengths=lengths, initial=initial)
        got = recurrence.gated_scan_backward(dy, y, gate, dim=dim, log_gate=True, lengths=lengths, initial=initial, dlast=dlast)
        rows = (lambda t: t.transpose(1, 2)) if dim == 1 else (lambda t: t)
        inside = (torch.arange(L, device="cuda") < lengths[:, None])[:, None]
        a = torch.where(inside, rows(gate).double().exp().repeat_interleave(share, 1), 1.0)

        def run(a, v, h):  # [B, D, L] in stretches of 128 steps side by side, then joined
            n = -(-L // 128)
            pad = (0, n * 128 - L)
            a = torch.nn.functional.pad(a, pad, value=1.0).view(B, D, n, 128)
            v = torch.nn.functional.pad(v, pad).reshape(B, D, n, 128)
            out, product = torch.empty_like(v), torch.cumprod(a, -1)
            z = torch.zeros_like(v[..., 0])
            for t in range(128):
                z = a[..., t] * z + v[..., t]
                out[..., t] = z
            for j in range(n):
                out[:, :, j] += product[:, :, j] * h[..., None]
                h = out[:, :, j, -1]
            return out.view(B, D, n * 128)[..., :L]

        h = run(a, torch.where(inside, rows(x).double(), 0.0), initial.double())
        later = torch.cat([a[..., 1:], torch.ones_like(a[..., :1])], -1)
        e = run(later.flip(-1), torch.where(inside, rows(dy).double(), 0.0).flip(-1), dlast.double()).flip(-1)
        before = torch.cat([initial.double()[..., None], rows(y).double()[..., :-1]], -1)
        dgate = torch.where(inside, e * before * a, 0.0).reshape(B, D // share, share, L).sum(2)
        for name, t, want in (("y", rows(y), torch.where(inside, h, 0.0)), ("last", last, h[..., -1]), ("dx", rows(got[0]), torch.where(inside, e, 0.0)),
                              ("dgate", rows(got[1]), dgate), ("dinitial", got[2], a[..., 0] * e[..., 0])):
            off = float((t.double() - want).norm() / want.norm())
            assert off <= 2.4e-6 + torch.finfo(t.dtype).eps / 2, (name, dtype, off)
            assert torch.isfinite(t).all(), name


@pytest.mark.parametrize("dim,B,L,D,share", [(1, 1, 66003, 70, 1), (1, 2, 50000, 96, 48), (1, 3, 34000, 40, 1), (2, 20, 17000, 15, 1),
                                             (2, 3, 20000, 12, 4), (2, 40, 9000, 30, 10), (2, 16, 600, 512, 64)])
def test_long_with_few_channels(dim, B, L, D, share):
    """The same where groups of chunks are joined in rows of their own, and where a few hundred long signals are taken apart back."""
    test_larger(dim, B, L, D, share)


def test_places():
    """Tensors at one address are taken element for element or refused."""
    x, gate, _, _, _, dy = make(2, 50, 8, states=False)
    y, _ = recurrence.gated_scan(x, gate)
    square = torch.randn(2, 8, 8, device="cuda")
    bad = [lambda: recurrence.gated_scan(x, gate, out=gate), lambda: recurrence.gated_scan(square, square.clone(), out=square.transpose(1, 2)),
           lambda: recurrence.gated_scan_backward(dy, y, gate, dx=y), lambda: recurrence.gated_scan_backward(dy, y, gate, dx=gate),
           lambda: recurrence.gated_scan_backward(dy, y, gate, dgate=gate), lambda: recurrence.gated_scan_backward(dy, y, gate, dgate=dy),
           lambda: recurrence.gated_scan_step(x[:, 0], gate[:, 0], y[:, 0], out=y[:, 0])]
    for i, call in enumerate(bad):
        with pytest.raises(fft_amd.ThunderFFTError):
            call()
            print("not refused:", i)
