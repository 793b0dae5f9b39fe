"""The gated recurrence and its gradients in fp64 on the CPU, step by step, with a bound on what fp32 arithmetic and one
rounding of the result may differ by.

Bound. h[t] is a sum of terms x[j] a[j+1] ... a[t]. Whatever the order of the products and sums, a term that travelled n
steps has passed at most n products, n sums and n decays, each of these off by at most one rounding, 2^-24 of
itself. The exponential of a log decay g is 2^(g log2 e): the power is off by one unit in the last place, two roundings, and the
rounded factor and product by at most 2^-25 + 2^-24 of |g log2 e|, which moves the result by 1.5 |g| ln 2 log2 e = 1.5 |g|
roundings. Joining the partial results adds at most a product and a sum for each level of the split, fewer than 8
levels. So |error| <= 2^-24 (4 N + 1.5 K + 24 H) with H the sum of the terms' magnitudes, N the same sum with every term
counted n times, K with every term counted as often as the sum of its |g| (0 for plain decays), and the stored value is
off by half a step of its type on top. All three sums are recurrences themselves."""
import numpy as np
import torch

UNIT = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half the distance of the smallest numbers of a type, which rounding may be off by whatever the value."""
    info = torch.finfo(dtype)
    return info.tiny * info.eps / 2


def _np(t):
    return None if t is None else t.detach().double().cpu().numpy()


def _time_first(t, dim):
    return np.moveaxis(t, dim, 0)  # [L, B, D]


def _decays(gate, dim, log, share, lengths):
    a = _time_first(_np(gate), dim)
    if log:
        a = np.exp(a)
    a = np.repeat(a, share, axis=2)
    L = a.shape[0]
    inside = np.ones(a.shape[:2], dtype=bool)
    if lengths is not None:
        inside = np.arange(L)[:, None] < np.clip(lengths.cpu().numpy(), 0, L)[None, :]
    # |g| of a log decay; a term that meets a decay of 0 is gone
    weight = np.where(a > 0, np.abs(np.log(np.maximum(a, 1e-300))), 0.0) if log else np.zeros_like(a)
    return a, weight, np.broadcast_to(inside[:, :, None], a.shape)


def scan(x, gate, dim=1, log=False, lengths=None, initial=None):
    """(y, y_bound, last, last_bound) as float64 tensors."""
    share = x.shape[3 - dim] // gate.shape[3 - dim]
    a, w, inside = _decays(gate, dim, log, share, lengths)
    v = _time_first(_np(x), dim)
    L, B, D = v.shape
    h = np.zeros((B, D)) if initial is None else _np(initial)
    H, N, K = np.abs(h), np.zeros((B, D)), np.zeros((B, D))
    y, bound = np.zeros((L, B, D)), np.zeros((L, B, D))
    for t in range(L):
        i = inside[t]
        N = np.where(i, np.abs(np.where(i, a[t], 0)) * (N + H), N)
        K = np.where(i, np.abs(np.where(i, a[t], 0)) * (K + np.where(i, w[t], 0) * H), K)
        H = np.where(i, np.abs(np.where(i, a[t], 0)) * H + np.abs(np.where(i, v[t], 0)), H)
        h = np.where(i, np.where(i, a[t], 0) * h + np.where(i, v[t], 0), h)
        y[t] = np.where(i, h, 0.0)
        bound[t] = np.where(i, UNIT * (4 * N + 1.5 * K + 24 * H) + half_step(x.dtype) * np.abs(h) + tiny(x.dtype), 0.0)
    back = lambda z: torch.from_numpy(np.ascontiguousarray(np.moveaxis(z, 0, dim)))  # noqa: E731
    last_bound = UNIT * (4 * N + 1.5 * K + 24 * H) + 1e-38
    return back(y), back(bound), torch.from_numpy(h.copy()), torch.from_numpy(last_bound)


def scan_grad(dy, y, gate, dim=1, log=False, lengths=None, initial=None, dlast=None):
    """[(value, bound)] of dx, dgate and dinitial as float64 tensors."""
    share = dy.shape[3 - dim] // gate.shape[3 - dim]
    a, w, inside = _decays(gate, dim, log, share, lengths)
    d, s = _time_first(_np(dy), dim), _time_first(_np(y), dim)
    L, B, D = d.shape
    c = np.zeros((B, D)) if dlast is None else _np(dlast)
    start = np.zeros((B, D)) if initial is None else _np(initial)
    H, N, K = np.abs(c), np.zeros((B, D)), np.zeros((B, D))
    dx, dx_bound = np.zeros((L, B, D)), np.zeros((L, B, D))
    da, da_bound = np.zeros((L, B, D)), np.zeros((L, B, D))
    for t in range(L - 1, -1, -1):
        i = inside[t]
        at = np.where(i, a[t], 0)
        e, He = np.where(i, d[t], 0) + c, np.abs(np.where(i, d[t], 0)) + H
        before = np.where(i, s[t - 1], 0) if t else start
        scale = at if log else 1.0
        off = UNIT * (4 * N + 1.5 * K + 24 * He)
        dx[t] = np.where(i, e, 0.0)
        dx_bound[t] = np.where(i, off + half_step(dy.dtype) * np.abs(e) + tiny(dy.dtype), 0.0)
        da[t] = np.where(i, e * before * scale, 0.0)
        # products with the stored state and the decay, the decay itself, and at most `share` sums
        da_bound[t] = np.where(i, np.abs(before * scale) * (off + UNIT * (6 + 1.5 * w[t] + share) * He), 0.0)
        N = np.where(i, np.abs(at) * (N + He), N)
        K = np.where(i, np.abs(at) * (K + np.where(i, w[t], 0) * He), K)
        H = np.where(i, np.abs(at) * He, H)
        c = np.where(i, at * e, c)
    G = D // share
    dgate, gate_bound = da.reshape(L, B, G, share).sum(-1), da_bound.reshape(L, B, G, share).sum(-1)
    gate_bound = gate_bound + half_step(gate.dtype) * np.abs(dgate) + tiny(gate.dtype)
    back = lambda z: torch.from_numpy(np.ascontiguousarray(np.moveaxis(z, 0, dim)))  # noqa: E731
    return [(back(dx), back(dx_bound)), (back(dgate), back(gate_bound)),
            (torch.from_numpy(c.copy()), torch.from_numpy(UNIT * (4 * N + 1.5 * K + 24 * H) + 1e-38))]


def close(got, want, bound, what=""):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.isfinite(got).all(), what
    over = (got - want).abs() - bound
    worst = over.argmax()
    assert over.max() <= 0, (what, "at", np.unravel_index(int(worst), tuple(want.shape)), float(got.flatten()[worst]),
                             float(want.flatten()[worst]), float(bound.flatten()[worst]))
