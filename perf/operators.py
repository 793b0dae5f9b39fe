"""The sequence operators beside the long convolution, as cases to be timed and compared.

Two operators, with every direction a program calls:

* the gated linear recurrence  h[t] = a[t] h[t-1] + x[t]  of every channel, over whole sequences (`scan`), its
  gradients (`scan_grad`) and one token of it (`step`); it is what the convolution of fft_amd.conv becomes when the
  decay depends on the input. "rows" is [batch, time, channel], "signals" the convolution's [batch, channel, time];
* rotary positions (`rotary`): pairs of a head's values times exp(i position frequency), for one tensor or for the
  queries and the keys of a layer together.

With `own` false, run() computes the plain form: elementary torch operations in fp32 (angles in fp64). With `own` true
it calls fft_amd.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"fp32": 4, "fp16": 2, "bf16": 2}


def listed():
    return [
        # one token of one sequence: a decoder that answers a single user, D = 768 (the model width of the
        # convolution benchmark). Latency alone counts.
        dict(name="step_one_token", op="step", batch=1, channels=768, share=1, dtype="bf16", gate="fp32", log=True),
        # one token of every sequence of a full serving batch
        dict(name="step_full_batch", op="step", batch=512, channels=4096, share=1, dtype="bf16", gate="bf16", log=True),
        # the forward pass of a training step: activations [B, L, D], log decays kept in fp32
        dict(name="scan_rows_train", op="scan", layout="rows", batch=8, length=4096, channels=2048, share=1,
             dtype="bf16", gate="fp32", log=True, ragged=False, initial=False),
        # one long document: few channels, so the work has to be split along the time axis; an odd length
        dict(name="scan_rows_long", op="scan", layout="rows", batch=1, length=65537, channels=1024, share=1,
             dtype="bf16", gate="bf16", log=True, ragged=False, initial=True),
        # prefill of a padded batch of short prompts, each behind its own state; odd sizes, decays instead of logs
        dict(name="scan_rows_ragged", op="scan", layout="rows", batch=16, length=517, channels=770, share=1,
             dtype="fp16", gate="fp32", log=False, ragged=True, initial=True),
        # the shape of the convolution benchmark: signals [B, D, N] in fp16
        dict(name="scan_signals_conv", op="scan", layout="signals", batch=64, length=4096, channels=768, share=1,
             dtype="fp16", gate="fp16", log=True, ragged=False, initial=False),
        # the backward pass of the training step above
        dict(name="grad_rows_train", op="scan_grad", layout="rows", batch=8, length=4096, channels=2048, share=1,
             dtype="bf16", gate="fp32", log=True, ragged=False, initial=False),
        # one decay per head of 64 channels, padded batch, a gradient of the last state too
        dict(name="grad_rows_heads", op="scan_grad", layout="rows", batch=4, length=8191, channels=2048, share=64,
             dtype="bf16", gate="fp32", log=True, ragged=True, initial=True),
        # a few very long signals (audio, genomes) in fp32, length near 2^20 and odd
        dict(name="grad_signals_long", op="scan_grad", layout="signals", batch=2, length=1048573, channels=8, share=1,
             dtype="fp32", gate="fp32", log=False, ragged=False, initial=False),
        # queries and keys of one new token of 64 sequences, at positions up to a million
        dict(name="rotary_decode", op="rotary", batch=64, length=1, heads=32, key_heads=8, head=128, rotary=128,
             dtype="bf16", pairs="half", scaling="none", far=True, inverse=False),
        # queries and keys of a training step
        dict(name="rotary_train", op="rotary", batch=8, length=4096, heads=32, key_heads=8, head=128, rotary=128,
             dtype="bf16", pairs="half", scaling="none", far=False, inverse=False),
        # gradients (the inverse rotation) of one fp32 tensor: interleaved pairs in half of the head, odd sizes,
        # frequencies stretched for a long context
        dict(name="rotary_grad_part", op="rotary", batch=3, length=3001, heads=12, key_heads=0, head=96, rotary=48,
             dtype="fp32", pairs="interleaved", scaling="ramp", far=True, inverse=True),
    ]


def _between(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["step", "scan", "scan", "scan_grad", "scan_grad", "rotary", "rotary"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "rotary":
        head = 2 * _between(rng, 8, 128)
        rotary = head if rng.random() < 0.6 else 2 * rng.randint(1, head // 2)
        heads, key_heads = _between(rng, 1, 64), rng.choice([0, 1, 2, 8])
        batch = _between(rng, 1, 128)
        length = _between(rng, 1, max(1, min(16384, 2 ** 27 // (batch * (heads + key_heads) * head))))
        return dict(op=op, batch=batch, length=length, heads=heads, key_heads=key_heads, head=head, rotary=rotary,
                    dtype=dtype, pairs=rng.choice(["half", "interleaved"]),
                    scaling=rng.choice(["none", "none", "linear", "base", "ramp"]), far=rng.random() < 0.5,
                    inverse=rng.random() < 0.4)
    share = rng.choice([1, 1, 1, 2, 8, 48, 64, 128])
    channels = share * max(1, _between(rng, 16, 4096) // share)
    gate = rng.choice(["fp32", dtype])
    if op == "step":
        return dict(op=op, batch=_between(rng, 1, 512), channels=channels, share=share, dtype=dtype, gate=gate,
                    log=rng.random() < 0.5)
    layout = rng.choice(["rows", "rows", "signals"])
    if layout == "signals":
        share = 1
    batch = _between(rng, 1, 64)
    length = _between(rng, 1, max(1, min(2 ** 18, 2 ** 26 // (batch * channels))))
    return dict(op=op, layout=layout, batch=batch, length=length, channels=channels, share=share, dtype=dtype,
                gate=gate, log=rng.random() < 0.5, ragged=rng.random() < 0.3, initial=rng.random() < 0.5)


def _frequencies(case):
    """Radians per position of every pair, in fp64."""
    size, base, factor, context = case["rotary"], 10000.0, 8.0, 8192.0
    if case["scaling"] == "base" and size > 2:  # the base grown so that the slowest pair is slowed by `factor`
        base = base * factor ** (size / (size - 2.0))
    f = base ** (-2.0 * torch.arange(size // 2, dtype=torch.float64) / size)
    if case["scaling"] == "linear":
        f = f / factor
    if case["scaling"] == "ramp":  # pairs with many turns in the old context keep their frequency, slow ones are stretched
        turns = context * f / (2.0 * math.pi)
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
        f = f * keep + f / factor * (1.0 - keep)
    return f


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, to=dtype):
        return torch.randn(*shape, device="cuda", generator=g).to(to)

    def uniform(*shape):
        return torch.rand(*shape, device="cuda", generator=g)

    if case["op"] == "rotary":
        B, L, P = case["batch"], case["length"], case["head"]
        if case["far"]:  # every sequence continues somewhere in a long context
            start = (uniform(B, 1).double() * 1000000.0).long()
        else:
            start = torch.zeros(B, 1, dtype=torch.int64, device="cuda")
        state = dict(case, q=normal(B, L, case["heads"], P),
                     k=normal(B, L, case["key_heads"], P) if case["key_heads"] else None,
                     positions=start + torch.arange(L, device="cuda"), frequencies=_frequencies(case).cuda(),
                     magnitude=0.1 * math.log(8.0) + 1.0 if case["scaling"] == "ramp" else 1.0)
        if own:  # the table that a program makes once from its configuration
            from fft_amd import rotary

            state["plan"] = rotary.RotaryPlan(
                case["rotary"], base=10000.0, scaling=None if case["scaling"] == "none" else case["scaling"],
                factor=1.0 if case["scaling"] == "none" else 8.0, original_length=8192, low_turns=1.0, high_turns=32.0,
                magnitude=state["magnitude"])
        return state
    B, D, G = case["batch"], case["channels"], case["channels"] // case["share"]
    L = case.get("length", 1)
    rows = case.get("layout", "rows") == "rows"
    shape = (lambda n: (B, n)) if case["op"] == "step" else (lambda n: (B, L, n) if rows else (B, n, L))
    # Memories of 1 to 1000 tokens: the log decay is spread over its logarithm.
    log = -torch.exp(uniform(*shape(G)) * -6.9)
    gate = (log if case["log"] else torch.exp(log)).to(DTYPES[case["gate"]])
    state = dict(case, gate=gate)
    if case["op"] == "step":
        return dict(state, x=normal(*shape(D)), state=normal(B, D, to=torch.float32))
    state["dim"] = 1 if rows else 2
    state["lengths"] = torch.randint(0, L + 1, (B,), device="cuda", generator=g).int() if case["ragged"] else None
    state["initial"] = normal(B, D, to=torch.float32) if case["initial"] else None
    if case["op"] == "scan":
        return dict(state, x=normal(*shape(D)))
    return dict(state, dy=normal(*shape(D)), y=normal(*shape(D)),
                dlast=normal(B, D, to=torch.float32) if case["initial"] else None)


def _behind(lengths, length, dim):
    """True at the padding behind each sequence, shaped to broadcast over [batch, ., .]."""
    behind = torch.arange(length, device=lengths.device) >= lengths[:, None]
    return behind[:, :, None] if dim == 1 else behind[:, None, :]


def _decays(s):
    """The decay of every channel, in fp32."""
    a = s["gate"].float()
    if s["log"]:
        a = torch.exp(a)
    return a.repeat_interleave(s["share"], dim=3 - s["dim"]) if s["share"] > 1 else a


def _running(a, x, dim):
    """x[t] <- a[t] x[t-1] + x[t] along `dim` by doubling: after the step of reach n, x[t] covers the last 2n inputs
    and a[t] is the product of as many decays. Overwrites its arguments."""
    n, length = 1, x.shape[dim]
    while n < length:
        late_a, late_x = a.narrow(dim, n, length - n), x.narrow(dim, n, length - n)
        carried = late_a * x.narrow(dim, 0, length - n)
        product = late_a * a.narrow(dim, 0, length - n)
        late_x += carried
        late_a.copy_(product)
        n *= 2
    return x


def _plain_scan(s):
    dim, L = s["dim"], s["x"].shape[s["dim"]]
    a, x = _decays(s), s["x"].float().clone()
    a = a.clone() if a.data_ptr() == s["gate"].data_ptr() else a
    if s["lengths"] is not None:
        behind = _behind(s["lengths"], L, dim)
        a.masked_fill_(behind, 1.0)
        x.masked_fill_(behind, 0.0)
    if s["initial"] is not None:
        x.select(dim, 0).add_(a.select(dim, 0) * s["initial"])
    h = _running(a, x, dim)
    last = h.select(dim, L - 1).clone()
    if s["lengths"] is not None:
        h.masked_fill_(behind, 0.0)
    return h.to(s["x"].dtype), last


def _plain_grad(s):
    dim, L = s["dim"], s["dy"].shape[s["dim"]]
    a, dy = _decays(s), s["dy"].float()
    if s["lengths"] is not None:
        behind = _behind(s["lengths"], L, dim)
        a = a.masked_fill(behind, 1.0)
        dy = dy.masked_fill(behind, 0.0)
    # c[t] = a[t] (dy[t] + c[t+1]) is what reaches h[t-1]; it runs backwards from the last state's gradient
    reverse_a, reverse_x = a.flip(dim), (a * dy).flip(dim)
    if s["dlast"] is not None:
        reverse_x.select(dim, 0).add_(reverse_a.select(dim, 0) * s["dlast"])
    c = _running(reverse_a, reverse_x, dim).flip(dim)
    dinitial = c.select(dim, 0).clone()
    end = torch.zeros_like(dinitial) if s["dlast"] is None else s["dlast"]
    dx = dy + torch.cat([c.narrow(dim, 1, L - 1), end.unsqueeze(dim)], dim)
    start = torch.zeros_like(dinitial) if s["initial"] is None else s["initial"]
    dgate = dx * torch.cat([start.unsqueeze(dim), s["y"].narrow(dim, 0, L - 1).float()], dim)
    if s["log"]:
        dgate = dgate * a
    if s["lengths"] is not None:
        dx = dx.masked_fill(behind, 0.0)
        dgate = dgate.masked_fill(behind, 0.0)
    if s["share"] > 1:
        dgate = dgate.unflatten(3 - dim, (-1, s["share"])).sum(4 - dim)
    return dx.to(s["dy"].dtype), dgate.to(s["gate"].dtype), dinitial


def _plain_step(s):
    a = s["gate"].float()
    if s["log"]:
        a = torch.exp(a)
    if s["share"] > 1:
        a = a.repeat_interleave(s["share"], dim=1)
    h = a * s["state"] + s["x"].float()
    return h.to(s["x"].dtype), h


def _plain_rotary(s, x, cos, sin):
    if x is None:
        return None
    r = s["rotary"]
    v = x[..., :r].float()
    if s["pairs"] == "half":
        re, im = v[..., :r // 2], v[..., r // 2:]
        turned = torch.cat([re * cos - im * sin, re * sin + im * cos], -1)
    else:
        re, im = v[..., 0::2], v[..., 1::2]
        turned = torch.stack([re * cos - im * sin, re * sin + im * cos], -1).flatten(-2)
    return torch.cat([turned.to(x.dtype), x[..., r:]], -1)


def run(state):
    s = state
    if s["op"] == "rotary":
        if own:
            from fft_amd import rotary

            turned = rotary.rotate(s["plan"], s["q"], s["k"], positions=s["positions"], pairs=s["pairs"],
                                   inverse=s["inverse"])
            return (turned, None) if s["k"] is None else turned
        angle = s["positions"][..., None].double() * s["frequencies"]
        if s["inverse"]:
            angle = -angle
        cos = (torch.cos(angle) * s["magnitude"]).float()[:, :, None]
        sin = (torch.sin(angle) * s["magnitude"]).float()[:, :, None]
        return _plain_rotary(s, s["q"], cos, sin), _plain_rotary(s, s["k"], cos, sin)
    if own:
        from fft_amd import recurrence

        if s["op"] == "scan":
            return recurrence.gated_scan(s["x"], s["gate"], dim=s["dim"], log_gate=s["log"], lengths=s["lengths"],
                                         initial=s["initial"])
        if s["op"] == "scan_grad":
            return recurrence.gated_scan_backward(s["dy"], s["y"], s["gate"], dim=s["dim"], log_gate=s["log"],
                                                  lengths=s["lengths"], initial=s["initial"], dlast=s["dlast"])
        h = torch.empty_like(s["state"])  # the old state is kept, as where a proposed token may be taken back
        return recurrence.gated_scan_step(s["x"], s["gate"], s["state"], log_gate=s["log"], new_state=h), h
    if s["op"] == "scan":
        return _plain_scan(s)
    return _plain_grad(s) if s["op"] == "scan_grad" else _plain_step(s)


def work(case):
    e, B = BYTES[case["dtype"]], case["batch"]
    if case["op"] == "rotary":
        L, tokens = case["length"], case["batch"] * case["length"]
        values = tokens * (case["heads"] + case["key_heads"]) * case["head"]
        turned = tokens * (case["heads"] + case["key_heads"]) * case["rotary"]
        return {"bytes": 2 * e * values + 8 * tokens + 8 * (case["rotary"] // 2), "flops": 3 * turned}
    D, G, ge = case["channels"], case["channels"] // case["share"], BYTES[case["gate"]]
    if case["op"] == "step":
        return {"bytes": B * (D * (2 * e + 8) + G * ge), "flops": 2 * B * D}
    n, states = B * case["length"], 4 * B * D
    small = (states if case["initial"] else 0) + (4 * B if case["ragged"] else 0) + states
    if case["op"] == "scan":
        return {"bytes": n * (2 * e * D + ge * G) + small, "flops": 2 * n * D}
    small += states if case["initial"] else 0  # the last state's gradient
    return {"bytes": n * (3 * e * D + 2 * ge * G) + small, "flops": 4 * n * D}


def _recurrence64(a, x, start):
    """h[t] = a[t] h[t-1] + x[t] along the last axis in fp64: stretches of 256 steps walked side by side, then joined
    one after the other."""
    length, m = x.shape[-1], 256
    pad = -length % m
    a = torch.nn.functional.pad(a, (0, pad), value=1.0).unflatten(-1, (-1, m))
    x = torch.nn.functional.pad(x, (0, pad)).unflatten(-1, (-1, m))
    h, product = torch.empty_like(x), torch.empty_like(a)
    for t in range(m):
        if t == 0:
            h[..., 0], product[..., 0] = x[..., 0], a[..., 0]
        else:
            h[..., t] = a[..., t] * h[..., t - 1] + x[..., t]
            product[..., t] = a[..., t] * product[..., t - 1]
    carry = start
    for j in range(h.shape[-2]):
        h[..., j, :] += product[..., j, :] * carry[..., None]
        carry = h[..., j, m - 1]
    return h.flatten(-2)[..., :length]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        r, m = case["rotary"], s["magnitude"]
        phase = torch.exp(1j * s["positions"].double()[:, :, None, None] * s["frequencies"])
        phase = m * (phase.conj() if case["inverse"] else phase)
        out = []
        for x in (s["q"], s["k"]):
            if x is None:
                out.append(None)
                continue
            y = x.double().clone()
            first, second = (slice(0, r // 2), slice(r // 2, r)) if case["pairs"] == "half" else (slice(0, r, 2), slice(1, r, 2))
            z = torch.complex(y[..., first], y[..., second]) * phase
            y[..., first], y[..., second] = z.real, z.imag
            out.append(y)
        return tuple(out)
    a = s["gate"].double()
    a = a.exp() if case["log"] else a
    if case["op"] == "step":
        h = torch.repeat_interleave(a, case["share"], 1) * s["state"].double() + s["x"].double()
        return h, h
    # channels before time, whatever the layout
    turn = (lambda t: t.transpose(1, 2).contiguous()) if case["layout"] == "rows" else (lambda t: t.contiguous())
    back = (lambda t: t.transpose(1, 2)) if case["layout"] == "rows" else (lambda t: t)
    a = torch.repeat_interleave(turn(a), case["share"], 1)
    B, D, L = a.shape
    inside = torch.ones(B, 1, L, dtype=torch.bool, device="cuda")
    if s["lengths"] is not None:
        inside = (torch.arange(L, device="cuda") < s["lengths"][:, None])[:, None]
        a = torch.where(inside, a, 1.0)
    zero = torch.zeros(B, D, dtype=torch.float64, device="cuda")
    start = zero if s["initial"] is None else s["initial"].double()
    if case["op"] == "scan":
        h = _recurrence64(a, torch.where(inside, turn(s["x"]).double(), 0.0), start)
        return back(torch.where(inside, h, 0.0)), h[..., -1]
    dy = torch.where(inside, turn(s["dy"]).double(), 0.0)
    end = zero if s["dlast"] is None else s["dlast"].double()
    # the gradient of h[t] is e[t] = dy[t] + a[t+1] e[t+1], with e[L] from the last state
    later = torch.cat([a[..., 1:], torch.ones_like(a[..., :1])], -1)
    e = _recurrence64(later.flip(-1), dy.flip(-1), end).flip(-1)
    before = torch.cat([start[..., None], turn(s["y"]).double()[..., :-1]], -1)
    dgate = e * before * (a if case["log"] else 1.0)
    dgate = torch.where(inside, dgate, 0.0).unflatten(1, (-1, case["share"])).sum(2)
    return back(torch.where(inside, e, 0.0)), back(dgate), a[..., 0] * e[..., 0]
