"""Gated linear recurrence h[t] = a[t] h[t-1] + x[t] over sequences: forward, gradients, one token at a time.

The sequence operator beside the long convolution of fft_amd.conv for decays that depend on the input. No counterpart
in the reference, whose convolutions have fixed taps (sample/conv1d/conv1d_fullfft_l4096_thunder.cu). Tensors stand in
for device pointers; the arithmetic, the padding rule and the layouts are those of tfft_scan_forward,
tfft_scan_backward and tfft_scan_step (include/thunderfft_c.h).

    y, last = gated_scan(x, gate)                               # x [B, L, D], gate [B, L, D] or [B, L, G], D = G share
    y, last = gated_scan(x, gate, dim=2)                        # the convolution's signals: x [B, D, L], gate [B, G, L]
    dx, dgate, dinitial = gated_scan_backward(dy, y, gate)      # y as gated_scan returned it
    y = gated_scan_step(x, gate, state)                         # x [B, D], gate [B, G], state fp32 [B, D], in place

Autograd does not see these calls: a torch.autograd.Function around gated_scan saves y and calls gated_scan_backward. Outside
one, a tensor that requires a gradient is taken for its values, with a warning while gradients are enabled.
"""
import ctypes
import warnings

import torch
from torch.autograd.graph import increment_version

from . import _lib
from .api import ThunderFFTError, _check

_FLOATS = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def _refuse(message, code=3):
    raise ThunderFFTError(code, message)


def _placed(call, device, stream, *args):
    """call(*args, raw stream) with torch's current device and stream those of the call, so that what it allocates belongs to
    the stream that it runs on. device: an index. Switching costs more than a short kernel, so it is left out where nothing
    changes."""
    if stream is None and device == torch._C._cuda_getDevice():
        return call(*args, torch._C._cuda_getCurrentRawStream(device))
    if stream is not None and stream.device.index != device:
        _refuse(f"{call.__name__.lstrip('_')}: the stream belongs to {stream.device}, the tensors to cuda:{device}")
    with torch.cuda.device(device):
        if stream is None:
            return call(*args, torch.cuda.current_stream(device).cuda_stream)
        with torch.cuda.stream(stream):
            return call(*args, stream.cuda_stream)


def _types(who, x, gate):
    code, gate_code = _FLOATS.get(x.dtype), _FLOATS.get(gate.dtype)
    if code is None or gate_code is None:
        _refuse(f"{who}: unsupported element types {x.dtype}, {gate.dtype}", 1)
    if gate_code not in (0, code):
        _refuse(f"{who}: the gate is float32 or of the values' type {x.dtype}, not {gate.dtype}", 1)
    return code, gate_code


def _same_device(who, x, *others):
    """Index of the device that all tensors lie on. Says so where the call cuts off the graph of one of them."""
    device, tracked = x.get_device(), x.requires_grad
    if device < 0:
        _refuse(f"{who} needs device tensors")
    for t in others:
        if t is not None:
            if t.get_device() != device:
                _refuse(f"{who}: tensors on {x.device} and {t.device}")
            if t.requires_grad:
                tracked = True
    if tracked and torch.is_grad_enabled():
        warnings.warn(f"{who}: autograd does not see this call, its results are cut off from the graph of a tensor that requires a "
                      "gradient (call it in a torch.autograd.Function, or under torch.no_grad())", stacklevel=3)
    return device


def _values(*tensors):
    """The tensors with their values in memory: torch only notes some negations (the imaginary part of a conjugated tensor),
    and what lies at their address has the other sign. Runs on the call's stream."""
    return [t if t is None else t.resolve_neg() for t in tensors]


def _state(who, name, t, B, D):
    if t is None:
        return 0
    if t.dtype != torch.float32 or t.shape != (B, D) or not t.is_contiguous():
        _refuse(f"{who}: {name} is a contiguous float32 tensor [{B}, {D}]")
    return t.data_ptr()


def _lengths(who, t, B):
    if t is None:
        return 0
    if t.dtype != torch.int32 or t.shape != (B,) or not t.is_contiguous():
        _refuse(f"{who}: lengths is a contiguous int32 tensor [{B}]")
    return t.data_ptr()


def _view(t, dim):
    b, p, q = t.stride()
    return (t.data_ptr(), b, p, q) if dim == 1 else (t.data_ptr(), b, q, p)


def _sizes(who, x, gate, dim):
    if dim not in (1, 2):
        _refuse(f"{who}: dim is 1 ([batch, time, channel]) or 2 ([batch, channel, time]), not {dim}")
    if x.dim() != 3 or gate.dim() != 3:
        _refuse(f"{who} needs tensors of three dimensions, got {tuple(x.shape)} and {tuple(gate.shape)}")
    shape, gates = x.shape, gate.shape
    B, L, D, G = shape[0], shape[dim], shape[3 - dim], gates[3 - dim]
    if gates[0] != B or gates[dim] != L or (D > 0 if G < 1 else D % G):
        _refuse(f"{who}: gate {tuple(gates)} does not fit {tuple(shape)}: the same batch and time, and a number of gates "
                "that divides the channels")
    return B, L, D, (D // G if G else 1)


def _out(who, name, t, like):
    if t is None:
        return torch.empty_like(like, memory_format=torch.contiguous_format)
    if t.dtype != like.dtype or t.shape != like.shape or t.is_neg():
        _refuse(f"{who}: {name} is a {like.dtype} tensor {tuple(like.shape)}, no negated view")
    increment_version(t)  # a tensor that autograd has saved and that is written into counts as changed
    return t


def _run(function, packer, values, forward, device, stream):
    """Workspace and launch; torch's current device and stream are already those of the call."""
    lib = _lib.load()
    need = ctypes.c_ulonglong()
    args = packer.pack(*values, 0, 0)
    rc = lib.tfft_scan_workspace_bytes(args if forward else None, None if forward else args, need)
    if rc:
        _check(rc)
    if need.value:
        # from torch's allocator on the call's stream: it is reused in stream order, and within a graph's own pool
        workspace = torch.empty(need.value, dtype=torch.uint8, device=device)
        args = packer.pack(*values, workspace.data_ptr(), need.value)
    rc = function(args, stream)
    if rc:
        _check(rc)


def gated_scan(x, gate, dim=1, log_gate=False, lengths=None, initial=None, out=None, stream=None):
    """(y, last): the recurrence over dimension `dim` of x, and the fp32 state [B, D] behind the last step.

    x: [B, L, D] (dim = 1) or [B, D, L] (dim = 2), float32, float16 or bfloat16, any strides. gate: the same with G
    channels, one for D / G neighbours, of x's type or float32; with log_gate the decay is exp(gate). Decays above 1 need
    a product over every stretch of steps, restarts or not, that is finite in fp32 (tfft_scan_forward). lengths (int32
    [B]): steps behind a sequence's length do not count, leave the state as it is, and y is 0 there. initial: fp32
    [B, D]. out: a tensor for y, x itself allowed. Inputs count by their values, a negation that torch has only noted
    (z.conj().imag) included; into such a view nothing is written. Asynchronous on `stream` (default: torch's current stream)."""
    return _placed(_gated_scan, _same_device("gated_scan", x, gate, lengths, initial, out), stream, x, gate, dim, log_gate,
                   lengths, initial, out)


def _gated_scan(x, gate, dim, log_gate, lengths, initial, out, stream):
    who = "gated_scan"
    if x.is_neg() or gate.is_neg() or (lengths is not None and lengths.is_neg()) or (initial is not None and initial.is_neg()):
        x, gate, lengths, initial = _values(x, gate, lengths, initial)
    code, gate_code = _types(who, x, gate)
    B, L, D, share = _sizes(who, x, gate, dim)
    y = _out(who, "out", out, x)
    last = torch.empty((B, D), dtype=torch.float32, device=x.device)
    _run(_lib.load().tfft_scan_forward, _lib.SCAN_ARGS,
         (_lib.SCAN_ARGS.size, code, gate_code, bool(log_gate), B, L, D, share, *_view(x, dim), *_view(gate, dim), *_view(y, dim),
          _lengths(who, lengths, B), _state(who, "initial", initial, B, D), last.data_ptr()), True, x.device, stream)
    return y, last


def gated_scan_backward(dy, y, gate, dim=1, log_gate=False, lengths=None, initial=None, dlast=None, dx=None, dgate=None,
                        stream=None):
    """(dx, dgate, dinitial): gradients of gated_scan from its output y (as stored), the gradient dy of y and, where
    the last state is used too, dlast (fp32 [B, D]).

    gate, dim, log_gate, lengths, initial: as the forward call had them. dgate has the gate's shape and type (the
    gradient of a gate that was broadcast by strides of 0 is the sum of it over those dimensions); dx and dgate may be
    given, dx may be dy. dinitial: fp32 [B, D]."""
    return _placed(_gated_scan_backward,
                   _same_device("gated_scan_backward", dy, y, gate, lengths, initial, dlast, dx, dgate), stream,
                   dy, y, gate, dim, log_gate, lengths, initial, dlast, dx, dgate)


def _gated_scan_backward(dy, y, gate, dim, log_gate, lengths, initial, dlast, dx, dgate, stream):
    who = "gated_scan_backward"
    if dy.is_neg() or y.is_neg() or gate.is_neg() or any([t.is_neg() for t in (lengths, initial, dlast) if t is not None]):
        dy, y, gate, lengths, initial, dlast = _values(dy, y, gate, lengths, initial, dlast)
    code, gate_code = _types(who, dy, gate)
    B, L, D, share = _sizes(who, dy, gate, dim)
    if y.dtype != dy.dtype or y.shape != dy.shape:
        _refuse(f"{who}: y is a {dy.dtype} tensor {tuple(dy.shape)} like dy")
    dx, dgate = _out(who, "dx", dx, dy), _out(who, "dgate", dgate, gate)
    dinitial = torch.empty((B, D), dtype=torch.float32, device=dy.device)
    _run(_lib.load().tfft_scan_backward, _lib.SCAN_GRAD_ARGS,
         (_lib.SCAN_GRAD_ARGS.size, code, gate_code, bool(log_gate), B, L, D, share, *_view(dy, dim), *_view(y, dim),
          *_view(gate, dim), *_view(dx, dim), *_view(dgate, dim), _lengths(who, lengths, B), _state(who, "initial", initial, B, D),
          _state(who, "dlast", dlast, B, D), dinitial.data_ptr()), False, dy.device, stream)
    return dx, dgate, dinitial


def gated_scan_step(x, gate, state, log_gate=False, new_state=None, out=None, stream=None):
    """y [B, D]: one token of the recurrence for every sequence. x: [B, D]; gate: [B, G]; state: fp32 [B, D], updated
    in place, or left as it is where new_state (fp32 [B, D]) is given. Rows may lie apart (any batch stride), the
    values of a row are contiguous."""
    return _placed(_gated_scan_step, _same_device("gated_scan_step", x, gate, state, new_state, out), stream, x, gate, state,
                   log_gate, new_state, out)


def _gated_scan_step(x, gate, state, log_gate, new_state, out, stream):
    who = "gated_scan_step"
    code, gate_code = _types(who, x, gate)
    shape, gates = x.shape, gate.shape
    if len(shape) != 2 or len(gates) != 2 or gates[0] != shape[0]:
        _refuse(f"{who} needs x [B, D] and gate [B, G], got {tuple(shape)} and {tuple(gates)}")
    B, D = shape
    G = gates[1]
    if D > 0 if G < 1 else D % G:
        _refuse(f"{who}: {G} gates do not divide {D} channels")
    if new_state is None:
        new_state = state
    if new_state.is_neg():
        _refuse(f"{who}: a state that is written into is no negated view")
    if x.is_neg() or gate.is_neg() or (state is not new_state and state.is_neg()):
        x, gate, state = _values(x, gate, state)
    for t in (state,) if new_state is state else (state, new_state):
        if t.dtype != torch.float32 or t.shape != shape:
            _refuse(f"{who}: state and new_state are float32 tensors [{B}, {D}]")
    y = _out(who, "out", out, x)
    rows = []
    for t in (x, gate, state, new_state, y):
        b, c = t.stride()
        if c != 1 and t.shape[1] > 1:
            _refuse(f"{who}: the values of a row are contiguous")
        rows.append(b)
    rc = _lib.load().tfft_scan_step(
        _lib.SCAN_STEP_ARGS.pack(_lib.SCAN_STEP_ARGS.size, code, gate_code, bool(log_gate), B, D, D // G if G else 1, x.data_ptr(),
                                 gate.data_ptr(), state.data_ptr(), new_state.data_ptr(), y.data_ptr(), *rows), stream)
    if rc:
        _check(rc)
    increment_version(new_state)
    return y
