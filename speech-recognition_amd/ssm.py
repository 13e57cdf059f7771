"""Trainable frame operators: the layers of an acoustic model that stands in front of the decoder.

The hidden Markov models of this package take frames as they come; a model that is trained by
gradients -- frames -> ``layer_norm`` -> projection -> ``causal_conv`` -> ``selective_scan`` ->
projection -> state log-densities -- gives ``viterbi_dense`` its emissions instead, and takes its targets
from ``HMMBank.posteriors``.  The reference has no such model; its own recursion over frames
(my_hmmlearn/utils.py:132-150) is the nearest relative of the scan.

Conventions of every function here:
  - frames are packed by utterance like ``Ragged.X``: (n_frames, channels), last dimension contiguous,
    rows at any pitch (a slice of a wider projection is taken as it is), float32, bfloat16 or float16;
  - ``offsets`` says where the utterances are: an int64 device tensor [U+1], a ``Ragged``, host
    numbers, or None for one utterance.  Rows outside offsets[0] .. offsets[U] belong to none: what they hold has
    no part in anything, they stay as they are in an ``out`` that is given, and are 0 in results that the
    functions make themselves and in gradients;
  - parameters, scan states and parameters' gradients are float32 whatever the frames are; arithmetic
    is in 32 bits, a result is rounded once;
  - work is queued on the current torch stream of the context's device.  Nothing is kept between calls
    and scratch comes from torch's allocator, so calls may be captured into graphs (but for those with host
    numbers as offsets, which copy them) and run on several streams of one context;
  - gradients are explicit: the ``*_backward`` functions are called with the gradient of the result,
    torch's autograd is not involved (a tensor that requires grad is refused while it records).
"""
import array
import ctypes as C

import numpy as np
import torch

from . import _lib
from ._lib import lib, check
from .runtime import Ragged, offsets_from_lengths

_CODES = {torch.float32: _lib.SRX_F32, torch.bfloat16: _lib.SRX_BF16, torch.float16: _lib.SRX_F16}
_ACTIVATIONS = {None: _lib.SRX_IDENTITY, "silu": _lib.SRX_SILU}


def _code(t, name):
    try:
        return _CODES[t.dtype]
    except KeyError:
        raise ValueError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}") from None


_TENSORS = {torch.Tensor, torch.nn.Parameter}


def _index(ctx):
    return -1 if ctx.device.index is None else ctx.device.index


def _on_device(ctx, t, name):
    if not isinstance(t, torch.Tensor) or t.device != ctx.device:
        raise ValueError(f"{name} must be a tensor on {ctx.device}")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires grad, which these functions do not record: detach it or call them "
                         "under torch.no_grad(), and use the *_backward functions")


# (The checks come before every launch, and a launch for a few live streams takes microseconds: what is in order is
# passed with one test of each property, the words for what is not are found afterwards.)

def _rows(ctx, t, name, shape, dtype, width):
    """Checks a matrix of rows, (n, ...) with `width` contiguous values a row; returns its pitch in elements."""
    if (isinstance(t, torch.Tensor) and t.shape == shape and t.dtype == dtype and t.device == ctx.device
            and t.is_contiguous() and not t.requires_grad):
        return width
    _on_device(ctx, t, name)
    if t.shape != shape:
        raise ValueError(f"Shape mismatch: {name} is {tuple(t.shape)}, expected {tuple(shape)}")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if t.is_contiguous():
        return width
    strides, want = t.stride(), 1
    for size, stride in zip(shape[:0:-1], strides[:0:-1]):
        if size > 1 and stride != want:
            raise ValueError(f"the rows of {name} must be contiguous")
        want *= size
    if shape[0] <= 1:
        return width
    if strides[0] < width:
        raise ValueError(f"the rows of {name} overlap")
    return strides[0]


def _parameter(ctx, t, name, shape):
    if t is None or (isinstance(t, torch.Tensor) and t.shape == shape and t.dtype == torch.float32
                     and t.device == ctx.device and t.is_contiguous() and not t.requires_grad):
        return t
    _on_device(ctx, t, name)
    if t.shape != shape:
        raise ValueError(f"Shape mismatch: {name} is {tuple(t.shape)}, expected {tuple(shape)}")
    if t.dtype != torch.float32:
        raise ValueError(f"{name} must be float32, got {t.dtype}")
    return t if t.is_contiguous() else t.contiguous()


def _state(ctx, t, name, shape, dtype):
    if t is None:
        return None
    _on_device(ctx, t, name)
    if t.shape != shape or t.dtype != dtype or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {tuple(shape)} {dtype} tensor")
    return t


def _offsets(ctx, offsets, n_frames):
    if isinstance(offsets, Ragged):
        if offsets.n_frames != n_frames:
            raise ValueError(f"Shape mismatch: {offsets.n_frames} frames in offsets, {n_frames} rows")
        offsets = offsets.offsets
    if isinstance(offsets, torch.Tensor):
        if offsets.dim() != 1 or offsets.numel() < 1 or offsets.dtype != torch.int64 or offsets.device != ctx.device:
            raise ValueError(f"offsets must be an int64 tensor [U+1] on {ctx.device}")
        return offsets.contiguous()
    if offsets is None:                             # (made on the device: nothing is copied or waited for)
        kind = dict(dtype=torch.int64, device=ctx.device)
        return torch.arange(0, 2 * n_frames, n_frames, **kind) if n_frames else torch.zeros(2, **kind)
    if ctx.device.type == "cuda":
        with torch.cuda.device(ctx.device):
            if torch.cuda.is_current_stream_capturing():
                raise ValueError("offsets in host memory would be copied while a graph is captured: give a device tensor")
    off = np.asarray(offsets, dtype=np.int64).reshape(-1)
    if off.size < 1 or off[0] < 0 or off[-1] > n_frames:
        raise ValueError(f"offsets must lie between 0 and {n_frames}")
    offsets_from_lengths(np.diff(off))              # (negative lengths are refused)
    return ctx.tensor(off)


def _extent(t):
    """(first byte, byte behind the last)"""
    begin, size = t.data_ptr(), t.element_size()
    if t.is_contiguous():
        return begin, begin + t.numel() * size
    return begin, begin + (sum((n - 1) * st for n, st in zip(t.shape, t.stride())) + 1) * size


def _apart(out, name, *inputs):
    """Refuses a result that shares memory with an input (rows of one wider matrix, side by side, do not)."""
    if out.numel() == 0:
        return
    a0, a1 = _extent(out)
    for t in inputs:
        if t is None:
            continue
        b0 = t.data_ptr()
        if b0 >= a1 or (t.is_contiguous() and b0 + t.nbytes <= a0) or t.numel() == 0:
            continue
        b0, b1 = _extent(t)
        if a0 >= b1:
            continue
        if out.dim() > 1 and t.dim() > 1 and out.shape[0] > 1 and t.shape[0] > 1:
            pitch, other = out.stride(0) * out.element_size(), t.stride(0) * t.element_size()
            width = a1 - a0 - (out.shape[0] - 1) * pitch
            wide = b1 - b0 - (t.shape[0] - 1) * other
            if pitch == other and 0 < width < pitch and width <= (b0 - a0) % pitch <= pitch - wide:
                continue
        raise ValueError(f"{name} shares memory with an input")


def _out(ctx, out, name, shape, dtype, inputs):
    """(the result's tensor, its pitch in elements); the first input has its type and shape"""
    if out is None:
        return _like(inputs[0]), shape[1]
    pitch = _rows(ctx, out, name, shape, dtype, shape[1])
    _apart(out, name, *inputs)
    return out, pitch


def _like(t):
    return None if t is None else torch.empty_like(t, memory_format=torch.contiguous_format)


def _address(t):
    return None if t is None else t.data_ptr()


def _workspace(ctx, nbytes):
    if nbytes < 0:
        check(_lib.SRX_EINVAL)
    return torch.empty((nbytes,), dtype=torch.uint8, device=ctx.device) if nbytes else None


# ---- selective state space scan ---------------------------------------------------------------

class _ScanCall:
    """The checked arguments that the three forms of the scan have in common."""

    def __init__(self, ctx, x, dt, A, B, C_, skip, gate, dt_bias, dt_softplus):
        if not (isinstance(x, torch.Tensor) and isinstance(A, torch.Tensor) and isinstance(B, torch.Tensor)
                and x.dim() == 2 and A.dim() == 2 and B.dim() in (2, 3)):
            self._refuse(ctx, x, A, B)
        self.code, dtype = _code(x, "x"), x.dtype
        n, c = rows = x.shape
        states = A.shape[1]
        groups = B.shape[1] if B.dim() == 3 else 1
        if groups < 1 or c % groups:
            raise ValueError(f"Shape mismatch: {c} channels in {groups} groups")
        wide = (n, groups, states) if B.dim() == 3 else (n, states)
        self.n, self.channels, self.states, self.groups = n, c, states, groups
        self.dtype, self.wide = dtype, wide
        A = _parameter(ctx, A, "A", (c, states))
        skip = _parameter(ctx, skip, "skip", (c,))
        dt_bias = _parameter(ctx, dt_bias, "dt_bias", (c,))
        self.keep = (A, skip, dt_bias)                   # (copies, where a parameter was not contiguous)
        self.scan = _lib.Scan(c, states, groups, 1 if dt_softplus else 0, A.data_ptr(), _address(skip),
                              _address(dt_bias))
        self.inputs = (x, dt, B, C_, gate)
        bc = groups * states
        pitches = (_rows(ctx, x, "x", rows, dtype, c), _rows(ctx, dt, "dt", rows, dtype, c),
                   _rows(ctx, B, "B", wide, dtype, bc), _rows(ctx, C_, "C", wide, dtype, bc),
                   0 if gate is None else _rows(ctx, gate, "gate", rows, dtype, c))
        self.rows = _lib.ScanInputs(x.data_ptr(), dt.data_ptr(), B.data_ptr(), C_.data_ptr(), _address(gate), *pitches)

    @staticmethod
    def _refuse(ctx, x, A, B):
        for t, name, dims, words in ((x, "x", (2,), "(n_frames, n_channels)"), (A, "A", (2,), "(n_channels, n_states)"),
                                     (B, "B", (2, 3), "(n_frames, n_states) or (n_frames, n_groups, n_states)")):
            if not isinstance(t, torch.Tensor):
                raise ValueError(f"{name} must be a tensor on {ctx.device}")
            if t.dim() not in dims:
                raise ValueError(f"{name} must be {'2-D ' if dims == (2,) else ''}{words}")


def selective_scan(ctx, x, dt, A, B, C, offsets=None, skip=None, gate=None, dt_bias=None, dt_softplus=True,
                   state=None, out=None, state_out=None, save=False):
    """For every utterance, with d = softplus(dt + dt_bias) (or dt + dt_bias without dt_softplus):

        h[t] = exp(d[t] A) h[t-1] + d[t] x[t] B[t],   y[t] = (C[t] . h[t] + skip x[t]) silu(gate[t])

    per channel c with its n_states states.  x, dt, gate: (n, channels); B, C: (n, states), or
    (n, groups, states) where channels // groups neighbouring channels share a group; A: (channels, states);
    skip, dt_bias: (channels,).  state: (U, channels, states) float32, the states before the first
    frames (zeros without it); state_out, which may be ``state`` itself, receives those behind the last
    frames (unchanged for an utterance without frames), so that a recording can come in pieces.  Up to 64
    states.  An A of minus infinity forgets at once; a step of 0 leaves a state as it is, whatever A is.  Returns (y, state_out), with save=True (y, state_out, saved): saved is what
    ``selective_scan_backward`` wants of this pass."""
    a = _ScanCall(ctx, x, dt, A, B, C, skip, gate, dt_bias, dt_softplus)
    off = _offsets(ctx, offsets, a.n)
    utts = off.numel() - 1
    shape = (utts, a.channels, a.states)
    state = _state(ctx, state, "state", shape, torch.float32)
    y, ld_y = _out(ctx, out, "out", (a.n, a.channels), a.dtype, (*a.inputs, *a.keep, state))
    if state_out is None:
        state_out = torch.empty(shape, dtype=torch.float32, device=ctx.device)
    else:
        _state(ctx, state_out, "state_out", shape, torch.float32)
        _apart(state_out, "state_out", *a.inputs, *a.keep, y, None if state_out is state else state)
    ws = _workspace(ctx, lib.srx_selective_scan_workspace(ctx.handle, _ref(a.scan), utts, a.n))
    saved = None
    if save:
        saved = torch.empty((lib.srx_selective_scan_saved(_ref(a.scan), utts, a.n),), dtype=torch.float32,
                            device=ctx.device)
    code = a.code if out is not None else a.code | _lib.SRX_ZERO_OTHER_ROWS
    check(lib.srx_selective_scan(ctx.handle, _ref(a.scan), _ref(a.rows), code, off.data_ptr(), utts, a.n,
                                 _address(state), state_out.data_ptr(), y.data_ptr(), ld_y,
                                 _address(saved), _address(ws), 0 if ws is None else ws.numel(),
                                 ctx.stream_ptr()), "srx_selective_scan")
    return (y, state_out, saved) if save else (y, state_out)


def selective_scan_backward(ctx, dy, x, dt, A, B, C, offsets=None, skip=None, gate=None, dt_bias=None,
                            dt_softplus=True, state=None, saved=None, dstate_out=None):
    """Gradients of ``selective_scan`` for the gradient dy of its y (and dstate_out of its
    state_out): a dict with x, dt, B, C, gate in the frames' type, A, skip, dt_bias and state in float32;
    None where an argument was not given.  saved: what the forward pass over the same arguments returned with
    save=True; without it that pass is run again here."""
    a = _ScanCall(ctx, x, dt, A, B, C, skip, gate, dt_bias, dt_softplus)
    off = _offsets(ctx, offsets, a.n)
    utts = off.numel() - 1
    shape = (utts, a.channels, a.states)
    state = _state(ctx, state, "state", shape, torch.float32)
    dstate_out = _state(ctx, dstate_out, "dstate_out", shape, torch.float32)
    ld_dy = _rows(ctx, dy, "dy", (a.n, a.channels), a.dtype, a.channels)
    size = lib.srx_selective_scan_saved(_ref(a.scan), utts, a.n)
    if saved is None:
        saved = selective_scan(ctx, x, dt, A, B, C, off, skip, gate, dt_bias, dt_softplus, state, save=True)[2]
    elif not (isinstance(saved, torch.Tensor) and saved.dtype == torch.float32 and saved.device == ctx.device
              and saved.shape == (size,) and saved.is_contiguous()):
        raise ValueError("saved must be what selective_scan(..., save=True) returned for these arguments")

    grads = {"x": _like(x), "dt": _like(dt), "A": _like(A), "B": _like(B), "C": _like(C), "skip": _like(skip),
             "gate": _like(gate), "dt_bias": _like(dt_bias), "state": _like(state)}
    bc = a.groups * a.states
    to = _lib.ScanGradients(grads["x"].data_ptr(), grads["dt"].data_ptr(), grads["B"].data_ptr(),
                            grads["C"].data_ptr(), _address(grads["gate"]), a.channels, a.channels, bc, bc,
                            a.channels)
    ws = _workspace(ctx, lib.srx_selective_scan_backward_workspace(ctx.handle, _ref(a.scan), utts, a.n))
    check(lib.srx_selective_scan_backward(ctx.handle, _ref(a.scan), _ref(a.rows), a.code, off.data_ptr(), utts, a.n,
                                          saved.data_ptr(), dy.data_ptr(), ld_dy, _address(dstate_out),
                                          _ref(to), grads["A"].data_ptr(), _address(grads["skip"]),
                                          _address(grads["dt_bias"]), _address(grads["state"]), ws.data_ptr(),
                                          ws.numel(), ctx.stream_ptr()), "srx_selective_scan_backward")
    return grads


def selective_scan_step(ctx, state, x, dt, A, B, C, skip=None, gate=None, dt_bias=None, dt_softplus=True,
                        out=None):
    """``selective_scan`` for one frame of each of n live streams: x, dt, gate (n, channels), B, C as there, state
    (n, channels, states) float32 moved on in place.  Returns y.  (Streams that have no frame this time
    go through ``selective_scan`` with utterances of no or one frame.)"""
    a = _ScanCall(ctx, x, dt, A, B, C, skip, gate, dt_bias, dt_softplus)
    if state is None:
        raise ValueError("state must be given")
    _state(ctx, state, "state", (a.n, a.channels, a.states), torch.float32)
    _apart(state, "state", *a.inputs, *a.keep)
    y, ld_y = _out(ctx, out, "out", (a.n, a.channels), a.dtype, (*a.inputs, *a.keep, state))
    check(lib.srx_selective_scan_step(ctx.handle, _ref(a.scan), _ref(a.rows), a.code, a.n, state.data_ptr(),
                                      y.data_ptr(), ld_y, ctx.stream_ptr()),
          "srx_selective_scan_step")
    return y


# ---- short causal convolution -----------------------------------------------------------------

class _ConvCall:
    def __init__(self, ctx, x, weight, bias, activation):
        if not isinstance(x, torch.Tensor) or x.dim() != 2:
            raise ValueError("x must be a 2-D (n_frames, n_channels) tensor")
        self.code = _code(x, "x")
        self.n, self.channels = rows = tuple(x.shape)
        if not isinstance(weight, torch.Tensor) or weight.dim() != 2:
            raise ValueError("weight must be a (n_channels, width) tensor")
        self.width = weight.shape[1]
        if not 1 <= self.width <= 8:
            raise ValueError(f"width {self.width} outside [1, 8]")
        if activation not in _ACTIVATIONS:
            raise ValueError(f"activation must be None or 'silu', got {activation!r}")
        weight = _parameter(ctx, weight, "weight", (self.channels, self.width))
        bias = _parameter(ctx, bias, "bias", (self.channels,))
        self.keep = (weight, bias)
        self.ld = _rows(ctx, x, "x", rows, x.dtype, self.channels)
        self.conv = _lib.Conv(self.channels, self.width, _ACTIVATIONS[activation], 0, weight.data_ptr(),
                              _address(bias))


def causal_conv(ctx, x, weight, offsets=None, bias=None, activation=None, state=None, out=None, state_out=None):
    """y[t, c] = act(bias[c] + sum_k weight[c, k] x[t - width + 1 + k, c]) inside every utterance; x (n, channels),
    weight (channels, width <= 8), activation None or "silu".  state: (U, width - 1, channels) in x's type, the
    frames before the utterances, oldest first (zeros without it); state_out, which may be ``state`` itself,
    receives the last width - 1 frames.  Returns (y, state_out)."""
    a = _ConvCall(ctx, x, weight, bias, activation)
    off = _offsets(ctx, offsets, a.n)
    utts = off.numel() - 1
    shape = (utts, a.width - 1, a.channels)
    state = _state(ctx, state, "state", shape, x.dtype)
    y, ld_y = _out(ctx, out, "out", (a.n, a.channels), x.dtype, (x, *a.keep, state))
    if state_out is None:
        state_out = torch.empty(shape, dtype=x.dtype, device=ctx.device)
    else:
        _state(ctx, state_out, "state_out", shape, x.dtype)
        _apart(state_out, "state_out", x, *a.keep, y, None if state_out is state else state)
    code = a.code if out is not None else a.code | _lib.SRX_ZERO_OTHER_ROWS
    check(lib.srx_causal_conv(ctx.handle, _ref(a.conv), code, x.data_ptr(), a.ld, off.data_ptr(), utts, a.n,
                              _address(state), state_out.data_ptr(), y.data_ptr(), ld_y,
                              ctx.stream_ptr()), "srx_causal_conv")
    return y, state_out


def causal_conv_backward(ctx, dy, x, weight, offsets=None, bias=None, activation=None, state=None,
                         dstate_out=None):
    """Gradients of ``causal_conv`` for the gradient dy of its y (and dstate_out of its state_out, in x's type):
    a dict with x and state in x's type, weight and bias in float32; None where an argument was not given."""
    a = _ConvCall(ctx, x, weight, bias, activation)
    off = _offsets(ctx, offsets, a.n)
    utts = off.numel() - 1
    shape = (utts, a.width - 1, a.channels)
    state = _state(ctx, state, "state", shape, x.dtype)
    dstate_out = _state(ctx, dstate_out, "dstate_out", shape, x.dtype)
    ld_dy = _rows(ctx, dy, "dy", (a.n, a.channels), x.dtype, a.channels)
    grads = {"x": _like(x), "weight": _like(weight), "bias": _like(bias), "state": _like(state)}
    ws = _workspace(ctx, lib.srx_causal_conv_backward_workspace(ctx.handle, _ref(a.conv), utts, a.n))
    check(lib.srx_causal_conv_backward(ctx.handle, _ref(a.conv), a.code, x.data_ptr(), a.ld, off.data_ptr(), utts,
                                       a.n, _address(state), dy.data_ptr(), ld_dy, _address(dstate_out),
                                       grads["x"].data_ptr(), a.channels, grads["weight"].data_ptr(),
                                       _address(grads["bias"]), _address(grads["state"]), ws.data_ptr(),
                                       ws.numel(), ctx.stream_ptr()), "srx_causal_conv_backward")
    return grads


def causal_conv_step(ctx, state, x, weight, bias=None, activation=None, out=None):
    """``causal_conv`` for one frame of each of n live streams: x (n, channels), state (n, width - 1, channels) in x's
    type, moved on in place.  Returns y."""
    a = _ConvCall(ctx, x, weight, bias, activation)
    if state is None:
        raise ValueError("state must be given")
    _state(ctx, state, "state", (a.n, a.width - 1, a.channels), x.dtype)
    _apart(state, "state", x, *a.keep)
    y, ld_y = _out(ctx, out, "out", (a.n, a.channels), x.dtype, (x, *a.keep, state))
    check(lib.srx_causal_conv_step(ctx.handle, _ref(a.conv), a.code, x.data_ptr(), a.ld, a.n, state.data_ptr(),
                                   y.data_ptr(), ld_y, ctx.stream_ptr()), "srx_causal_conv_step")
    return y


# ---- layer norm ---------------------------------------------------------------------------------

def layer_norm(ctx, x, weight=None, bias=None, eps=1e-5, out=None):
    """y = (x - mean) rstd weight + bias for every row of x (n, features), rstd = 1 / sqrt(variance + eps) with the
    variance over n values.  Returns (y, mean, rstd), the last two (n,) float32: what
    ``layer_norm_backward`` wants of this pass."""
    if not isinstance(x, torch.Tensor) or x.dim() != 2:
        raise ValueError("x must be a 2-D (n_rows, n_features) tensor")
    n, d = rows = tuple(x.shape)
    code, ld = _code(x, "x"), _rows(ctx, x, "x", rows, x.dtype, d)
    weight, bias = _parameter(ctx, weight, "weight", (d,)), _parameter(ctx, bias, "bias", (d,))
    y, ld_y = _out(ctx, out, "out", rows, x.dtype, (x, weight, bias))
    mean, rstd = torch.empty((2, n), dtype=torch.float32, device=ctx.device).unbind(0)
    check(lib.srx_layer_norm(ctx.handle, x.data_ptr(), ld, code, n, d, _address(weight), _address(bias), float(eps),
                             y.data_ptr(), ld_y, mean.data_ptr(), rstd.data_ptr(), ctx.stream_ptr()),
          "srx_layer_norm")
    return y, mean, rstd


def layer_norm_backward(ctx, dy, x, mean, rstd, weight=None):
    """(dx, dweight, dbias) of ``layer_norm`` for the gradient dy of its y; dx in x's type, the others float32."""
    if not isinstance(x, torch.Tensor) or x.dim() != 2:
        raise ValueError("x must be a 2-D (n_rows, n_features) tensor")
    n, d = rows = tuple(x.shape)
    code, ld = _code(x, "x"), _rows(ctx, x, "x", rows, x.dtype, d)
    ld_dy = _rows(ctx, dy, "dy", rows, x.dtype, d)
    for t, name in ((mean, "mean"), (rstd, "rstd")):
        if t is None:
            raise ValueError(f"{name} must be what layer_norm returned")
    mean, rstd = _parameter(ctx, mean, "mean", (n,)), _parameter(ctx, rstd, "rstd", (n,))
    weight = _parameter(ctx, weight, "weight", (d,))
    dx = _like(x)
    dweight = torch.empty((d,), dtype=torch.float32, device=ctx.device)
    dbias = torch.empty((d,), dtype=torch.float32, device=ctx.device)
    ws = _workspace(ctx, lib.srx_layer_norm_backward_workspace(ctx.handle, n, d))
    check(lib.srx_layer_norm_backward(ctx.handle, dy.data_ptr(), ld_dy, x.data_ptr(), ld, code, n, d,
                                      mean.data_ptr(), rstd.data_ptr(), _address(weight), dx.data_ptr(), d,
                                      dweight.data_ptr(), dbias.data_ptr(), ws.data_ptr(), ws.numel(),
                                      ctx.stream_ptr()), "srx_layer_norm_backward")
    return dx, dweight, dbias


# ---- gradient clipping ----------------------------------------------------------------------------

def _dense(t):
    """Whether a tensor's values fill their memory without gaps, in whatever order."""
    if t.layout != torch.strided:
        return False
    want = 1
    for stride, size in sorted((st, sz) for sz, st in zip(t.shape, t.stride()) if sz > 1):
        if stride != want:
            return False
        want *= size
    return True


def _array(kind, code, values):
    values = array.array(code, values)
    return (kind * len(values)).from_buffer(values)


def _codes(tensors, name):
    try:
        return [_CODES[t.dtype] for t in tensors]
    except KeyError:
        return [_code(t, f"{name}[{i}]") for i, t in enumerate(tensors)]


def clip_gradients(ctx, grads, max_norm, out=None):
    """Scales all gradients by min(1, max_norm / (norm + 1e-6)), norm the root of the sum of squares over all their
    values, and returns norm (float64, on the device; nothing waits for it).  grads: device tensors, float32,
    bfloat16 or float16 in any mixture, without gaps in memory; none may share memory with another.  They
    are scaled in place, or written to ``out`` -- tensors of the same shapes and order, each in its
    gradient's type or float32, such as views of an optimiser's flat buffer.  A norm that is not finite
    leaves the values as they are; the caller sees it in what is returned."""
    grads = list(grads)
    outs = None if out is None else list(out)
    if outs is not None and len(outs) != len(grads):
        raise ValueError(f"{len(grads)} gradients but {len(outs)} outputs")
    n = len(grads)
    # (in order: passed by one look at each property of all; else the first that is not is found)
    even = True                                          # every tensor contiguous
    for name, tensors in (("grads", grads), ("out", outs or ())):
        if not (set(map(type, tensors)) <= _TENSORS and set(map(torch.Tensor.get_device, tensors)) <= {_index(ctx)}
                and not any([t.requires_grad for t in tensors])):
            for i, t in enumerate(tensors):
                _on_device(ctx, t, f"{name}[{i}]")
        if not all(map(torch.Tensor.is_contiguous, tensors)):
            even = False
            for i, t in enumerate(tensors):
                if not t.is_contiguous() and not _dense(t):
                    raise ValueError(f"{name}[{i}] must fill its memory without gaps")
    counts = _array(C.c_int64, "q", map(torch.Tensor.numel, grads))
    tensors = _array(C.c_void_p, "Q", map(torch.Tensor.data_ptr, grads))
    dtypes = _array(C.c_int32, "i", _codes(grads, "grads"))
    to = to_types = None
    if outs is not None:
        if not (even and all(map(torch.Tensor.is_same_size, grads, outs))):
            for i, (t, o) in enumerate(zip(grads, outs)):
                if o.shape != t.shape or not (o.is_contiguous() and t.is_contiguous() or o.stride() == t.stride()):
                    raise ValueError(f"out[{i}] must have its gradient's shape and order")
        to = _array(C.c_void_p, "Q", map(torch.Tensor.data_ptr, outs))
        to_types = _array(C.c_int32, "i", _codes(outs, "out"))
    norm = torch.empty((), dtype=torch.float64, device=ctx.device)
    ws = _workspace(ctx, lib.srx_clip_gradients_workspace(ctx.handle, n, counts))
    check(lib.srx_clip_gradients(ctx.handle, n, tensors, counts, dtypes, to, to_types, float(max_norm),
                                 norm.data_ptr(), ws.data_ptr(), ws.numel(), ctx.stream_ptr()),
          "srx_clip_gradients")
    return norm


_ref = C.byref
