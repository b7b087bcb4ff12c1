"""What a sequence model does with packed feature rows: short causal convolution, selective state space
scan, and the norms around a block -- with their gradients, and single-token forms for serving.

They take the ``(total_frames, channels)`` device rows of a ragged batch and its ``frame_offsets``, as
``mfcc_batch(..., return_tensor=True)``, ``MfccPlan.execute`` and :func:`delta_batch` do: sequence ``s``
is rows ``frame_offsets[s] .. frame_offsets[s + 1]``.  (An extension: the reference's own model,
/root/reference/src/transformer.py, is plain PyTorch.)

Common to all of them:

* rows are float32, bfloat16 or float16 with unit stride along the channels (a column range of a wider
  matrix is fine); learned tables and their gradients are float32; arithmetic is float32, rounded once;
* ``frame_offsets`` is ``None`` (one sequence), a host array (checked, uploaded), or an int64 device tensor
  (taken as it is, without a synchronisation: what a captured graph is replayed with).  Rows in no sequence
  -- the end of a padded batch -- are zero in a new output, left as they are in ``out``, and have zero
  gradients; what they hold is not looked at;
* calls run on the current stream of the tensors' device; the same call gives the same bits;
* arguments that do not fit raise :class:`ParameterError`;
* what a call writes into the caller's tensors (``out``, the states of single-token calls) counts as an in-place
  operation of torch: their version counters go up, and tensors that require a gradient are not written;
* with gradients enabled and a differentiable input, the result has a ``grad_fn``.  Such a call cannot be
  made while a graph is captured (autograd may tie the capture to another stream): capture the plain call
  and the ``*_backward`` function under ``torch.no_grad()`` instead;
* ``*_backward`` and single-token calls have no gradient: with gradients enabled they take no tensor that requires
  one.  There are no derivatives in forward mode, and ``torch.jit.trace`` is refused.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional

import numpy as np
import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from .config import ParameterError

_DTYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}     # MFCC_F32, MFCC_BF16, MFCC_F16
_NORM = {"rms": 0, "layer": 1}
_ACTIVATION = {None: 0, "silu": 1}


class ConvGradients(NamedTuple):
    x: torch.Tensor
    weight: torch.Tensor
    bias: Optional[torch.Tensor]
    initial_state: Optional[torch.Tensor]


class ScanGradients(NamedTuple):
    u: torch.Tensor
    delta: torch.Tensor
    A: torch.Tensor
    B: torch.Tensor
    C: torch.Tensor
    D: Optional[torch.Tensor]
    delta_bias: Optional[torch.Tensor]
    initial_state: Optional[torch.Tensor]


class AddNormGradients(NamedTuple):
    x: torch.Tensor
    residual: torch.Tensor
    weight: Optional[torch.Tensor]
    bias: Optional[torch.Tensor]
    scale: Optional[torch.Tensor]


class GateNormGradients(NamedTuple):
    x: torch.Tensor
    z: torch.Tensor
    weight: Optional[torch.Tensor]
    bias: Optional[torch.Tensor]


# ---- arguments ---------------------------------------------------------------------------------------
def _check(rc: int) -> None:
    if rc == _lib.MFCC_E_INVALID:
        raise ParameterError(_lib.last_error())
    _lib.check(rc)


def _rows(t, name, like=None, dtype=None):
    """Rows of an operator: (rows, channels) on a GPU, unit stride along the channels."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ParameterError(f"{name} must be a device tensor: there is no CPU fallback")
    shape = t.shape
    if len(shape) != 2 or shape[1] == 0 or (t.stride(1) != 1 and shape[1] > 1):
        raise ParameterError(f"{name} must be (rows, channels) with unit stride along the channels, "
                             f"got shape {tuple(shape)}, strides {t.stride()}")
    if like is None:
        if t.dtype not in _DTYPE:
            raise ParameterError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    else:
        if shape != like.shape or t.get_device() != like.get_device():
            raise ParameterError(f"{name} must be {tuple(like.shape)} on {like.device}, got {tuple(shape)} on {t.device}")
        if t.dtype is not (dtype or like.dtype):
            raise ParameterError(f"{name} must be {dtype or like.dtype}, got {t.dtype}")
    return t


def _described(t):
    return f"{tuple(t.shape)} {t.dtype} on {t.device}" if isinstance(t, torch.Tensor) else type(t).__name__


def _table(t, name, shape, x, optional=True):
    """A learned table: float32 of the given shape on the rows' device (laid out contiguously if it is not)."""
    if t is None:
        if optional:
            return None
        raise ParameterError(f"{name} is missing")
    if not isinstance(t, torch.Tensor) or t.dtype is not torch.float32 or t.shape != shape or t.get_device() != x.get_device():
        raise ParameterError(f"{name} must be a float32 tensor of shape {shape} on {x.device}, got {_described(t)}")
    return t if t.is_contiguous() else t.contiguous()


def _state(t, name, shape, dtype, x, writable=False):
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.shape != shape or t.get_device() != x.get_device():
        raise ParameterError(f"{name} must be a {dtype} tensor of shape {shape} on {x.device}, got {_described(t)}")
    if t.is_contiguous():
        return t
    if writable:
        raise ParameterError(f"{name} must be contiguous")
    return t.contiguous()


def _span(t):
    """Bytes [first, last) that the rows occupy."""
    e = t.element_size()
    return t.data_ptr(), t.data_ptr() + ((t.shape[0] - 1) * t.stride(0) + t.shape[1]) * e


def _overlap(a, b) -> bool:
    if a is None or b is None or a.numel() == 0 or b.numel() == 0:
        return False
    a0, a1 = _span(a)
    b0, b1 = _span(b)
    if a1 <= b0 or b1 <= a0:
        return False
    step = a.stride(0) * a.element_size()
    if step > 0 and (step == b.stride(0) * b.element_size() or b.shape[0] == 1):         # column ranges of one matrix
        off = (b0 - a0) % step
        return not (off >= a.shape[1] * a.element_size() and off + b.shape[1] * b.element_size() <= step)
    return True


def _flat(t):
    """A contiguous state, table or list as rows, for the overlap check."""
    return None if t is None else t.reshape(1, -1)


def _out(out, x, inputs, dtype=None):
    """The output rows: new ones, or the caller's after a check."""
    if out is None:
        return _like(x, dtype)
    _rows(out, "out", x, dtype)
    if out.requires_grad and torch.is_grad_enabled():
        raise ParameterError("out requires a gradient: the call would overwrite it unseen")
    if out.shape[0] > 1 and out.stride(0) < out.shape[1]:
        raise ParameterError("the rows of out overlap")
    if any(_overlap(out, t) for t in inputs):
        raise ParameterError("out overlaps an input")
    return out


def _wrote(*tensors):
    """Raises the version counters of the caller's tensors that a call wrote through their pointers (None: no tensor), so
    that a backward pass that needs what they held says so, as after torch's own in-place operations."""
    for t in tensors:
        if t is not None:
            torch.autograd.graph.increment_version(t)


def _device_offsets(frame_offsets, x):
    """The frame offsets as a device tensor, or None: host arrays are checked and uploaded."""
    if frame_offsets is None:
        return None
    if isinstance(frame_offsets, torch.Tensor) and frame_offsets.is_cuda:
        t = frame_offsets
        if t.dtype != torch.int64 or t.ndim != 1 or not t.is_contiguous() or t.numel() < 1 or t.device != x.device:
            raise ParameterError(f"frame_offsets on a device must be a contiguous int64 vector on {x.device}")
        return t
    fo = np.ascontiguousarray(frame_offsets, dtype=np.int64)
    if fo.ndim != 1 or len(fo) < 1 or fo[0] < 0 or fo[-1] > x.shape[0] or (np.diff(fo) < 0).any():
        raise ParameterError(f"frame_offsets must ascend from >= 0 to <= {x.shape[0]} rows")
    if torch.cuda.is_current_stream_capturing():
        raise ParameterError("host frame_offsets cannot be uploaded while a graph is captured: pass a device tensor")
    return torch.from_numpy(fo).to(x.device)


def _offsets(frame_offsets, x):
    """(device pointer, sequences, tensor to keep alive) of the frame offsets."""
    t = _device_offsets(frame_offsets, x)
    return (None, 1, None) if t is None else (t.data_ptr(), t.numel() - 1, t)


def _ptr(t):
    return None if t is None else t.data_ptr()


# the handle of a device's current stream, without the Stream object torch.cuda.current_stream makes (3 us)
_stream_of = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _run(x, fn, *args):
    """fn(*args, current stream) on the device of the rows x."""
    index = x.get_device()
    if torch.cuda.current_device() == index:
        _check(fn(*args, _stream_of(index)))
    else:
        with torch.cuda.device(index):
            _check(fn(*args, _stream_of(index)))


def _workspace(size, x):
    return x.new_empty(size, dtype=torch.uint8) if size else None


def _like(t, dtype=None):
    """An uninitialised contiguous tensor of t's shape (1.2 us; new_empty 1.9 us)."""
    return torch.empty_like(t, dtype=dtype, memory_format=torch.contiguous_format)


def _new(x, shape, dtype=None):
    """An uninitialised contiguous tensor beside x, in the current stream's memory."""
    return x.new_empty(shape, dtype=dtype or x.dtype)


def _unseen(tensors):
    """Refuses calls whose derivative or whose very work would be lost: tangents of forward mode, and a trace, which
    records torch's own operations only."""
    if getattr(forward_ad, "_current_level", 0) >= 0 and any(
            isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise ParameterError("there are no derivatives in forward mode: take them in reverse mode")
    if torch.jit.is_tracing():
        raise ParameterError("a call cannot be traced by torch.jit")


def _differentiable(out, *tensors) -> bool:
    _unseen(tensors)
    if not torch.is_grad_enabled() or not any(isinstance(t, torch.Tensor) and t.requires_grad for t in tensors):
        return False
    if torch.cuda.is_current_stream_capturing():
        raise ParameterError("a differentiable call cannot be captured into a graph: capture the plain call and its "
                             "*_backward function under torch.no_grad()")
    if out is not None:
        raise ParameterError("out cannot be given to a differentiable call")
    return True


def _incoming(d, like):
    """A gradient from autograd as rows (an expanded one has no unit stride)."""
    if torch.cuda.is_current_stream_capturing():
        raise ParameterError("a differentiable call's backward pass cannot be captured into a graph: capture the "
                             "*_backward function under torch.no_grad()")
    if d is None:
        return torch.zeros(like.shape, dtype=like.dtype, device=like.device)
    return d if d.stride(1) == 1 or d.shape[1] == 1 else d.contiguous()


# ---- causal convolution --------------------------------------------------------------------------------
def _conv_args(x, weight, bias, frame_offsets, activation, initial_state):
    x = _rows(x, "x")
    rows, channels = x.shape
    if not isinstance(weight, torch.Tensor) or weight.ndim != 2:
        raise ParameterError("weight must be (channels, width)")
    width = weight.shape[1]
    if not 1 <= width <= 8:
        raise ParameterError(f"the width must lie between 1 and 8, got {width}")
    weight = _table(weight, "weight", (channels, width), x, optional=False)
    bias = _table(bias, "bias", (channels,), x)
    if activation not in _ACTIVATION:
        raise ParameterError(f"activation must be None or 'silu', got {activation!r}")
    off, n_seqs, keep = _offsets(frame_offsets, x)
    initial_state = _state(initial_state, "initial_state", (n_seqs, width - 1, channels), x.dtype, x)
    a = _lib.ConvArgsC(C.sizeof(_lib.ConvArgsC), _DTYPE[x.dtype], channels, width, _ACTIVATION[activation], n_seqs, 0, rows,
                       off, x.data_ptr(), x.stride(0), weight.data_ptr(), _ptr(bias), _ptr(initial_state))
    return a, x, (weight, bias, initial_state, keep), n_seqs, width


def _conv_forward(x, weight, bias, frame_offsets, activation, initial_state, return_state, out):
    a, x, keep, n_seqs, width = _conv_args(x, weight, bias, frame_offsets, activation, initial_state)
    y = _out(out, x, (x, *map(_flat, keep)) if out is not None else ())
    a.d_y, a.y_stride, a.zero_rest = y.data_ptr(), y.stride(0), out is None
    state = None
    if return_state:
        state = _new(x, (n_seqs, width - 1, x.shape[1]))
        a.d_state = state.data_ptr()
    _run(x, _lib.lib().mfcc_causal_conv, a)
    if out is not None:
        _wrote(out)
    return y, state


class _Conv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, initial_state, frame_offsets, activation, return_state):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, weight, bias, initial_state, frame_offsets)
        ctx.activation = activation
        y, state = _conv_forward(x, weight, bias, frame_offsets, activation, initial_state, return_state, None)
        return (y, state) if return_state else y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dstate=None):
        x, weight, bias, initial_state, frame_offsets = ctx.saved_tensors
        g = causal_conv_backward(_incoming(dy, x), x, weight, bias, frame_offsets, activation=ctx.activation,
                                 initial_state=initial_state, dstate=dstate)
        return g.x, g.weight, g.bias, g.initial_state, None, None, None


def causal_conv(x, weight, bias=None, frame_offsets=None, *, activation=None, initial_state=None, return_state=False, out=None):
    """Causal convolution along each sequence, channel by channel, of width 1 to 8:
    ``y[t] = act(bias + sum_j weight[:, j] * x[t - (width - 1) + j])`` with ``activation`` None or ``'silu'``.

    ``x`` is (rows, channels), ``weight`` (channels, width) and ``bias`` (channels) float32.  The rows before
    a sequence are zero, or ``initial_state`` (sequences, width - 1, channels) of x's type.  With
    ``return_state`` the result is ``(y, state)``: the last ``width - 1`` rows of every sequence (the end of
    its initial state standing before a short one), to go on with in a later call or token by token."""
    if _differentiable(out, x, weight, bias, initial_state):
        frame_offsets = _device_offsets(frame_offsets, _rows(x, "x"))
        return _Conv.apply(x, weight, bias, initial_state, frame_offsets, activation, return_state)
    y, state = _conv_forward(x, weight, bias, frame_offsets, activation, initial_state, return_state, out)
    return (y, state) if return_state else y


def causal_conv_backward(dy, x, weight, bias=None, frame_offsets=None, *, activation=None, initial_state=None, dstate=None):
    """Gradients of :func:`causal_conv` for the gradient ``dy`` of its rows and, or None, ``dstate`` of the
    state it returned.  ``bias`` and ``initial_state`` have gradients where they are given."""
    _no_second_derivative(dy, x, weight, bias, initial_state, dstate)
    a, x, keep, n_seqs, width = _conv_args(x, weight, bias, frame_offsets, activation, initial_state)
    dy = _rows(dy, "dy", x)
    channels = x.shape[1]
    dstate = _state(dstate, "dstate", (n_seqs, width - 1, channels), x.dtype, x)
    dx = _like(x)
    dweight = _new(x, (channels, width), torch.float32)
    dbias = None if bias is None else _new(x, (channels,), torch.float32)
    dinitial = None if initial_state is None else _new(x, (n_seqs, width - 1, channels))
    a.d_dy, a.dy_stride, a.d_dstate = dy.data_ptr(), dy.stride(0), _ptr(dstate)
    a.d_dx, a.dx_stride, a.d_dweight, a.d_dbias, a.d_dinitial = dx.data_ptr(), channels, dweight.data_ptr(), _ptr(dbias), _ptr(dinitial)
    ws = _workspace(_lib.lib().mfcc_causal_conv_backward_workspace(a), x)
    a.d_workspace, a.workspace_bytes = _ptr(ws), 0 if ws is None else ws.numel()
    _run(x, _lib.lib().mfcc_causal_conv_backward, a)
    return ConvGradients(dx, dweight, dbias, dinitial)


def _slots(slots, batch, x):
    if slots is None:
        return None
    if (not isinstance(slots, torch.Tensor) or slots.dtype != torch.int32 or tuple(slots.shape) != (batch,)
            or slots.device != x.device or not slots.is_contiguous()):
        raise ParameterError(f"slots must be a contiguous int32 tensor of shape ({batch},) on {x.device}")
    return slots


def _no_grad_step(*tensors):
    _unseen(tensors)
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in tensors):
        raise ParameterError("single-token calls have no gradient: call them under torch.no_grad()")


def _no_second_derivative(*tensors):
    _unseen(tensors)
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in tensors):
        raise ParameterError("explicit gradients have no gradient of their own: call them under torch.no_grad()")


def _next_state(state, new_state):
    if new_state is None or new_state.data_ptr() == state.data_ptr():
        return state
    a, b = state.data_ptr(), new_state.data_ptr()
    if a < b + new_state.numel() * new_state.element_size() and b < a + state.numel() * state.element_size():
        raise ParameterError("new_state overlaps state")
    return new_state


def causal_conv_step(x, state, weight, bias=None, *, activation=None, slots=None, new_state=None, out=None):
    """One token of :func:`causal_conv` for each row of ``x`` (batch, channels).  ``state`` (slots, width - 1,
    channels) holds the sequences' last rows; row e continues the sequence in slot ``slots[e]`` (int32 device
    tensor; slot e without it), whose state after the token replaces it -- or is written to the same slot of
    ``new_state``, the others being left alone; neither pool overlaps another argument.  Rows that name one
    slot are successive tokens of it, in their order; a slot outside the pool (a padded row) gives a zero
    row.  Returns y."""
    _no_grad_step(x, state, weight, bias, new_state)
    x = _rows(x, "x")
    batch, channels = x.shape
    if not isinstance(weight, torch.Tensor) or weight.ndim != 2 or not 1 <= weight.shape[1] <= 8:
        raise ParameterError("weight must be (channels, width) with a width between 1 and 8")
    width = weight.shape[1]
    weight = _table(weight, "weight", (channels, width), x, optional=False)
    bias = _table(bias, "bias", (channels,), x)
    if activation not in _ACTIVATION:
        raise ParameterError(f"activation must be None or 'silu', got {activation!r}")
    n_slots = state.shape[0] if isinstance(state, torch.Tensor) and state.ndim == 3 else -1
    if state is None:
        raise ParameterError("state is missing")
    state = _state(state, "state", (n_slots, width - 1, channels), x.dtype, x, writable=True)
    into = _next_state(state, _state(new_state, "new_state", (n_slots, width - 1, channels), x.dtype, x, writable=True))
    slots = _slots(slots, batch, x)
    y = _out(out, x, (x, *map(_flat, (state, into, weight, bias, slots))) if out is not None else ())
    _run(x, _lib.lib().mfcc_causal_conv_step, _DTYPE[x.dtype], batch, n_slots, channels, width, _ACTIVATION[activation],
         x.data_ptr(), x.stride(0), state.data_ptr(), into.data_ptr(), weight.data_ptr(), _ptr(bias), _ptr(slots),
         y.data_ptr(), y.stride(0))
    _wrote(into, None if new_state is into else new_state, out)
    return y


# ---- selective scan -------------------------------------------------------------------------------------
def _groups(B, name, u, state):
    """(rows, N) or (rows, G, N) with contiguous groups and states: (row stride, G)."""
    if not isinstance(B, torch.Tensor) or B.dtype != u.dtype or B.device != u.device:
        raise ParameterError(f"{name} must be a {u.dtype} tensor on {u.device}")
    groups = 1 if B.ndim == 2 else B.shape[1] if B.ndim == 3 else 0
    if groups < 1 or B.shape[0] != u.shape[0] or B.shape[-1] != state:
        raise ParameterError(f"{name} must be ({u.shape[0]}, {state}) or ({u.shape[0]}, groups, {state}), got {tuple(B.shape)}")
    if (B.stride(-1) != 1 and state > 1) or (B.ndim == 3 and groups > 1 and B.stride(1) != state):
        raise ParameterError(f"{name} must be contiguous within a row, got strides {B.stride()}")
    return B.stride(0), groups


def _scan_args(u, delta, A, B, Cm, D, delta_bias, softplus, n_seqs, off):
    u = _rows(u, "u")
    rows, channels = u.shape
    delta = _rows(delta, "delta", u)
    if not isinstance(A, torch.Tensor) or A.ndim != 2:
        raise ParameterError("A must be (channels, state)")
    state = A.shape[1]
    if not 1 <= state <= 64:
        raise ParameterError(f"a channel has 1 to 64 states, got {state}")
    A = _table(A, "A", (channels, state), u, optional=False)
    D = _table(D, "D", (channels,), u)
    delta_bias = _table(delta_bias, "delta_bias", (channels,), u)
    b_stride, groups = _groups(B, "B", u, state)
    c_stride, c_groups = _groups(Cm, "C", u, state)
    if groups != c_groups or channels % groups:
        raise ParameterError(f"B and C need the same number of groups, a divisor of {channels} channels; got {groups} and {c_groups}")
    a = _lib.ScanArgsC(C.sizeof(_lib.ScanArgsC), _DTYPE[u.dtype], channels, state, groups, bool(softplus), n_seqs, 0, rows,
                       off, u.data_ptr(), u.stride(0), delta.data_ptr(), delta.stride(0), A.data_ptr(),
                       B.data_ptr(), b_stride, Cm.data_ptr(), c_stride, _ptr(D), _ptr(delta_bias))
    return a, (A, D, delta_bias), state


def _scan_forward(u, delta, A, B, Cm, D, delta_bias, frame_offsets, softplus, initial_state, return_state, out):
    u = _rows(u, "u")
    off, n_seqs, keep_off = _offsets(frame_offsets, u)
    a, keep, state = _scan_args(u, delta, A, B, Cm, D, delta_bias, softplus, n_seqs, off)
    shape = (n_seqs, u.shape[1], state)
    initial_state = _state(initial_state, "initial_state", shape, torch.float32, u)
    a.d_initial = _ptr(initial_state)
    y = _out(out, u, (u, delta, B.flatten(1), Cm.flatten(1), *map(_flat, (initial_state, keep_off, *keep))) if out is not None else ())
    a.d_y, a.y_stride, a.zero_rest = y.data_ptr(), y.stride(0), out is None
    final = None
    if return_state:
        final = _new(u, shape, torch.float32)
        a.d_final = final.data_ptr()
    ws = _workspace(_lib.lib().mfcc_selective_scan_workspace(a), u)
    a.d_workspace, a.workspace_bytes = _ptr(ws), 0 if ws is None else ws.numel()
    _run(u, _lib.lib().mfcc_selective_scan, a)
    if out is not None:
        _wrote(out)
    return y, final


class _Scan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, u, delta, A, B, Cm, D, delta_bias, initial_state, frame_offsets, softplus, return_state):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(u, delta, A, B, Cm, D, delta_bias, initial_state, frame_offsets)
        ctx.softplus = softplus
        y, final = _scan_forward(u, delta, A, B, Cm, D, delta_bias, frame_offsets, softplus, initial_state, return_state, None)
        return (y, final) if return_state else y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dstate=None):
        u, delta, A, B, Cm, D, delta_bias, initial_state, frame_offsets = ctx.saved_tensors
        g = selective_scan_backward(_incoming(dy, u), u, delta, A, B, Cm, D, delta_bias, frame_offsets,
                                    softplus=ctx.softplus, initial_state=initial_state, dstate=dstate)
        return (*g, None, None, None)


def selective_scan(u, delta, A, B, C, D=None, delta_bias=None, frame_offsets=None, *, softplus=False, initial_state=None,
                   return_state=False, out=None):
    """Selective state space scan along each sequence: with ``d = softplus(delta + delta_bias)`` (or the plain
    sum), ``h[c, n] = exp(d A[c, n]) h[c, n] + d u[c] B[n]`` and ``y[c] = sum_n C[n] h[c, n] + D[c] u[c]``.

    ``u`` and ``delta`` are (rows, channels); ``A`` (channels, state), ``D`` and ``delta_bias`` (channels)
    float32; ``B`` and ``C`` (rows, state) or (rows, groups, state), of u's type, each group serving
    channels / groups neighbouring channels.  1 to 64 states.  ``initial_state`` and, with
    ``return_state``, the second result are (sequences, channels, state) float32."""
    if _differentiable(out, u, delta, A, B, C, D, delta_bias, initial_state):
        frame_offsets = _device_offsets(frame_offsets, _rows(u, "u"))
        return _Scan.apply(u, delta, A, B, C, D, delta_bias, initial_state, frame_offsets, softplus, return_state)
    y, final = _scan_forward(u, delta, A, B, C, D, delta_bias, frame_offsets, softplus, initial_state, return_state, out)
    return (y, final) if return_state else y


def selective_scan_backward(dy, u, delta, A, B, C, D=None, delta_bias=None, frame_offsets=None, *, softplus=False,
                            initial_state=None, dstate=None):
    """Gradients of :func:`selective_scan` for the gradient ``dy`` of its rows and, or None, ``dstate`` of the
    state it returned.  The states are recomputed; optional inputs have gradients where they are given."""
    _no_second_derivative(dy, u, delta, A, B, C, D, delta_bias, initial_state, dstate)
    u = _rows(u, "u")
    off, n_seqs, keep_off = _offsets(frame_offsets, u)
    a, keep, state = _scan_args(u, delta, A, B, C, D, delta_bias, softplus, n_seqs, off)
    dy = _rows(dy, "dy", u)
    shape = (n_seqs, u.shape[1], state)
    initial_state = _state(initial_state, "initial_state", shape, torch.float32, u)
    dstate = _state(dstate, "dstate", shape, torch.float32, u)

    def new(like, dtype):
        return None if like is None else _like(like, dtype)

    f32 = torch.float32
    g = ScanGradients(new(u, u.dtype), new(u, u.dtype), new(A, f32), new(B, u.dtype), new(C, u.dtype), new(D, f32),
                      new(delta_bias, f32), new(initial_state, f32))
    a.d_initial, a.d_dy, a.dy_stride, a.d_dfinal = _ptr(initial_state), dy.data_ptr(), dy.stride(0), _ptr(dstate)
    (a.d_du, a.d_ddelta, a.d_dA, a.d_dB, a.d_dC, a.d_dD, a.d_ddelta_bias, a.d_dinitial) = map(_ptr, g)
    ws = _workspace(_lib.lib().mfcc_selective_scan_backward_workspace(a), u)
    a.d_workspace, a.workspace_bytes = _ptr(ws), 0 if ws is None else ws.numel()
    _run(u, _lib.lib().mfcc_selective_scan_backward, a)
    return g


def selective_scan_step(u, delta, A, B, C, state, D=None, delta_bias=None, *, softplus=False, slots=None, new_state=None,
                        out=None):
    """One token of :func:`selective_scan` for each row of ``u`` (batch, channels).  ``state`` (slots, channels,
    state) float32 holds the sequences' states; ``slots``, ``new_state`` and padded rows are as in
    :func:`causal_conv_step`.  Returns y."""
    _no_grad_step(u, delta, A, B, C, state, D, delta_bias, new_state)
    u = _rows(u, "u")
    a, keep, n_state = _scan_args(u, delta, A, B, C, D, delta_bias, softplus, 0, None)
    if state is None:
        raise ParameterError("state is missing")
    n_slots = state.shape[0] if isinstance(state, torch.Tensor) and state.ndim == 3 else -1
    shape = (n_slots, u.shape[1], n_state)
    state = _state(state, "state", shape, torch.float32, u, writable=True)
    into = _next_state(state, _state(new_state, "new_state", shape, torch.float32, u, writable=True))
    slots = _slots(slots, u.shape[0], u)
    y = _out(out, u, (u, delta, B.flatten(1), C.flatten(1), *map(_flat, (state, into, slots, *keep))) if out is not None else ())
    a.d_initial, a.d_final = state.data_ptr(), into.data_ptr()
    a.d_y, a.y_stride = y.data_ptr(), y.stride(0)
    _run(u, _lib.lib().mfcc_selective_scan_step, a, n_slots, _ptr(slots))
    _wrote(into, None if new_state is into else new_state, out)
    return y


# ---- norms ------------------------------------------------------------------------------------------------
def _norm_args(x, weight, bias, scale, norm, eps, groups, gate_first, res_dtype):
    rows, channels = x.shape
    if norm not in _NORM:
        raise ParameterError(f"norm must be 'rms' or 'layer', got {norm!r}")
    if not eps > 0:
        raise ParameterError(f"eps must be positive, got {eps}")
    if groups < 1 or channels % groups:
        raise ParameterError(f"groups must divide the {channels} channels, got {groups}")
    if channels // groups > 32768:
        raise ParameterError(f"a norm runs over at most 32768 channels, got {channels // groups}")
    weight = _table(weight, "weight", (channels,), x)
    bias = _table(bias, "bias", (channels,), x)
    value = 1.0
    if isinstance(scale, torch.Tensor):
        scale = _table(scale, "scale", (channels,), x)
    elif scale is not None:
        value, scale = float(scale), None
    a = _lib.NormArgsC(C.sizeof(_lib.NormArgsC), _DTYPE[x.dtype], _DTYPE[res_dtype], channels, groups, _NORM[norm],
                       bool(gate_first), eps, value, rows, _ptr(weight), _ptr(bias), _ptr(scale))
    return a, (weight, bias, scale)


def _residual_dtype(x, residual, residual_dtype):
    dtype = residual_dtype or (x.dtype if residual is None else residual.dtype)
    if dtype not in (x.dtype, torch.float32):
        raise ParameterError(f"the residual must be {x.dtype} or float32, got {dtype}")
    return dtype


def _add_norm_forward(x, residual, weight, bias, scale, norm, eps, residual_dtype):
    x = _rows(x, "x")
    if residual is not None and not isinstance(residual, torch.Tensor):
        raise ParameterError("residual must be a device tensor")
    rt = _residual_dtype(x, residual, residual_dtype)
    if residual is not None:
        residual = _rows(residual, "residual", x, rt)
    a, keep = _norm_args(x, weight, bias, scale, norm, eps, 1, False, rt)
    y, r = _like(x), _like(x, rt)
    a.d_x, a.x_stride = x.data_ptr(), x.stride(0)
    if residual is not None:
        a.d_residual, a.residual_stride = residual.data_ptr(), residual.stride(0)
    a.d_y, a.y_stride, a.d_r, a.r_stride = y.data_ptr(), x.shape[1], r.data_ptr(), x.shape[1]
    _run(x, _lib.lib().mfcc_add_norm, a)
    return y, r


class _AddNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, bias, scale, norm, eps, residual_dtype):
        ctx.set_materialize_grads(False)
        y, r = _add_norm_forward(x, residual, weight, bias, scale, norm, eps, residual_dtype)
        learned = isinstance(scale, torch.Tensor)
        ctx.save_for_backward(r, weight, bias, x if learned else None, scale if learned else None)
        ctx.number, ctx.norm, ctx.eps, ctx.dtype, ctx.residual = None if learned else scale, norm, eps, x.dtype, residual is not None
        return y, r

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dr):
        r, weight, bias, x, scale = ctx.saved_tensors
        if dy is None and dr is None:
            return (None,) * 8
        dy, dr = (None if d is None else _incoming(d, r) for d in (dy, dr))
        g = add_norm_backward(dy, dr, r, weight, bias, x=x, scale=ctx.number if scale is None else scale, norm=ctx.norm,
                              eps=ctx.eps, dtype=ctx.dtype)
        return g.x, g.residual if ctx.residual else None, g.weight, g.bias, g.scale, None, None, None


def add_norm(x, residual=None, weight=None, bias=None, *, scale=None, norm="rms", eps=1e-5, residual_dtype=None):
    """The norm before a block, with the sum that precedes it: ``r = residual + scale * x`` and
    ``y = norm(r) * weight + bias``; returns ``(y, r)``.

    ``x`` (rows, channels) is the last block's output, ``residual`` the stream it is added to (x's type or
    float32; None for the first block, whose ``r`` then has ``residual_dtype`` or x's type).  ``scale`` is a
    number or a learned (channels) tensor.  ``norm`` is ``'rms'`` or ``'layer'``; the norm is taken of the
    unrounded sum.  At most 32768 channels."""
    learned = scale if isinstance(scale, torch.Tensor) else None
    if _differentiable(None, x, residual, weight, bias, learned):
        return _AddNorm.apply(x, residual, weight, bias, scale, norm, eps, residual_dtype)
    return _add_norm_forward(x, residual, weight, bias, scale, norm, eps, residual_dtype)


def add_norm_backward(dy, dr, r, weight=None, bias=None, *, x=None, scale=None, norm="rms", eps=1e-5, dtype=None):
    """Gradients of :func:`add_norm` from the ``r`` it returned: ``dy`` and ``dr`` are the gradients of its two
    results (one of them may be None).  ``x`` is needed for the gradient of a learned ``scale`` only;
    ``dtype`` is x's type where ``dy`` does not tell it.  Without a scale and with one type the gradients of x
    and of the residual are the same numbers and are returned as one tensor."""
    _no_second_derivative(dy, dr, r, weight, bias, x, scale)
    r = _rows(r, "r")
    dtype = dy.dtype if dy is not None else dtype or (x.dtype if x is not None else r.dtype)
    if dtype not in _DTYPE or r.dtype not in (dtype, torch.float32):
        raise ParameterError(f"r must be {dtype} or float32, got {r.dtype}")
    if dy is not None:
        _rows(dy, "dy", r, dtype)
    if dr is not None:
        _rows(dr, "dr", r)
    learned = isinstance(scale, torch.Tensor)
    if learned:
        if x is None:
            raise ParameterError("the gradient of a learned scale needs x")
        _rows(x, "x", r, dtype)
    a, keep = _norm_args(r, weight, bias, scale, norm, eps, 1, False, r.dtype)
    a.dtype = _DTYPE[dtype]
    channels = r.shape[1]

    def vector(like):
        return None if like is None else _new(r, (channels,), torch.float32)

    dresidual = _like(r)
    one = r.dtype == dtype and not learned and a.scale_value == 1.0
    dx = dresidual if one else _like(r, dtype)
    g = AddNormGradients(dx, dresidual, vector(weight), vector(bias), vector(scale if learned else None))
    a.d_r, a.r_stride = r.data_ptr(), r.stride(0)
    if dy is not None:
        a.d_dy, a.dy_stride = dy.data_ptr(), dy.stride(0)
    if dr is not None:
        a.d_dr, a.dr_stride = dr.data_ptr(), dr.stride(0)
    if learned:
        a.d_x, a.x_stride = x.data_ptr(), x.stride(0)
    a.d_dresidual, a.d_dx = dresidual.data_ptr(), None if one else dx.data_ptr()
    a.d_dweight, a.d_dbias, a.d_dscale = _ptr(g.weight), _ptr(g.bias), _ptr(g.scale)
    ws = None
    if g.weight is not None or g.bias is not None or g.scale is not None:
        ws = _workspace(_lib.lib().mfcc_norm_backward_workspace(a), r)
    a.d_workspace, a.workspace_bytes = _ptr(ws), 0 if ws is None else ws.numel()
    _run(r, _lib.lib().mfcc_add_norm_backward, a)
    return g


class _GateNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, z, weight, bias, norm, groups, gate_first, eps):
        ctx.save_for_backward(x, z, weight, bias)
        ctx.kw = dict(norm=norm, groups=groups, gate_first=gate_first, eps=eps)
        return _gate_norm_forward(x, z, weight, bias, norm, groups, gate_first, eps, None)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, z, weight, bias = ctx.saved_tensors
        g = gate_norm_backward(_incoming(dy, x), x, z, weight, bias, **ctx.kw)
        return g.x, g.z, g.weight, g.bias, None, None, None, None


def _gate_norm_forward(x, z, weight, bias, norm, groups, gate_first, eps, out):
    x = _rows(x, "x")
    z = _rows(z, "z", x)
    a, keep = _norm_args(x, weight, bias, None, norm, eps, groups, gate_first, x.dtype)
    y = _out(out, x, (x, z, *map(_flat, keep)) if out is not None else ())
    a.d_x, a.x_stride, a.d_z, a.z_stride = x.data_ptr(), x.stride(0), z.data_ptr(), z.stride(0)
    a.d_y, a.y_stride = y.data_ptr(), y.stride(0)
    _run(x, _lib.lib().mfcc_gate_norm, a)
    if out is not None:
        _wrote(out)
    return y


def gate_norm(x, z, weight=None, bias=None, *, norm="rms", groups=1, gate_first=True, eps=1e-5, out=None):
    """The norm after a block, with its gate: ``norm(x * silu(z)) * weight + bias``, or, with
    ``gate_first=False``, ``(norm(x) * weight + bias) * silu(z)``.  ``x`` and ``z`` are (rows, channels); the
    norm (``'rms'`` or ``'layer'``) runs over each of ``groups`` equal slices of a row, at most 32768 wide."""
    if _differentiable(out, x, z, weight, bias):
        return _GateNorm.apply(x, z, weight, bias, norm, groups, gate_first, eps)
    return _gate_norm_forward(x, z, weight, bias, norm, groups, gate_first, eps, out)


def gate_norm_backward(dy, x, z, weight=None, bias=None, *, norm="rms", groups=1, gate_first=True, eps=1e-5):
    """Gradients of :func:`gate_norm` for the gradient ``dy`` of its result."""
    _no_second_derivative(dy, x, z, weight, bias)
    x = _rows(x, "x")
    z = _rows(z, "z", x)
    dy = _rows(dy, "dy", x)
    a, keep = _norm_args(x, weight, bias, None, norm, eps, groups, gate_first, x.dtype)
    channels = x.shape[1]

    def vector(like):
        return None if like is None else _new(x, (channels,), torch.float32)

    g = GateNormGradients(_like(x), _like(x), vector(weight), vector(bias))
    a.d_x, a.x_stride, a.d_z, a.z_stride = x.data_ptr(), x.stride(0), z.data_ptr(), z.stride(0)
    a.d_dy, a.dy_stride = dy.data_ptr(), dy.stride(0)
    a.d_dx, a.d_dz, a.d_dweight, a.d_dbias = g.x.data_ptr(), g.z.data_ptr(), _ptr(g.weight), _ptr(g.bias)
    ws = None
    if g.weight is not None or g.bias is not None:
        ws = _workspace(_lib.lib().mfcc_norm_backward_workspace(a), x)
    a.d_workspace, a.workspace_bytes = _ptr(ws), 0 if ws is None else ws.numel()
    _run(x, _lib.lib().mfcc_gate_norm_backward, a)
    return g
