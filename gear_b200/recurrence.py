"""Linear recurrences over sequences, with gradients: h_t = a_t * h_(t-1) + x_t.

The form behind discounted returns and advantage estimates (one channel, `reverse=True`) and behind
recurrent sequence layers (many channels), over the batches this framework samples:

    dense    x [batch, time, width]                 every batch entry is one sequence
    padded   x [batch, time, width], lengths        the first lengths[b] rows of entry b (tail padding, what
                                                    StorageHandler.gather leaves)
    packed   x [rows, width], offsets               rows [offsets[s], offsets[s+1]) are sequence s (what
                                                    StorageHandler.gather_packed leaves)

    returns, _ = linear_recurrence(rewards, gamma * (1 - done), offsets=offsets, reverse=True)
    h, state = linear_recurrence(x, log_decay, h0=state, gate_kind="log")     # one more chunk, or one token

The reference has no counterpart: its loader stops at the padded batch (gear/loader/offline_loader.py:178-203).
"""
from __future__ import annotations

import ctypes as C
import functools
from typing import NamedTuple, Optional

import torch
import torch.autograd.forward_ad as _forward_ad

from . import _native as N
from ._native import GearError, check, lib
from .core import _Scope, _stream

__all__ = ["linear_recurrence"]

_DTYPES = {torch.float32: N.DT_F32, torch.float16: N.DT_F16, torch.bfloat16: N.DT_BF16}
_PACK = N.RECURRENCE_ARGS.pack
_FORWARD, _BACKWARD = lib.gearb_recurrence_forward, lib.gearb_recurrence_backward


def _bad(msg: str):
    raise GearError(N.ERR_INVALID, "linear_recurrence: " + msg)


def _vector(t, what: str, dtype: torch.dtype, shape: tuple, device) -> None:
    if t.dtype is not dtype or tuple(t.shape) != shape:
        _bad(f"{what} must be {dtype} of shape {list(shape)}")
    if t.device != device:
        _bad(f"{what} is on {t.device}, x on {device}")


def _unit(t: torch.Tensor) -> torch.Tensor:
    """The tensor itself where its last dimension is consecutive (any other strides), else a copy."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _no_tangents(*tensors) -> None:
    if getattr(_forward_ad, "_current_level", 0) >= 0:     # inside a dual level
        for t in tensors:
            if t is not None and _forward_ad.unpack_dual(t).tangent is not None:
                _bad("forward-mode derivatives are not supported: the tangent would be dropped")


def _at(t) -> int:
    return 0 if t is None else t.data_ptr()


class _Sizes(NamedTuple):
    """What the entry points are told about a call besides its tensors."""
    x_dtype: int
    gate_dtype: int
    batch: int
    time: int
    width: int
    gates: int
    sequences: int
    packed: bool
    padded: bool
    reverse: int
    log: int


@functools.lru_cache(maxsize=1024)
def _buffers(s: _Sizes):
    """Bytes of (forward scratch, backward scratch, carry): they depend on the sizes alone."""
    a = N.RecurrenceArgs()
    a.x_dtype, a.gate_dtype, a.batch, a.time, a.width, a.gates = s[:6]
    a.sequences, a.offsets, a.lengths = s.sequences, int(s.packed) or None, int(s.padded) or None
    out = []
    for backward in (0, 1):
        scratch, carry = C.c_int64(0), C.c_int64(0)
        check(lib.gearb_recurrence_bytes(C.byref(a), backward, C.byref(scratch), C.byref(carry)))
        out.append(scratch.value)
    return out[0], out[1], carry.value


def _strides(t):
    s = t.stride()
    return (0, s[0]) if len(s) == 2 else (s[0], s[1])


def _forward(s, x, gate, h0, offsets, lengths, carry, return_state, out, state_out, status):
    dev = x.device
    state = state_out
    if state is None and return_state:
        state = torch.empty((s.sequences, s.width), dtype=torch.float32, device=dev)
    elif state is not None and h0 is not None and s.time != 1 and state.data_ptr() == h0.data_ptr():
        h0 = h0.clone()    # rows of one sequence are worked on in several places: one may be done before another reads h0
    h = torch.empty(x.shape, dtype=x.dtype, device=dev) if out is None else out
    nbytes = _buffers(s)[0]
    scratch = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    check(_FORWARD(_PACK(x.data_ptr(), gate.data_ptr(), s.x_dtype, s.gate_dtype, s.batch, s.time, s.width, s.gates,
                         *_strides(x), *_strides(gate), _at(offsets), _at(lengths), s.sequences, _at(h0),
                         s.reverse, s.log, int(out is None), h.data_ptr(), _at(state), _at(carry),
                         0, 0, 0, 0, 0, 0, 0, _at(scratch), nbytes, _at(status)), _stream()))
    return h, state


class _LinearRecurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, h0, offsets, lengths, s, return_state, status):
        carry = torch.empty(_buffers(s)[2] // 4, dtype=torch.float32, device=x.device)
        h, state = _forward(s, x, gate, h0, offsets, lengths, carry, return_state, None, None, status)
        ctx.save_for_backward(x, gate, h0, offsets, lengths, carry)
        ctx.s, ctx.status = s, status
        ctx.set_materialize_grads(False)
        return h, state

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh, dstate):
        x, gate, h0, offsets, lengths, carry = ctx.saved_tensors
        s = ctx.s
        _no_tangents(dh, dstate)
        with _Scope(x.device):
            dh = torch.zeros_like(x) if dh is None else _unit(dh)
            dstate = None if dstate is None else dstate.contiguous()
            dev = x.device
            dx = torch.empty(x.shape, dtype=x.dtype, device=dev)
            dgate = torch.empty(gate.shape, dtype=gate.dtype, device=dev)
            dh0 = None if h0 is None else torch.empty(h0.shape, dtype=torch.float32, device=dev)
            nbytes = _buffers(s)[1]
            scratch = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
            check(_BACKWARD(_PACK(x.data_ptr(), gate.data_ptr(), s.x_dtype, s.gate_dtype, s.batch, s.time, s.width,
                                  s.gates, *_strides(x), *_strides(gate), _at(offsets), _at(lengths), s.sequences,
                                  _at(h0), s.reverse, s.log, 1, 0, 0, carry.data_ptr(), dh.data_ptr(), *_strides(dh),
                                  _at(dstate), dx.data_ptr(), dgate.data_ptr(), _at(dh0), _at(scratch), nbytes,
                                  _at(ctx.status)), _stream()))
        return dx, dgate, dh0, None, None, None, None, None


def linear_recurrence(x: torch.Tensor, gate: torch.Tensor, *, h0: Optional[torch.Tensor] = None,
                      offsets: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None,
                      reverse: bool = False, gate_kind: str = "decay", return_state: bool = True,
                      out: Optional[torch.Tensor] = None, state_out: Optional[torch.Tensor] = None,
                      status: Optional[torch.Tensor] = None, stream=None):
    """(h, state): h_t = a_t * h_(t-1) + x_t for every sequence and channel, and every sequence's last h.

    x           [batch, time, width], or [rows, width] with offsets; float32, float16 or bfloat16; any
                strides whose last one is 1 (others are copied first)
    gate        x's leading shape and `gates` channels, width / gates consecutive channels sharing one; float32
                or x's type.  gate_kind "decay": a = gate; "log": a = exp(gate)
    h0          float32 [sequences, width], h before the first row (None: the first row is h = x there)
    offsets     int64 [sequences + 1], ascending; lengths int64 [batch].  Rows of no sequence are not used and
                come out as zeros (gradients too)
    reverse     from each sequence's last row to its first
    state       float32 [sequences, width] (None with return_state=False); an empty sequence keeps its h0
    out, state_out   write there instead of allocating (no gradients then); with `out` the rows of no
                sequence are left as they were.  state_out may be h0 itself; apart from that nothing may overlap
    status      int32[4] as of the other launches: ST_SCAN_ABORTED if a wait inside the launch ran out (rows and
                states that were not worked out, and those that depend on them, are NaN then, status or not)
    stream      where to launch (None: the current stream of x's device); gradients follow it

    Arithmetic and state are float32 whatever x's type; h is rounded once to x's type.  The bits of the result
    depend on nothing but the inputs' values and shape (a shared gate's gradient: and their alignment).  Differentiable
    once in x, gate and h0, in reverse mode (forward mode is refused); the backward pass recomputes h in float32.

    Rows are worked on in parallel, by products of gates: of up to 512 consecutive rows of a sequence, of up to 16
    channels 32768 / channels rows.  These, and exp(gate), must stay inside float32's range.  Where |a| is above 1 for so
    long that they pass it, h is infinite or NaN, even where it is zero by the formula; and an infinite h may become
    NaN, as products below the range are zero.

    Capturing a backward pass into a CUDA graph: as for any autograd function, let no eager graph of the same leaves
    live meanwhile, and warm up on a side stream."""
    if not isinstance(x, torch.Tensor) or not isinstance(gate, torch.Tensor):
        _bad("x and gate must be tensors")
    xd, gd = _DTYPES.get(x.dtype), _DTYPES.get(gate.dtype)
    if xd is None:
        _bad("x must be float32, float16 or bfloat16")
    if gd != N.DT_F32 and gd != xd:
        _bad("gate must be float32 or of x's type")
    if gate_kind != "decay" and gate_kind != "log":
        _bad(f"unknown gate_kind {gate_kind!r}")
    if offsets is not None and lengths is not None:
        _bad("offsets and lengths exclude each other")
    xs, gs, dev = tuple(x.shape), tuple(gate.shape), x.device
    if len(xs) != (2 if offsets is not None else 3) or gs[:-1] != xs[:-1]:
        _bad("x and gate must be [rows, channels] with offsets, else [batch, time, channels]")
    width, gates = xs[-1], gs[-1]
    if width < 1 or gates < 1 or width % gates:
        _bad(f"{width} channels cannot be shared by {gates} gates")
    if offsets is not None:
        if offsets.dim() != 1 or offsets.numel() < 1:
            _bad("offsets must be one-dimensional, one entry more than there are sequences")
        batch, time, sequences = 1, xs[0], offsets.numel() - 1
        _vector(offsets, "offsets", torch.int64, (sequences + 1,), dev)
    else:
        batch, time = xs[0], xs[1]
        sequences = batch
        if lengths is not None:
            _vector(lengths, "lengths", torch.int64, (batch,), dev)
    if gate.device != dev:
        _bad(f"gate is on {gate.device}, x on {dev}")
    if h0 is not None:
        _vector(h0, "h0", torch.float32, (sequences, width), dev)
    _no_tangents(x, gate, h0)
    if not x.is_cuda:
        _bad("x must be a CUDA tensor")
    if status is not None and (status.dtype != torch.int32 or status.numel() < N.STATUS_WORDS
                               or status.device != dev or not status.is_contiguous()):
        _bad(f"status must be {N.STATUS_WORDS} int32 on x's device")
    grad = torch.is_grad_enabled() and (x.requires_grad or gate.requires_grad or (h0 is not None and h0.requires_grad))
    for what, t, dtype, shape in (("out", out, x.dtype, xs), ("state_out", state_out, torch.float32, (sequences, width))):
        if t is not None:
            if grad:
                _bad("out and state_out cannot be differentiated through: detach the inputs or use torch.no_grad()")
            _vector(t, what, dtype, shape, dev)
            if not t.is_contiguous():
                _bad(f"{what} must be contiguous")
    s = _Sizes(xd, gd, batch, time, width, gates, sequences, offsets is not None, lengths is not None, int(reverse),
               int(gate_kind == "log"))
    with _Scope(dev, stream):
        x, gate = _unit(x), _unit(gate)
        if h0 is not None:
            h0 = h0.contiguous()
        if offsets is not None:
            offsets = offsets.contiguous()
        if lengths is not None:
            lengths = lengths.contiguous()
        if grad:
            return _LinearRecurrence.apply(x, gate, h0, offsets, lengths, s, return_state, status)
        return _forward(s, x, gate, h0, offsets, lengths, None, return_state, out, state_out, status)
