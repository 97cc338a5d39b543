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
from typing import Optional

import torch

from . import _native as N
from ._native import GearError, call
from .core import _ptr, _stream, _stream_scope

__all__ = ["linear_recurrence"]

_DTYPES = {torch.float32: N.DT_F32, torch.float16: N.DT_F16, torch.bfloat16: N.DT_BF16}


def _bad(msg: str):
    raise GearError(N.ERR_INVALID, "linear_recurrence: " + msg)


def _vector(t: Optional[torch.Tensor], what: str, dtype: torch.dtype, shape, device) -> None:
    if t is None:
        return
    if t.dtype != dtype or tuple(t.shape) != tuple(shape):
        _bad(f"{what} must be {dtype} of shape {list(shape)}")
    if t.device != device:
        _bad(f"{what} is on {t.device}, x on {device}")


def _unit(t: torch.Tensor) -> torch.Tensor:
    """The tensor itself where its last dimension is consecutive (any other strides), else a copy."""
    return t if t.shape[-1] == 1 or t.stride(-1) == 1 else t.contiguous()


class _Problem:
    """Sizes and checks of one call; fills the argument block of either direction."""

    def __init__(self, x, gate, h0, offsets, lengths, reverse, gate_kind):
        if not isinstance(x, torch.Tensor) or not isinstance(gate, torch.Tensor):
            _bad("x and gate must be tensors")
        if x.dtype not in _DTYPES:
            _bad("x must be float32, float16 or bfloat16")
        if gate.dtype != torch.float32 and gate.dtype != x.dtype:
            _bad("gate must be float32 or of x's type")
        if gate_kind not in ("decay", "log"):
            _bad(f"unknown gate_kind {gate_kind!r}")
        if offsets is not None and lengths is not None:
            _bad("offsets and lengths exclude each other")
        want = 2 if offsets is not None else 3
        if x.dim() != want or gate.dim() != want or gate.shape[:-1] != x.shape[:-1]:
            _bad("x and gate must be [rows, channels] with offsets, else [batch, time, channels]")
        self.width, self.gates = int(x.shape[-1]), int(gate.shape[-1])
        if self.width < 1 or self.gates < 1 or self.width % self.gates:
            _bad(f"{self.width} channels cannot be shared by {self.gates} gates")
        if offsets is not None:
            if offsets.dim() != 1 or offsets.numel() < 1:
                _bad("offsets must be one-dimensional, one entry more than there are sequences")
            self.batch, self.time, self.sequences = 1, int(x.shape[0]), int(offsets.numel()) - 1
        else:
            self.batch, self.time = int(x.shape[0]), int(x.shape[1])
            self.sequences = self.batch
        dev = x.device
        if gate.device != dev:
            _bad(f"gate is on {gate.device}, x on {dev}")
        _vector(offsets, "offsets", torch.int64, (self.sequences + 1,), dev)
        _vector(lengths, "lengths", torch.int64, (self.batch,), dev)
        _vector(h0, "h0", torch.float32, (self.sequences, self.width), dev)
        if not x.is_cuda:
            _bad("x must be a CUDA tensor")
        self.reverse, self.log = bool(reverse), gate_kind == "log"

    def args(self, x, gate, h0, offsets, lengths) -> "N.RecurrenceArgs":
        a = N.RecurrenceArgs()
        a.x, a.gate = x.data_ptr(), gate.data_ptr()
        a.x_dtype, a.gate_dtype = _DTYPES[x.dtype], _DTYPES[gate.dtype]
        a.batch, a.time, a.width, a.gates = self.batch, self.time, self.width, self.gates
        a.x_batch_stride, a.x_row_stride = self.strides(x)
        a.gate_batch_stride, a.gate_row_stride = self.strides(gate)
        a.offsets, a.lengths, a.sequences = _ptr(offsets), _ptr(lengths), self.sequences
        a.h0 = _ptr(h0)
        a.reverse, a.gate_log = int(self.reverse), int(self.log)
        return a

    @staticmethod
    def strides(t):
        return (0, t.stride(0)) if t.dim() == 2 else (t.stride(0), t.stride(1))

    @staticmethod
    def sizes(a, backward: bool):
        scratch, carry = C.c_int64(0), C.c_int64(0)
        call("gearb_recurrence_bytes", C.byref(a), int(backward), C.byref(scratch), C.byref(carry))
        return scratch.value, carry.value


def _forward(p, x, gate, h0, offsets, lengths, need_carry, return_state, out, state_out, status):
    if state_out is not None and h0 is not None and p.time != 1 and state_out.data_ptr() == h0.data_ptr():
        h0 = h0.clone()    # rows of one sequence are worked on in several places: one may be done before another reads h0
    a = p.args(x, gate, h0, offsets, lengths)
    a.zero_rest = int(out is None)
    h = torch.empty(x.shape, dtype=x.dtype, device=x.device) if out is None else out
    state = state_out
    if state is None and return_state:
        state = torch.empty((p.sequences, p.width), dtype=torch.float32, device=x.device)
    scratch_bytes, carry_bytes = p.sizes(a, False)
    scratch = torch.empty(scratch_bytes, dtype=torch.uint8, device=x.device)
    carry = torch.empty(carry_bytes // 4 if need_carry else 0, dtype=torch.float32, device=x.device)
    a.out, a.state_out = h.data_ptr(), _ptr(state)
    a.carry = carry.data_ptr() if need_carry else None
    a.scratch, a.scratch_bytes, a.status = scratch.data_ptr(), scratch_bytes, _ptr(status)
    call("gearb_recurrence_forward", C.byref(a), _stream())
    return h, state, carry


class _LinearRecurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, h0, offsets, lengths, p, return_state, status):
        h, state, carry = _forward(p, x, gate, h0, offsets, lengths, True, return_state, None, None, status)
        ctx.save_for_backward(x, gate, h0, offsets, lengths, carry)
        ctx.p, ctx.status = p, status
        ctx.set_materialize_grads(False)
        return h, state

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh, dstate):
        x, gate, h0, offsets, lengths, carry = ctx.saved_tensors
        p = ctx.p
        with torch.cuda.device(x.device):
            dh = torch.zeros_like(x) if dh is None else _unit(dh)
            dstate = None if dstate is None else dstate.contiguous()
            a = p.args(x, gate, h0, offsets, lengths)
            a.zero_rest = 1
            dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
            dgate = torch.empty(gate.shape, dtype=gate.dtype, device=x.device)
            dh0 = None if h0 is None else torch.empty(h0.shape, dtype=torch.float32, device=x.device)
            scratch_bytes, _ = p.sizes(a, True)
            scratch = torch.empty(scratch_bytes, dtype=torch.uint8, device=x.device)
            a.carry, a.dout, a.dstate = carry.data_ptr(), dh.data_ptr(), _ptr(dstate)
            a.dout_batch_stride, a.dout_row_stride = p.strides(dh)
            a.dx, a.dgate, a.dh0 = dx.data_ptr(), dgate.data_ptr(), _ptr(dh0)
            a.scratch, a.scratch_bytes, a.status = scratch.data_ptr(), scratch_bytes, _ptr(ctx.status)
            call("gearb_recurrence_backward", C.byref(a), _stream())
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
    status      int32[4] as of the other launches: ST_SCAN_ABORTED if a wait inside the launch ran out (h is
                NaN from there on)

    Arithmetic and state are float32 whatever x's type; h is rounded once to x's type.  Results do not depend
    on timing, nor on the other sequences of the batch except through the tiling of the sums (float32
    rounding).  Differentiable once in x, gate and h0; the backward pass recomputes h in float32.  Gates whose
    product over some thousand rows passes float32's range (|a| well above 1) overflow."""
    p = _Problem(x, gate, h0, offsets, lengths, reverse, gate_kind)
    if status is not None and (status.dtype != torch.int32 or status.numel() < N.STATUS_WORDS
                               or status.device != x.device or not status.is_contiguous()):
        _bad(f"status must be {N.STATUS_WORDS} int32 on x's device")
    grad = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, gate, h0))
    if grad and (out is not None or state_out is not None):
        _bad("out and state_out cannot be differentiated through: detach the inputs or use torch.no_grad()")
    for what, t, dtype, shape in (("out", out, x.dtype, x.shape),
                                  ("state_out", state_out, torch.float32, (p.sequences, p.width))):
        _vector(t, what, dtype, shape, x.device)
        if t is not None and not t.is_contiguous():
            _bad(f"{what} must be contiguous")
    with torch.cuda.device(x.device), _stream_scope(stream):
        x, gate = _unit(x), _unit(gate)
        h0 = None if h0 is None else h0.contiguous()
        offsets = None if offsets is None else offsets.contiguous()
        lengths = None if lengths is None else lengths.contiguous()
        if grad:
            return _LinearRecurrence.apply(x, gate, h0, offsets, lengths, p, return_state, status)
        h, state, _ = _forward(p, x.detach(), gate.detach(), h0, offsets, lengths, False, return_state, out, state_out,
                               status)
        return h, state
