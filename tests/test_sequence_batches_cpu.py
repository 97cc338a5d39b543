"""Argument checks of the sequence-batch operators that need no GPU, and the reference the GPU tests use."""
import ctypes as C

import numpy as np
import pytest
import torch

import recurrence_ref as R
from gear_b200 import _native as N
from gear_b200 import core, layout, recurrence


def test_python_side_refuses_cpu_tensors_and_bad_shapes():
    x = torch.zeros(2, 3, 4)
    for f in (lambda: recurrence.linear_recurrence(x, x), lambda: recurrence.linear_recurrence(x, x[..., :3]),
              lambda: recurrence.linear_recurrence(x, x[:1]), lambda: recurrence.linear_recurrence(x.int(), x.int()),
              lambda: recurrence.linear_recurrence(x, x, gate_kind="?"),
              lambda: recurrence.linear_recurrence(x[0], x[0]),
              lambda: recurrence.linear_recurrence(x, x, offsets=torch.zeros(2, dtype=torch.int64)),
              lambda: recurrence.linear_recurrence(x, x, offsets=torch.zeros(2, dtype=torch.int64),
                                                   lengths=torch.zeros(2, dtype=torch.int64)),
              lambda: layout.paged_layout(torch.zeros(2, dtype=torch.int64), 4, torch.zeros(2, 2, dtype=torch.int32),
                                          torch.zeros(1, dtype=torch.int64), num_pages=3)):
        with pytest.raises(core.GearError) as e:
            f()
        assert e.value.code == N.ERR_INVALID


def recurrence_args(**kw):
    a = N.RecurrenceArgs()
    base = dict(x=4096, gate=4096, out=4096, x_dtype=N.DT_F32, gate_dtype=N.DT_F32, batch=2, time=3, width=4, gates=4,
                sequences=2)
    for k, v in {**base, **kw}.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw", [
    dict(batch=-1), dict(time=-1), dict(width=0), dict(gates=0), dict(width=5, gates=2), dict(x_dtype=N.DT_I64),
    dict(x_dtype=N.DT_F16, gate_dtype=N.DT_BF16), dict(sequences=3), dict(offsets=4096), dict(x=None), dict(gate=None),
    dict(out=None), dict(offsets=4096, lengths=4096, batch=1), dict(width=(1 << 24) + 1, gates=1),
    dict(batch=1 << 30, time=1 << 30, sequences=1 << 30),
])
def test_recurrence_entry_points_refuse(kw):
    a = recurrence_args(**kw)
    assert N.lib.gearb_recurrence_forward(C.byref(a), None) == N.ERR_INVALID and N.last_error()


def test_recurrence_backward_entry_refuses_missing_buffers_and_short_scratch():
    a = recurrence_args()
    assert N.lib.gearb_recurrence_backward(C.byref(a), None) == N.ERR_INVALID
    for f in (N.lib.gearb_recurrence_forward, N.lib.gearb_recurrence_backward):
        assert f(None, None) == N.ERR_INVALID
    s, c = C.c_int64(), C.c_int64()
    assert N.lib.gearb_recurrence_bytes(C.byref(a), 1, C.byref(s), C.byref(c)) == N.OK
    assert s.value >= 0 and c.value >= 0
    assert N.lib.gearb_recurrence_bytes(None, 1, C.byref(s), C.byref(c)) == N.ERR_INVALID
    bad = recurrence_args(width=0)
    assert N.lib.gearb_recurrence_bytes(C.byref(bad), 0, C.byref(s), C.byref(c)) == N.ERR_INVALID


def layout_args(**kw):
    a = N.LayoutArgs()
    base = dict(lengths=4096, requests=3, page=4, max_blocks=2, block_table=4096, num_pages=5, used_in=4096,
                used_out=4096, offsets=4096, scratch=4096, scratch_bytes=1 << 20)
    for k, v in {**base, **kw}.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw", [
    dict(requests=-1), dict(page=0), dict(max_blocks=0), dict(num_pages=-1), dict(max_tokens=-1), dict(max_tokens=4),
    dict(used_in=None), dict(used_out=None), dict(offsets=None), dict(lengths=None), dict(block_table=None),
    dict(scratch=None), dict(scratch_bytes=0), dict(page=1 << 31), dict(page=1 << 40, max_blocks=1 << 40),
    dict(requests=1 << 31), dict(num_pages=(1 << 31) + 1),
])
def test_layout_entry_point_refuses(kw):
    a = layout_args(**kw)
    assert N.lib.gearb_layout_paged(C.byref(a), None) == N.ERR_INVALID and N.last_error()


def test_gather_packed_entry_refuses():
    t = core.TrajectoryTable([8, 4], 10, 3)
    t.connect()
    h = core.StorageHandler(t)
    h.set([0, 1], [core.SubscribePattern(0, 3), core.SubscribePattern(0, 4)])
    one = (C.c_void_p * 2)(4096, 4096)
    rows = (C.c_int64 * 2)(5, 5)
    cols = (C.c_int32 * 2)(0, 1)
    p = C.c_void_p(4096)
    f = N.lib.gearb_handler_gather_packed
    assert f(h._h, cols, 2, p, p, p, 1, p, None, 0, 0, None, one, rows, None, None) != N.OK
    assert N.lib.gearb_handler_segment_lengths(h._h, 0, None, None, None, 2, None, None) == N.ERR_INVALID
    assert N.lib.gearb_handler_segment_lengths(h._h, 5, p, p, p, 2, p, None) == N.ERR_INVALID
    assert N.lib.gearb_handler_segment_lengths(h._h, 0, p, p, p, -1, p, None) == N.ERR_INVALID
    assert N.lib.gearb_handler_segment_lengths(h._h, 0, None, None, None, 0, None, None) == N.OK


@pytest.mark.parametrize("reverse,log", [(False, False), (True, True)])
def test_reference_gradients_agree_with_autograd(reverse, log):
    """The float64 reference against torch's own differentiation of the definition."""
    rng = np.random.default_rng(0)
    rows, d, g = 40, 6, 3
    off = [0, 13, 13, 40]
    x, gate = rng.standard_normal((rows, d)), rng.uniform(-1, -0.1, (rows, g))
    h0, dh, dst = rng.standard_normal((3, d)), rng.standard_normal((rows, d)), rng.standard_normal((3, d))
    r = R.reference(x, gate, [(0, 13), (13, 13), (13, 40)], h0, reverse, log, dh, dst)
    tx, tg, th = (torch.from_numpy(v).requires_grad_(True) for v in (x, gate, h0))
    a = (tg.exp() if log else tg).repeat_interleave(2, 1)
    loss = 0.0
    for s in range(3):
        cur = th[s]
        order = range(off[s], off[s + 1])
        for i in (reversed(order) if reverse else order):
            cur = a[i] * cur + tx[i]
            assert np.allclose(cur.detach(), r["h"][0][i])
            loss = loss + (cur * torch.from_numpy(dh[i])).sum()
        loss = loss + (cur * torch.from_numpy(dst[s])).sum()
    loss.backward()
    for got, key in ((tx.grad, "dx"), (tg.grad, "dgate"), (th.grad, "dh0")):
        assert np.allclose(got.numpy(), r[key][0])
