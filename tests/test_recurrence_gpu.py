"""Linear recurrences on the GPU against a row-by-row float64 reference (recurrence_ref.py derives the tolerances)."""
import numpy as np
import pytest
import torch

import recurrence_ref as R
from gear_b200 import _native as N
from gear_b200 import core, recurrence

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def make(seed, lead, width, gates, dtype, gate_dtype, log, one_step=False):
    rng = np.random.default_rng(seed)
    x = torch.from_numpy(rng.standard_normal(lead + (width,)).astype(np.float32)).to(dtype).to(DEV)
    a = np.exp(-np.exp(rng.uniform(-7, 1, lead + (gates,))))
    if not log:
        a = a * np.where(rng.random(a.shape) < 0.02, 0.0, np.sign(rng.uniform(-0.2, 1, a.shape)))
    gate = torch.from_numpy((np.log(a) if log else a).astype(np.float32)).to(gate_dtype).to(DEV)
    return x, gate


def dbl(t):
    return None if t is None else t.detach().double().cpu().numpy()


def run_and_check(x, gate, h0=None, offsets=None, lengths=None, reverse=False, log=False, train=True, seed=0,
                  with_dstate=True):
    """Forward without and with gradients, backward; everything against the reference."""
    width, gates = x.shape[-1], gate.shape[-1]
    time = x.shape[0] if offsets is not None else x.shape[1]
    rows = x.shape[0] if offsets is not None else x.shape[0] * x.shape[1]
    ns = offsets.numel() - 1 if offsets is not None else x.shape[0]
    seqs = R.spans(rows, time, dbl(offsets), dbl(lengths))
    kind = "log" if log else "decay"
    rng = np.random.default_rng(seed + 99)
    dh = torch.from_numpy(rng.standard_normal(tuple(x.shape)).astype(np.float32)).to(x.dtype).to(DEV)
    dstate = torch.from_numpy(rng.standard_normal((ns, width)).astype(np.float32)).to(DEV) if with_dstate else None
    owned = np.zeros(rows, bool)
    for lo, hi in seqs:
        owned[lo:hi] = True
    # what no sequence owns must not matter: NaN there for the kernel, zeros for the reference
    hole = torch.from_numpy(~owned).to(DEV).reshape(x.shape[:-1] + (1,))
    xk, gk, dk = (torch.where(hole, float("nan"), t.float()).to(t.dtype) for t in (x, gate, dh))
    flat = lambda t, c: dbl(t).reshape(rows, c)
    want = R.reference(flat(x, width), flat(gate, gates), seqs, dbl(h0), reverse, log, flat(dh, width), dbl(dstate))
    kw = dict(offsets=offsets, lengths=lengths, reverse=reverse, gate_kind=kind)

    h, state = recurrence.linear_recurrence(xk, gk, h0=h0, **kw)
    R.check(h, want["h"], x.dtype, "h")
    R.check(state, want["state"], F32, "state")
    assert h.dtype == x.dtype and state.dtype == F32 and h.shape == x.shape
    if not owned.all():
        assert (h.reshape(rows, width)[torch.from_numpy(~owned).to(DEV)] == 0).all()
    if not train:
        return h, state
    leaves = [t.clone().requires_grad_(True) for t in (xk, gk)] + ([h0.clone().requires_grad_(True)] if h0 is not None else [])
    h2, state2 = recurrence.linear_recurrence(leaves[0], leaves[1], h0=leaves[2] if h0 is not None else None, **kw)
    assert torch.equal(h2, h) and torch.equal(state2, state)
    outs, gouts = ([h2, state2], [dk, dstate]) if with_dstate else ([h2], [dk])
    grads = torch.autograd.grad(outs, leaves, gouts)
    R.check(grads[0], want["dx"], x.dtype, "dx")
    R.check(grads[1], want["dgate"], gate.dtype, "dgate")
    if h0 is not None:
        R.check(grads[2], want["dh0"], F32, "dh0")
    if not owned.all():
        sel = torch.from_numpy(~owned).to(DEV)
        assert (grads[0].reshape(rows, width)[sel] == 0).all() and (grads[1].reshape(rows, gates)[sel] == 0).all()
    return h, state


def state_of(seed, n, width):
    return torch.from_numpy(np.random.default_rng(seed).standard_normal((n, width)).astype(np.float32)).to(DEV)


DENSE = [
    # batch, time, width, gates
    (1, 1, 1, 1), (1, 1, 5, 5), (3, 1, 64, 64), (7, 1, 130, 2), (1, 2, 33, 33), (2, 63, 32, 32), (2, 64, 32, 1),
    (2, 65, 31, 31), (1, 127, 64, 64), (1, 128, 128, 4), (3, 129, 129, 1), (1, 1000, 1, 1), (5, 333, 1, 1),
    (2, 517, 2, 2), (1, 700, 3, 1), (2, 300, 7, 7), (1, 900, 16, 4), (2, 257, 100, 5), (1, 2500, 40, 8),
    (1, 1537, 256, 256), (2, 640, 300, 3), (9, 40, 257, 257), (1, 5000, 8, 8), (1, 20000, 1, 1), (300, 3, 4, 2),
]


@pytest.mark.parametrize("batch,time,width,gates", DENSE)
@pytest.mark.parametrize("dtype,gate_dtype", [(F32, F32), (BF16, F32)])
def test_dense(batch, time, width, gates, dtype, gate_dtype):
    seed = batch * 1000003 + time * 101 + width
    log, reverse = bool((time + width) & 1), bool((batch + gates) & 1)
    x, gate = make(seed, (batch, time), width, gates, dtype, gate_dtype, log)
    h0 = state_of(seed, batch, width) if (time + gates) % 3 else None
    run_and_check(x, gate, h0, reverse=reverse, log=log, seed=seed, with_dstate=bool(time % 2))


@pytest.mark.parametrize("dtype,gate_dtype", [(F32, F32), (F16, F32), (F16, F16), (BF16, F32), (BF16, BF16)])
@pytest.mark.parametrize("log", [False, True])
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("width,gates", [(96, 96), (96, 3), (6, 6), (6, 2)])
def test_types_and_directions(dtype, gate_dtype, log, reverse, width, gates):
    x, gate = make(7, (3, 210), width, gates, dtype, gate_dtype, log)
    run_and_check(x, gate, state_of(8, 3, width), reverse=reverse, log=log)


LENGTHS = [
    [0], [0, 0, 0], [5], [1, 1, 1, 1], [64, 64, 64], [63, 1, 64, 0, 65, 0], [0, 300, 0, 0, 7, 129, 0],
    [1] * 200, [0, 1] * 100, [1000, 3, 0, 500, 31, 32, 33], [2000],
]


@pytest.mark.parametrize("lens", LENGTHS)
@pytest.mark.parametrize("width,gates", [(1, 1), (3, 3), (40, 8), (64, 1), (200, 200)])
@pytest.mark.parametrize("reverse", [False, True])
def test_packed(lens, width, gates, reverse):
    off = torch.from_numpy(np.concatenate([[0], np.cumsum(lens)])).to(DEV)
    rows = sum(lens) + (len(lens) % 3) * 50        # rows behind the last sequence
    seed = rows + width
    log = bool(len(lens) & 1)
    x, gate = make(seed, (rows,), width, gates, BF16 if gates == 8 else F32, F32, log)
    h0 = state_of(seed, len(lens), width) if len(lens) % 2 or reverse else None
    run_and_check(x, gate, h0, offsets=off, reverse=reverse, log=log)


@pytest.mark.parametrize("width,gates", [(1, 1), (5, 1), (48, 48), (136, 2)])
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("time", [1, 31, 64, 200, 777])
def test_padded(width, gates, reverse, time):
    rng = np.random.default_rng(time)
    lens = rng.integers(0, time + 1, 9)
    lens[0], lens[1] = 0, time
    x, gate = make(time, (9, time), width, gates, F32, F32, True)
    run_and_check(x, gate, state_of(time, 9, width), lengths=torch.from_numpy(lens).to(DEV), reverse=reverse, log=True)


def slow(seed, lead, width, gates, dtype, gate_dtype):
    """Log gates that remember thousands of rows."""
    rng = np.random.default_rng(seed)
    x = torch.from_numpy(rng.standard_normal(lead + (width,)).astype(np.float32)).to(dtype).to(DEV)
    g = torch.from_numpy((-rng.uniform(0, 1e-3, lead + (gates,))).astype(np.float32)).to(gate_dtype).to(DEV)
    return x, g


# One channel block of the streaming kernels, rows that only the fallback reads, few channels at 4 and 16 rows a thread.
@pytest.mark.parametrize("batch,time,width,gates", [(1, 9500, 48, 48), (2, 8500, 64, 4), (1, 9500, 43, 43), (2, 4400, 33, 3),
                                                    (2, 9000, 16, 16), (1, 40000, 16, 4), (1, 140000, 1, 1)])
@pytest.mark.parametrize("reverse", [False, True])
def test_states_over_thousands_of_rows(batch, time, width, gates, reverse):
    x, gate = slow(time + width, (batch, time), width, gates, F32, F32)
    run_and_check(x, gate, h0=state_of(8, batch, width), reverse=reverse, log=True)


@pytest.mark.parametrize("width,gates", [(48, 48), (43, 43), (64, 2), (12, 12)])
@pytest.mark.parametrize("reverse", [False, True])
def test_packed_starts_anywhere_in_thousands_of_rows(width, gates, reverse):
    # starts on, before and behind the ends of tiles, of eight tiles and of sixty-four
    lens = [3, 700, 3393, 4096, 0, 1, 4607, 512, 63, 5000, 1, 4200]
    off = torch.tensor(np.cumsum([0] + lens), dtype=torch.int64, device=DEV)
    x, gate = slow(17, (int(off[-1]),), width, gates, BF16, F32)
    run_and_check(x, gate, h0=state_of(9, len(lens), width), offsets=off, reverse=reverse, log=True)


@pytest.mark.parametrize("width", [48, 45, 5])
def test_padded_ends_anywhere_in_thousands_of_rows(width):
    x, gate = slow(18, (4, 6000), width, width, F32, F32)
    lens = torch.tensor([6000, 4097, 0, 4544], dtype=torch.int64, device=DEV)
    for reverse in (False, True):
        run_and_check(x, gate, lengths=lens, reverse=reverse, log=True)


def test_offsets_need_not_start_at_row_zero():
    off = torch.tensor([10, 10, 75, 200], device=DEV)
    for width, reverse in ((1, True), (70, False), (70, True), (4, False)):
        x, gate = make(3, (260,), width, width, F32, F32, False)
        run_and_check(x, gate, state_of(1, 3, width), offsets=off, reverse=reverse)


@pytest.mark.parametrize("width,gates", [(64, 64), (2, 1), (72, 8)])
def test_strides(width, gates):
    """Slices of wider rows, time-major storage, a gate expanded over time or over the batch, odd base addresses."""
    rng = np.random.default_rng(0)
    wide = torch.from_numpy(rng.standard_normal((3, 150, 2 * width + 3)).astype(np.float32)).to(DEV)
    x, g = wide[..., 3:3 + width], torch.sigmoid(wide[..., 1:1 + gates])
    run_and_check(x, g, state_of(0, 3, width))
    tm = torch.from_numpy(rng.standard_normal((150, 3, width)).astype(np.float32)).to(BF16).to(DEV).transpose(0, 1)
    run_and_check(tm, g, state_of(0, 3, width))
    per_channel = torch.sigmoid(wide[0, 0, :gates]).expand(3, 150, gates)
    per_step = torch.sigmoid(wide[0, :, :gates]).unsqueeze(0).expand(3, 150, gates)
    for e in (per_channel, per_step):
        h, _ = recurrence.linear_recurrence(x, e)
        assert torch.equal(h, recurrence.linear_recurrence(x.contiguous(), e.contiguous())[0])
    p = wide.reshape(-1, 2 * width + 3)[:, 2:2 + width]
    off = torch.tensor([0, 100, 450], device=DEV)
    run_and_check(p, torch.sigmoid(wide.reshape(-1, 2 * width + 3)[:, :gates]), None, offsets=off, reverse=True)
    # last dimension not consecutive: copied
    t = torch.from_numpy(rng.standard_normal((2, width, 50)).astype(np.float32)).to(DEV).transpose(1, 2)
    run_and_check(t, torch.sigmoid(t[..., :gates]), None)


def test_gradient_of_a_broadcast_gate_and_of_a_summed_loss():
    x, gate = make(5, (2, 130), 32, 32, F32, F32, False)
    decay = gate[0, 0].clone().requires_grad_(True)
    h, _ = recurrence.linear_recurrence(x, decay.expand(2, 130, 32), return_state=False)
    h.sum().backward()                     # an expanded gradient of ones: strides 0
    d2 = gate[0, 0].clone().double().cpu().requires_grad_(True)
    cur, tot = torch.zeros(2, 32, dtype=torch.float64), 0.0
    for t in range(130):
        cur = d2 * cur + x[:, t].double().cpu()
        tot = tot + cur.sum()
    tot.backward()
    scale = d2.grad.abs().max()
    # 260 rows are summed, each a few dozen roundings of values that may be hundreds of times the result
    assert (decay.grad.double().cpu() - d2.grad).abs().max() <= 1e-4 * scale


@pytest.mark.parametrize("width,gates,reverse,log", [(3, 3, False, True), (64, 4, True, False), (1, 1, True, False)])
def test_gradients_against_differences(width, gates, reverse, log):
    """<gradient, v> against central differences of the float64 reference's loss along v."""
    x, gate = make(11, (2, 90), width, gates, F32, F32, log)
    h0 = state_of(12, 2, width)
    rng = np.random.default_rng(1)
    dh, dst = rng.standard_normal((180, width)), rng.standard_normal((2, width))
    dh, dst = dh.astype(np.float32).astype(np.float64), dst.astype(np.float32).astype(np.float64)
    seqs = R.spans(180, 90, None, None)

    def loss(xx, gg, hh):
        r = R.reference(xx, gg, seqs, hh, reverse, log)
        return (r["h"][0] * dh).sum() + (r["state"][0] * dst).sum()

    base = [dbl(x).reshape(180, width), dbl(gate).reshape(180, gates), dbl(h0)]
    full = R.reference(*base[:2], seqs, base[2], reverse, log, dh, dst)
    leaves = [t.clone().requires_grad_(True) for t in (x, gate, h0)]
    h, s = recurrence.linear_recurrence(*leaves[:2], h0=leaves[2], reverse=reverse, gate_kind="log" if log else "decay")
    grads = torch.autograd.grad([h, s], leaves, [torch.from_numpy(dh).float().reshape(h.shape).to(DEV),
                                                 torch.from_numpy(dst).float().to(DEV)])
    for i, key in enumerate(("dx", "dgate", "dh0")):
        v = rng.standard_normal(base[i].shape)
        eps = 1e-5
        up, dn = list(base), list(base)
        up[i], dn[i] = base[i] + eps * v, base[i] - eps * v
        diff = (loss(*up) - loss(*dn)) / (2 * eps)
        got = (dbl(grads[i]).reshape(v.shape) * v).sum()
        # the kernel's own bound, and what the difference loses: 1e-11 of the loss's size over eps, eps^2 relative
        size = np.abs(full[key][0] * v).sum()
        tol = ((full[key][1] + U32 * np.abs(full[key][0])) * np.abs(v)).sum() + 1e-6 * size + 1e-6
        assert abs(got - diff) <= tol, (key, got, diff, tol)


U32 = 2.0 ** -24


def test_a_poisoned_sequence_stays_alone():
    """NaN and infinities inside one sequence do not reach its neighbours, in either direction or pass."""
    lens = [70, 64, 1, 200, 90]
    off = torch.from_numpy(np.concatenate([[0], np.cumsum(lens)])).to(DEV)
    for width in (1, 4, 64):
        for reverse in (False, True):
            x, gate = make(2, (sum(lens),), width, width, F32, F32, False)
            clean = run_and_check(x, gate, None, offsets=off, reverse=reverse)[0]
            bx, bg = x.clone(), gate.clone()
            bx[140:150], bg[150:160] = float("nan"), float("inf")     # in sequence 3 (rows 135..334)
            leaves = [bx.requires_grad_(True), bg.requires_grad_(True)]
            h, _ = recurrence.linear_recurrence(*leaves, offsets=off, reverse=reverse)
            assert torch.equal(h[:135], clean[:135]) and torch.equal(h[335:], clean[335:])
            dx, dg = torch.autograd.grad(h, leaves, torch.ones_like(h))
            for t in (dx, dg):
                assert torch.isfinite(t[:135]).all() and torch.isfinite(t[335:]).all()


def test_log_gate_of_minus_infinity_forgets():
    x, gate = make(4, (1, 200), 64, 64, F32, F32, True)
    gate[:, 77] = -float("inf")
    h, _ = recurrence.linear_recurrence(x, gate, gate_kind="log")
    assert torch.equal(h[:, 77], x[:, 77])
    rest, _ = recurrence.linear_recurrence(x[:, 77:], gate[:, 77:], gate_kind="log")
    want = R.reference(dbl(x[0, 77:]), dbl(gate[0, 77:]), [(0, 123)], log=True)["h"]
    R.check(h[0, 77:], want, F32, "h behind the reset")
    R.check(rest[0], want, F32, "h from the reset")


@pytest.mark.parametrize("width,gates,lead", [(1, 1, (4, 3000)), (64, 64, (1, 4000)), (96, 3, (2, 2000))])
def test_same_bits_every_time(width, gates, lead):
    x, gate = make(6, lead, width, gates, BF16, F32, True)
    dh = torch.randn(lead + (width,), device=DEV).to(BF16)

    def once():
        leaves = [x.clone().requires_grad_(True), gate.clone().requires_grad_(True)]
        h, s = recurrence.linear_recurrence(*leaves, gate_kind="log")
        return [h, s, *torch.autograd.grad(h, leaves, dh)]

    first = once()
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(first, once()))


def test_out_state_out_and_rows_left_alone():
    lens = [30, 0, 101]
    off = torch.tensor([0, 30, 30, 131], device=DEV)
    for width in (1, 64):
        x, gate = make(9, (150,), width, width, F32, F32, False)
        h0 = state_of(1, 3, width)
        want, ws = recurrence.linear_recurrence(x, gate, h0=h0, offsets=off)
        out = torch.full_like(x, 7.0)
        state = h0.clone()
        h, s = recurrence.linear_recurrence(x, gate, h0=state, offsets=off, out=out, state_out=state)
        assert h is out and s is state
        assert torch.equal(out[:131], want[:131]) and (out[131:] == 7.0).all() and torch.equal(state, ws)
        assert torch.equal(ws[1], h0[1])


def test_step_by_step_equals_the_whole():
    """One token at a time with the carried state gives the whole sequence's values (within float32 rounding)."""
    x, gate = make(10, (3, 25), 130, 130, F32, F32, True)
    want = R.reference(dbl(x).reshape(75, 130), dbl(gate).reshape(75, 130), R.spans(75, 25, None, None), log=True)
    state = torch.zeros(3, 130, device=DEV)
    got = []
    for t in range(25):
        h, _ = recurrence.linear_recurrence(x[:, t:t + 1], gate[:, t:t + 1], h0=state, state_out=state, gate_kind="log")
        got.append(h)
    R.check(torch.cat(got, 1), want["h"], F32, "h")
    R.check(state, want["state"], F32, "state")


def test_graph_replay_and_other_streams():
    x, gate = make(13, (2, 900), 72, 72, BF16, F32, True)
    want, ws = recurrence.linear_recurrence(x, gate, gate_kind="log")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    h, s = recurrence.linear_recurrence(x, gate, gate_kind="log", stream=side)
    side.synchronize()
    assert torch.equal(h, want) and torch.equal(s, ws)
    # two captured graphs of the forward and one of a training step, replayed together on two streams
    xs = [x.clone(), x.clone()]
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(recurrence.linear_recurrence(xs[i], gate, gate_kind="log"))
        graphs.append(g)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for k in range(3):
        xs[0].copy_(x * (k + 1)), xs[1].copy_(x * -(k + 1))
        torch.cuda.synchronize()
        for g, s in zip(graphs, (s1, s2)):
            with torch.cuda.stream(s):
                for _ in range(4):
                    g.replay()
        torch.cuda.synchronize()
        for i in range(2):
            e, _ = recurrence.linear_recurrence(xs[i], gate, gate_kind="log")
            assert torch.equal(outs[i][0], e)


def test_training_step_in_a_graph():
    x, gate = make(14, (2, 300), 64, 64, F32, F32, False)
    dh = torch.randn_like(x)
    eager = [t.clone().requires_grad_(True) for t in (x, gate)]
    h, _ = recurrence.linear_recurrence(*eager)
    want = torch.autograd.grad(h, eager, dh)
    leaves = [t.clone().requires_grad_(True) for t in (x, gate)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):                  # warm up as torch asks
        hh, _ = recurrence.linear_recurrence(*leaves)
        torch.autograd.grad(hh, leaves, dh)
        del hh
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        hh, _ = recurrence.linear_recurrence(*leaves)
        got = torch.autograd.grad(hh, leaves, dh)
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_concurrent_calls_on_two_streams():
    x, gate = make(15, (1, 6000), 64, 64, F32, F32, True)
    want, _ = recurrence.linear_recurrence(x, gate, gate_kind="log")
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for _ in range(10):
        for s in streams:
            outs.append(recurrence.linear_recurrence(x, gate, gate_kind="log", stream=s)[0])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_empty_batches():
    for width in (1, 64):
        e = torch.zeros(0, width, device=DEV)
        h0 = state_of(0, 2, width)
        h, s = recurrence.linear_recurrence(e, e, h0=h0, offsets=torch.zeros(3, dtype=torch.int64, device=DEV))
        assert h.shape == (0, width) and torch.equal(s, h0)
        h, s = recurrence.linear_recurrence(e, e, offsets=torch.zeros(1, dtype=torch.int64, device=DEV))
        assert s.shape == (0, width)
        z = torch.zeros(3, 0, width, device=DEV, requires_grad=True)
        h0 = state_of(0, 3, width).requires_grad_(True)
        h, s = recurrence.linear_recurrence(z, torch.zeros(3, 0, width, device=DEV), h0=h0)
        assert torch.equal(s, h0)
        d, = torch.autograd.grad(s, [h0], torch.ones_like(s))
        assert (d == 1).all()
        n = torch.zeros(0, 4, width, device=DEV)
        h, s = recurrence.linear_recurrence(n, n)
        assert h.shape == (0, 4, width) and s.shape == (0, width)
        # rows, but no sequence
        h, s = recurrence.linear_recurrence(torch.ones(5, width, device=DEV), torch.ones(5, width, device=DEV),
                                            offsets=torch.zeros(1, dtype=torch.int64, device=DEV))
        assert (h == 0).all()


def test_offsets_and_lengths_outside_the_rows_are_cut():
    x, gate = make(1, (100,), 64, 64, F32, F32, False)
    off = torch.tensor([0, 40, 1 << 40], device=DEV)
    h, s = recurrence.linear_recurrence(x, gate, offsets=off)
    want, ws = recurrence.linear_recurrence(x, gate, offsets=torch.tensor([0, 40, 100], device=DEV))
    assert torch.equal(h, want) and torch.equal(s, ws)
    h, s = recurrence.linear_recurrence(x[None], gate[None], lengths=torch.tensor([1 << 50], device=DEV))
    assert torch.equal(h, recurrence.linear_recurrence(x[None], gate[None])[0])
    h, s = recurrence.linear_recurrence(x[None], gate[None], lengths=torch.tensor([-3], device=DEV))
    assert (h == 0).all() and (s == 0).all()


def test_refusals():
    x = torch.zeros(2, 5, 6, device=DEV)
    g = torch.zeros(2, 5, 6, device=DEV)
    bad = [
        lambda: recurrence.linear_recurrence(x.double(), g.double()),
        lambda: recurrence.linear_recurrence(x, g.half()),
        lambda: recurrence.linear_recurrence(x, g[..., :4]),
        lambda: recurrence.linear_recurrence(x, g[:, :4]),
        lambda: recurrence.linear_recurrence(x, g, gate_kind="tanh"),
        lambda: recurrence.linear_recurrence(x, g, h0=torch.zeros(2, 5, device=DEV)),
        lambda: recurrence.linear_recurrence(x, g, h0=torch.zeros(2, 6, device=DEV).half()),
        lambda: recurrence.linear_recurrence(x, g, h0=torch.zeros(2, 6)),
        lambda: recurrence.linear_recurrence(x, g, lengths=torch.zeros(3, dtype=torch.int64, device=DEV)),
        lambda: recurrence.linear_recurrence(x, g, lengths=torch.zeros(2, dtype=torch.int32, device=DEV)),
        lambda: recurrence.linear_recurrence(x, g, offsets=torch.zeros(2, dtype=torch.int64, device=DEV)),
        lambda: recurrence.linear_recurrence(x, g, out=torch.zeros(2, 5, 5, device=DEV)),
        lambda: recurrence.linear_recurrence(x, g, out=torch.zeros(2, 6, 5, device=DEV).transpose(1, 2)),
        lambda: recurrence.linear_recurrence(x.clone().requires_grad_(True), g, out=torch.zeros_like(x)),
        lambda: recurrence.linear_recurrence(x, g, status=torch.zeros(2, dtype=torch.int32, device=DEV)),
        lambda: recurrence.linear_recurrence(x.cpu(), g.cpu()),
        lambda: recurrence.linear_recurrence(x, g.cpu()),
    ]
    for f in bad:
        with pytest.raises(core.GearError) as e:
            f()
        assert e.value.code == N.ERR_INVALID
    # only once differentiable
    xg = x.clone().requires_grad_(True)
    h, _ = recurrence.linear_recurrence(xg, g)
    d, = torch.autograd.grad(h.sum(), xg, create_graph=True)
    with pytest.raises(RuntimeError):
        d.sum().backward()


@pytest.mark.parametrize("width,gates", [(96, 48), (96, 32), (99, 33), (99, 9), (102, 6), (130, 10), (128, 8), (143, 11), (66, 3),
                                         (96, 4), (50, 2), (58, 2), (200, 1), (63, 7), (18, 9), (260, 130)])
@pytest.mark.parametrize("dtype,gate_dtype", [(F32, F32), (BF16, BF16)])
def test_shared_gates_of_any_share(width, gates, dtype, gate_dtype):
    """Shares of 2 to 200 channels, with blocks that hold many gates, a few or a part of one."""
    x, gate = make(width + gates, (2, 150), width, gates, dtype, gate_dtype, False)
    run_and_check(x, gate, h0=state_of(1, 2, width))
    off = torch.tensor([0, 40, 41, 200, 290], dtype=torch.int64, device=DEV)
    run_and_check(x.reshape(300, width), gate.reshape(300, gates), h0=state_of(2, 4, width), offsets=off, reverse=True)


@pytest.mark.parametrize("width,gates", [(64, 64), (64, 16), (63, 63), (63, 9), (64, 1)])
def test_rows_that_start_anywhere(width, gates):
    """Tensors inside larger ones, at offsets of one element: no vector access, no tensor copy."""
    big = torch.empty(2, 70, width + 3, dtype=BF16, device=DEV)
    gbig = torch.empty(2, 70, gates + 5, dtype=F32, device=DEV)
    x, gate = make(5, (2, 70), width, gates, BF16, F32, False)
    big[..., 1:1 + width], gbig[..., 3:3 + gates] = x, gate
    xv, gv = big[..., 1:1 + width], gbig[..., 3:3 + gates]
    want, ws = run_and_check(x, gate)
    h, st = recurrence.linear_recurrence(xv, gv)
    assert torch.equal(h, want) and torch.equal(st, ws)
    # one row a sequence
    h0 = state_of(3, 2, width)
    one, s1 = recurrence.linear_recurrence(x[:, :1], gate[:, :1], h0=h0)
    two, s2 = recurrence.linear_recurrence(xv[:, :1], gv[:, :1], h0=h0)
    assert torch.equal(one, two) and torch.equal(s1, s2)
    ref = R.reference(dbl(x[:, 0]), dbl(gate[:, 0]), [(0, 1), (1, 2)], dbl(h0))
    R.check(one, ref["h"], BF16, "h")
    R.check(s1, ref["state"], F32, "state")


@pytest.mark.parametrize("width", [5, 40, 64])
def test_state_in_place_with_one_row(width):
    """state_out may be h0: padded and packed rows of one step too."""
    x, gate = make(6, (7, 1), width, width, F32, F32, False)
    h0 = state_of(4, 7, width)
    for kw in (dict(lengths=torch.tensor([1, 0, 1, 1, 0, 1, 1], device=DEV)), {}):
        want, ws = recurrence.linear_recurrence(x, gate, h0=h0, **kw)
        state = h0.clone()
        got, _ = recurrence.linear_recurrence(x, gate, h0=state, state_out=state, **kw)
        assert torch.equal(got, want) and torch.equal(state, ws)
    off = torch.tensor([0, 0, 1, 1], device=DEV)
    want, ws = recurrence.linear_recurrence(x[0], gate[0], h0=h0[:3], offsets=off)
    state = h0[:3].clone()
    got, _ = recurrence.linear_recurrence(x[0], gate[0], h0=state, offsets=off, state_out=state)
    assert torch.equal(got, want) and torch.equal(state, ws) and torch.equal(ws[0], h0[0])


@pytest.mark.parametrize("width", [64, 33, 1])
def test_beyond_32_bits(width):
    """A sequence behind element 2^31 of every tensor, in the streaming, the fallback and the narrow kernels."""
    tail = 5000
    rows = (1 << 31) // width + 3 * tail
    x = torch.zeros(rows, width, dtype=BF16, device=DEV)
    gate = torch.full((rows, width), 0.5, dtype=BF16, device=DEV)
    xs, gs = make(3, (tail,), width, width, BF16, BF16, False)
    x[-tail:], gate[-tail:] = xs, gs
    dh = torch.zeros_like(x)
    dh[-tail:] = torch.randn(tail, width, device=DEV).to(BF16)
    off = torch.tensor([0, rows - tail, rows], device=DEV)
    x.requires_grad_(True), gate.requires_grad_(True)
    h, state = recurrence.linear_recurrence(x, gate, offsets=off)
    dx, dgate = torch.autograd.grad(h, [x, gate], dh)
    want = R.reference(dbl(xs), dbl(gs), [(0, tail)], dh=dbl(dh[-tail:]))
    R.check(h[-tail:], want["h"], BF16, "h")
    R.check(state[1:], want["state"], F32, "state")
    R.check(dx[-tail:], want["dx"], BF16, "dx")
    R.check(dgate[-tail:], want["dgate"], BF16, "dgate")
    for t in (h, dx, dgate):
        assert not t[:-tail].any()


@pytest.mark.parametrize("width", [64, 200, 320, 512, 520, 640])
@pytest.mark.parametrize("time", [300, 6000])
@pytest.mark.parametrize("gate_dtype", [F32, BF16])
def test_the_same_bits_whatever_the_alignment(width, time, gate_dtype):
    x, gate = slow(width, (2, time), width, width, BF16, gate_dtype)
    dh = torch.randn(2, time, width, device=DEV).to(BF16)
    h0 = state_of(6, 2, width)

    def both(x, gate):
        leaves = [x.detach().requires_grad_(True), gate.detach().requires_grad_(True)]
        h, s = recurrence.linear_recurrence(*leaves, h0=h0, gate_kind="log")
        return [h, s] + list(torch.autograd.grad(h, leaves, dh))

    shifted = []
    for t in (x, gate):
        room = torch.empty(2, time, width + 3, dtype=t.dtype, device=DEV)
        room[..., 1:1 + width] = t
        shifted.append(room[..., 1:1 + width])
    for a, b in zip(both(x, gate), both(*shifted)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("width,gates,dtype", [(64, 64, F32), (256, 256, F32), (256, 2, BF16), (700, 700, F32), (520, 4, BF16)])
@pytest.mark.parametrize("reverse", [False, True])
def test_states_behind_tiles_that_wait_for_nothing(width, gates, dtype, reverse):
    """Tiles of many short sequences with states (slow to look at), then one that starts a sequence in the last tile of
    eight, so that the state behind the eight depends on that tile's own rows alone; and padding.  Every time the bits of
    the kernels without roles."""
    rng = np.random.default_rng(width)
    lens = []
    for _ in range(40):                       # 512 rows: short ones up to row 448 or so, one over the end of the eight tiles
        room = 448 - (64 if lens else 0)
        while room > 0:
            lens.append(int(min(room, rng.integers(1, 6))))
            room -= lens[-1]
        lens.append(128)
    lens += [0, 3000, 5]
    off = torch.tensor(np.cumsum([0] + lens), dtype=torch.int64, device=DEV)
    rows = int(off[-1]) + 1500                # rows of no sequence behind the last
    x, gate = slow(width, (rows,), width, gates, dtype, F32)
    h0 = state_of(5, len(lens), width)
    dh = torch.randn(rows, width, device=DEV).to(dtype)
    dst = state_of(6, len(lens), width)

    def once(x, gate):
        leaves = [t.detach().requires_grad_(True) for t in (x, gate, h0)]
        h, s = recurrence.linear_recurrence(*leaves[:2], h0=leaves[2], offsets=off, reverse=reverse, gate_kind="log")
        return [h, s, *torch.autograd.grad([h, s], leaves, [dh, dst])]

    room = torch.empty(rows, width + 1, dtype=dtype, device=DEV)
    room[:, 1:] = x
    groom = torch.empty(rows, gates + 1, dtype=F32, device=DEV)
    groom[:, 1:] = gate
    want = once(room[:, 1:], groom[:, 1:])
    for _ in range(20):
        got = once(x, gate)
        for i, (a, b) in enumerate(zip(got, want)):
            if i != 3 or gates == width:      # the sums of shared gates depend on alignment
                assert torch.equal(a, b), i
    if not reverse:
        run_and_check(x, gate, h0, offsets=off, log=True)


class polls:
    """Waits inside the launches of the block give up after `n` polls."""

    def __init__(self, n):
        self.n = n

    def __enter__(self):
        self.before = N.lib.gearb_recurrence_wait_limit(self.n)

    def __exit__(self, *exc):
        torch.cuda.synchronize()
        N.lib.gearb_recurrence_wait_limit(self.before)


# streaming (a gate per channel, shared; long sections and short ones), a CTA per tile, few channels
WAITS = [(64, 64, F32, False), (1024, 1024, BF16, False), (256, 4, BF16, False), (80, 1, F32, False), (63, 63, F32, True),
         (130, 10, BF16, True), (1, 1, F32, True), (6, 2, F32, True)]


@pytest.mark.parametrize("width,gates,dtype,polled", WAITS)
@pytest.mark.parametrize("reverse", [False, True])
def test_a_wait_that_runs_out(width, gates, dtype, polled, reverse):
    """With no polls at all: the status says so, and what was not worked out is NaN, nothing else; `polled`: kernels that
    only wait for words of other tiles, and may find them there at the first look."""
    rows = 60000 if width <= 16 else 9000
    lens = [700, 0, rows - 1500, 1, 99]
    off = torch.tensor(np.cumsum([0] + lens), dtype=torch.int64, device=DEV)
    owned = int(off[-1])
    x, gate = slow(width, (rows,), width, gates, dtype, F32)
    h0 = state_of(1, len(lens), width)
    dh = torch.randn(rows, width, device=DEV).to(dtype)
    dst = state_of(2, len(lens), width)

    def forward(status=None):
        leaves = [t.detach().requires_grad_(True) for t in (x, gate, h0)]
        h, s = recurrence.linear_recurrence(*leaves[:2], h0=leaves[2], offsets=off, reverse=reverse, gate_kind="log",
                                            status=status)
        return leaves, h, s

    def backward(leaves, h, s):
        return torch.autograd.grad([h, s], leaves, [dh, dst], retain_graph=True)

    leaves, h, s = forward()
    want = [h, s, *backward(leaves, h, s)]
    for n in (0, 1, 3):
        status = torch.zeros(N.STATUS_WORDS, dtype=torch.int32, device=DEV)
        leaves, h, s = forward(status)
        with polls(n):
            _, bad_h, bad_s = forward(status)
        gave_up = bool(status[0].item() & N.ST_SCAN_ABORTED)
        status.zero_()
        with polls(n):
            grads = backward(leaves, h, s)
        gave_up_back = bool(status[0].item() & N.ST_SCAN_ABORTED)
        got = [bad_h, bad_s, *grads]
        for i, (a, b) in enumerate(zip(got, want)):
            lost = torch.isnan(a)
            assert torch.equal(torch.where(lost, b, a), b), (n, i)
            assert not lost.any() or (gave_up if i < 2 else gave_up_back), (n, i)
        assert not any(torch.isnan(t[owned:]).any() for t in (bad_h, grads[0], grads[1]))
        assert torch.equal(bad_s[1], h0[1]) and torch.equal(grads[2][1], dst[1])
        if n == 0 and not polled:
            assert gave_up and gave_up_back
            assert torch.isnan(bad_h[:owned]).all() and torch.isnan(grads[0][:owned]).all() and torch.isnan(grads[1][:owned]).all()
            assert torch.isnan(bad_s[[0, 2, 3, 4]]).all() and torch.isnan(grads[2][[0, 2, 3, 4]]).all()
    # and the next launches are as ever
    leaves, h, s = forward()
    for a, b in zip([h, s, *backward(leaves, h, s)], want):
        assert torch.equal(a, b)


def test_transforms_that_the_launch_cannot_follow_are_refused():
    import torch.autograd.forward_ad as fwd
    x, gate = make(1, (2, 30), 8, 8, F32, F32, False)
    x.requires_grad_(True)
    h, _ = recurrence.linear_recurrence(x, gate)
    with fwd.dual_level():
        with pytest.raises(core.GearError, match="forward-mode"):
            recurrence.linear_recurrence(x, fwd.make_dual(gate, gate))
        with pytest.raises(core.GearError, match="forward-mode"):         # of a gradient
            torch.autograd.grad(h, x, fwd.make_dual(torch.ones_like(h), torch.ones_like(h)), retain_graph=True)
        plain, = torch.autograd.grad(h, x, torch.ones_like(h))
        assert torch.isfinite(plain).all()
    x = x.detach()
    for f in (lambda: torch.func.vmap(lambda t: recurrence.linear_recurrence(t, gate)[0])(torch.stack([x, x])),
              lambda: torch.func.grad(lambda t: recurrence.linear_recurrence(t, gate)[0].sum())(x),
              lambda: torch.func.jvp(lambda t: recurrence.linear_recurrence(t, gate)[0], (x,), (x,))):
        with pytest.raises(RuntimeError):
            f()


@pytest.mark.parametrize("width,gates", [(1, 1), (12, 3), (64, 64), (64, 1), (45, 45)])
def test_gradients_of_some_inputs_and_of_the_state_alone(width, gates):
    x, gate = make(21, (3, 200), width, gates, F32, F32, True)
    h0 = state_of(22, 3, width)
    rng = np.random.default_rng(5)
    dst = torch.from_numpy(rng.standard_normal((3, width)).astype(np.float32)).to(DEV)
    flat = lambda t, c: dbl(t).reshape(600, c)
    want = R.reference(flat(x, width), flat(gate, gates), R.spans(600, 200, None, None), dbl(h0), False, True,
                       np.zeros((600, width)), dbl(dst))
    for wanted in ((1, 1, 1), (1, 0, 0), (0, 1, 0), (0, 0, 1)):
        leaves = [t.clone().requires_grad_(bool(w)) for t, w in zip((x, gate, h0), wanted)]
        _, s = recurrence.linear_recurrence(leaves[0], leaves[1], h0=leaves[2], gate_kind="log")
        s.backward(dst)
        for t, w, key in zip(leaves, wanted, ("dx", "dgate", "dh0")):
            assert (t.grad is not None) == bool(w)
            if w:
                R.check(t.grad, want[key], F32, key)


@pytest.mark.parametrize("width,gates", [(64, 64), (96, 2), (160, 160), (8, 8), (43, 43)])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("step", [8, 16, 0])
def test_rows_that_overlap(width, gates, dtype, step):
    """Windows over one line of values: rows fewer elements apart than they are wide (or all the same one)."""
    rows = 300
    line, gline = make(3, (rows * max(step, 1) + width,), 1, 1, dtype, F32, False)
    x = line.reshape(-1).as_strided((rows, width), (step, 1))
    gate = gline.reshape(-1).as_strided((rows, gates), (step, 1))
    dh = torch.randn(rows * max(step, 1) + width, device=DEV).to(dtype).as_strided((rows, width), (step, 1))
    off = torch.tensor([0, 100, 101, 290], device=DEV)

    def once(x, gate, dh, **kw):
        leaves = [x.detach(), gate.detach()]
        for t in leaves:
            t.requires_grad_(True)
        h, s = recurrence.linear_recurrence(*leaves, **kw)
        return [h, s, *torch.autograd.grad(h, leaves, dh)]

    for a, b in zip(once(x, gate, dh, offsets=off), once(x.contiguous(), gate.contiguous(), dh.contiguous(), offsets=off)):
        assert torch.equal(a, b)
    batch = lambda t: t.as_strided((3, 100, t.shape[1]), (100 * step, step, 1))
    for a, b in zip(once(*map(batch, (x, gate, dh))), once(*(batch(t).contiguous() for t in (x, gate, dh)))):
        assert torch.equal(a, b)


@pytest.mark.parametrize("width,gates", [(64, 64), (66, 66), (256, 4), (96, 48), (1, 1), (6, 2)])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("with_state", [False, True])
def test_the_sign_of_zero(width, gates, dtype, with_state):
    """Without h0 a first row is x, to the sign of its zero; the same bits whatever the alignment, gradients too."""
    lens = [5, 1, 64, 130, 0, 60, 40]
    off = torch.tensor(np.cumsum([0] + lens), dtype=torch.int64, device=DEV)
    rows = int(off[-1])
    x, gate = make(31, (rows,), width, gates, dtype, F32, False)
    x[torch.rand(rows, width, device=DEV, generator=torch.Generator(DEV).manual_seed(3)) < 0.5] = -0.0
    first = off[:-1][torch.tensor(lens, device=DEV) > 0]
    dh = torch.randn(rows, width, device=DEV).to(dtype)
    bits = lambda t: t.view(torch.int32 if t.dtype is F32 else torch.int16)
    room, groom = torch.empty(rows, width + 1, dtype=dtype, device=DEV), torch.empty(rows, gates + 1, device=DEV)
    room[:, 1:], groom[:, 1:] = x, gate

    def once(x, gate):
        leaves = [x.detach().requires_grad_(True), gate.detach().requires_grad_(True)]
        h, s = recurrence.linear_recurrence(*leaves, offsets=off, return_state=with_state)
        return [h, *torch.autograd.grad(h, leaves, dh)] + ([s] if with_state else [])

    got, other = once(x, gate), once(room[:, 1:], groom[:, 1:])
    assert torch.equal(bits(got[0])[first], bits(x)[first])
    for i, (a, b) in enumerate(zip(got, other)):
        if i != 2 or gates == width:              # the sums of shared gates depend on alignment
            assert torch.equal(bits(a), bits(b)), i


@pytest.mark.parametrize("width", [1, 2, 3, 5, 8, 16, 17, 64, 512])
@pytest.mark.parametrize("reverse", [False, True])
def test_gates_above_one_up_to_the_stated_products(width, reverse):
    """Gates whose products over the stated number of rows just stay in range, over four times as many rows: where there is
    nothing to multiply, zeros and finite gradients (a product beyond the range would make them NaN)."""
    reach = 32768 // width if width <= 16 else 512
    rows, tail = 4 * reach + 77, 60
    a = float(np.float32(np.exp(86.0 / reach)))           # float32 ends at e^88.7
    x = torch.zeros(1, rows, width, device=DEV)
    gate = torch.full((1, rows, width), a, device=DEV)
    dh = torch.zeros_like(x)
    last, first = (slice(0, tail), slice(rows - tail, rows)) if reverse else (slice(rows - tail, rows), slice(0, tail))
    rng = np.random.default_rng(width)
    x[0, last] = torch.from_numpy(rng.standard_normal((tail, width)).astype(np.float32)).to(DEV)
    dh[0, first] = torch.from_numpy(rng.standard_normal((tail, width)).astype(np.float32)).to(DEV)
    for h0 in (None, torch.zeros(1, width, device=DEV)):
        leaves = [x.clone().requires_grad_(True), gate.clone().requires_grad_(True)]
        h, s = recurrence.linear_recurrence(*leaves, h0=h0, reverse=reverse)
        dx, dg = torch.autograd.grad(h, leaves, dh)
        want = R.reference(dbl(x[0, last]), dbl(gate[0, last]), [(0, tail)], np.zeros((1, width)), reverse)
        R.check(h[0, last], want["h"], F32, "h")
        R.check(s, want["state"], F32, "state")
        h[0, last] = 0
        assert (h == 0).all()
        back = R.reference(np.zeros((tail, width)), dbl(gate[0, first]), [(0, tail)], np.zeros((1, width)), reverse,
                           dh=dbl(dh[0, first]))
        R.check(dx[0, first], back["dx"], F32, "dx")
        dx[0, first] = 0
        assert (dx == 0).all() and (dg == 0).all()
