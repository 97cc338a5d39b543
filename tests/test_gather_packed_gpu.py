"""Packed and paged gathers against a plain restatement on the host: every byte, those left alone too."""
import numpy as np
import pytest
import torch

from gear_b200 import _native as N
from gear_b200 import core, layout, recurrence

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def make_table(rows, T, cap, residency=N.RES_HBM, seed=1):
    t = core.TrajectoryTable(rows, T, cap, residency=residency)
    t.connect()
    img = np.random.default_rng(seed).integers(0, 256, t.nbytes, dtype=np.uint8)
    t.write(0, img)
    return t, img


def requests(rng, n, T, cap):
    idx = rng.integers(0, cap, n).astype(np.int64)
    ts = rng.integers(0, T, n).astype(np.int64)
    ln = rng.integers(0, T + 1, n).astype(np.int64)
    return idx, ts, ln


def clip(t, pat, idx, ts, ln):
    start = np.maximum(ts + pat.offset, 0)
    n = np.maximum(np.minimum(start + pat.length, np.minimum(ln, t.trajectory_length)) - start, 0)
    return start, np.where((idx >= 0) & (idx < t.capacity), n, 0)


def plain(t, img, col, start, count, idx, offsets, dst, table=None, page=0, past=None):
    dst = dst.copy()
    row = t.row_bytes[col]
    for r in range(len(idx)):
        n = min(count[r], max(0, offsets[r + 1] - offsets[r]))
        base = idx[r] * t.trajectory_stride + t.column_offset(col) + start[r] * row
        for k in range(n):
            if table is None:
                slot = offsets[r] + k
            else:
                pos = (0 if past is None else past[r]) + k
                b = pos // page
                page_id = table[r, b] if b < table.shape[1] else -1
                if page_id < 0:
                    continue
                slot = int(page_id) * page + pos % page
            if 0 <= slot < len(dst):
                dst[slot] = img[base + k * row: base + (k + 1) * row]
    return dst


ROWS = [[156, 24, 4, 4, 1], [68, 24, 4, 1], [4096, 4, 4], [3, 7, 13, 1, 2, 5], [16, 32, 48], [2049, 2047, 15, 17], [8]]


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("page", [0, 1, 4, 16, 24])
@pytest.mark.parametrize("offset", [0, -5, 3])
def test_every_byte(rows, page, offset):
    T, cap = 90, 13
    t, img = make_table(rows, T, cap)
    h = core.StorageHandler(t)
    cols = list(range(len(rows)))
    rng = np.random.default_rng(len(rows) * 100 + page)
    for length, n in ((1, 5), (17, 40), (90, 33)):
        pat = core.SubscribePattern(offset, length, int(rng.integers(0, 3)))
        h.set(cols, [pat] * len(cols))
        idx, ts, ln = requests(rng, n, T, cap)
        start, count = clip(t, pat, idx, ts, ln)
        dev = [torch.from_numpy(a).to(DEV) for a in (idx, ts, ln)]
        lens = h.segment_lengths(*dev, cols[0])
        assert np.array_equal(lens.cpu().numpy(), count)
        offsets = np.concatenate([[0], np.cumsum(count)])
        doff = torch.from_numpy(offsets).to(DEV)
        table = past = None
        total = int(offsets[-1])
        if page:
            past = rng.integers(0, 20, n) if n % 2 else None
            m = -(-(length + 20) // page)
            order = rng.permutation(n * m + 2).astype(np.int32)
            table = order[: n * m].reshape(n, m)
            total = (n * m + 2) * page
        dsts = [np.full((total + 2, r), 0xA5, np.uint8) for r in rows]
        ddst = [torch.from_numpy(d).to(DEV) for d in dsts]
        h.gather_packed(cols, *dev, doff, ddst, block_table=None if table is None else torch.from_numpy(table).to(DEV),
                        page=page, past=None if past is None else torch.from_numpy(past).to(DEV))
        torch.cuda.synchronize()
        for c in cols:
            want = plain(t, img, c, start, count, idx, offsets, dsts[c], table, page, past)
            assert np.array_equal(ddst[c].cpu().numpy(), want), (c, length)
        assert h.status() & ~N.ST_LEN_CLAMPED == 0


@pytest.mark.parametrize("residency", [N.RES_HOST, N.RES_HOST | N.RES_HBM])
def test_residencies_and_unaligned_destinations(residency):
    rows, T, cap = [156, 24, 4, 1, 16], 50, 7
    t, img = make_table(rows, T, cap, residency)
    h = core.StorageHandler(t)
    pat = core.SubscribePattern(0, 30)
    cols = list(range(5))
    h.set(cols, [pat] * 5)
    rng = np.random.default_rng(3)
    idx, ts, ln = requests(rng, 60, T, cap)
    start, count = clip(t, pat, idx, ts, ln)
    offsets = np.concatenate([[0], np.cumsum(count)])
    dev = [torch.from_numpy(a).to(DEV) for a in (idx, ts, ln, offsets)]
    for shift in (0, 1, 4, 8):
        bufs = [torch.zeros(int(offsets[-1]) * r + 16, dtype=torch.uint8, device=DEV) for r in rows]
        dsts = [b[shift: shift + int(offsets[-1]) * r].view(-1, r) for b, r in zip(bufs, rows)]
        h.gather_packed(cols, *dev[:3], dev[3], dsts)
        for c in cols:
            want = plain(t, img, c, start, count, idx, offsets, np.zeros((int(offsets[-1]), rows[c]), np.uint8))
            assert np.array_equal(dsts[c].cpu().numpy(), want), c


def test_bad_requests_and_pages_are_skipped():
    rows, T, cap = [24, 5, 16], 40, 5
    t, img = make_table(rows, T, cap)
    h = core.StorageHandler(t)
    pat = core.SubscribePattern(0, 10)
    h.set([0, 1, 2], [pat] * 3)
    big = 1 << 62
    idx = np.array([0, -1, 5, 2, 3, 1], np.int64)
    ts = np.array([0, 0, 0, 35, 3, 1], np.int64)
    ln = np.array([40, 40, 40, 40, 100, 40], np.int64)
    start, count = clip(t, pat, idx, ts, ln)
    dev = [torch.from_numpy(a).to(DEV) for a in (idx, ts, ln)]
    assert h.segment_lengths(*dev, 0).tolist() == [10, 0, 0, 5, 10, 10]
    for offsets in ([0, 10, 20, 30, 33, 43, 53], [0, 10, 20, 30, -7, 33, 500], [40, 50, 60, big, -big, big, big]):
        offsets = np.array(offsets, np.int64)
        dsts = [np.full((45, r), 9, np.uint8) for r in rows]
        dd = [torch.from_numpy(d).to(DEV) for d in dsts]
        h.gather_packed([0, 1, 2], *dev, torch.from_numpy(offsets).to(DEV), dd)
        for c in range(3):
            want = dsts[c]
            for r in range(6):                       # a negative first row means the request is skipped
                if offsets[r] >= 0:
                    one = np.array([offsets[r], offsets[r + 1]])
                    want = plain(t, img, c, start[r:], count[r:r + 1], idx[r:r + 1], one, want)
            assert bool(np.array_equal(dd[c].cpu().numpy(), want)), (c, offsets)
        assert h.status() & N.ST_BAD_REQUEST
    offsets = np.arange(7, dtype=np.int64) * 10
    table = np.array([[0, 1, 2], [3, 4, 5], [6, 7, 8], [-1, 1 << 30, 9], [-5, 10, 11], [12, 2147483647, 3]], np.int32)
    past = np.array([0, 0, 0, 2, 1, 3], np.int64)
    for p in (past, past + np.array([0, 0, 0, 0, big, 0]), past - np.array([5, 0, 0, 0, 0, 0])):
        dsts = [np.full((60, r), 9, np.uint8) for r in rows]
        dd = [torch.from_numpy(d).to(DEV) for d in dsts]
        h.gather_packed([0, 1, 2], *dev, torch.from_numpy(offsets).to(DEV), dd,
                        block_table=torch.from_numpy(table).to(DEV), page=4, past=torch.from_numpy(p).to(DEV))
        ok = (p >= 0) & (p <= 12)
        for c in range(3):
            want = dsts[c]
            for r in range(6):
                if ok[r]:
                    want = plain(t, img, c, start[r:], count[r:r + 1], idx[r:r + 1], offsets[r:r + 2], want,
                                 table[r:r + 1], 4, p[r:r + 1])
            assert np.array_equal(dd[c].cpu().numpy(), want), c


def test_refusals():
    t, _ = make_table([24, 5], 40, 5)
    h = core.StorageHandler(t)
    i = torch.zeros(3, dtype=torch.int64, device=DEV)
    off = torch.zeros(4, dtype=torch.int64, device=DEV)
    d = [torch.zeros(10, 24, dtype=torch.uint8, device=DEV), torch.zeros(10, 5, dtype=torch.uint8, device=DEV)]
    bt = torch.zeros(3, 2, dtype=torch.int32, device=DEV)
    with pytest.raises(core.GearError, match="without setting its SubscribePattern"):
        h.gather_packed([0], i, i, i, off, d[:1])
    with pytest.raises(core.GearError, match="without setting its SubscribePattern"):
        h.segment_lengths(i, i, i, 0)
    h.set([0, 1], [core.SubscribePattern(0, 4), core.SubscribePattern(0, 5)])
    bad = [
        lambda: h.gather_packed([0, 1], i, i, i, off, d),                    # different patterns
        lambda: h.gather_packed([0], i, i, i, off[:3], d[:1]),
        lambda: h.gather_packed([0], i, i[:2], i, off, d[:1]),
        lambda: h.gather_packed([0], i, i, i, off, d),
        lambda: h.gather_packed([2], i, i, i, off, d[:1]),
        lambda: h.gather_packed([0], i, i, i, off, d[1:]),                   # rows of another size
        lambda: h.gather_packed([0], i.int(), i, i, off, d[:1]),
        lambda: h.gather_packed([0], i, i, i, off.int(), d[:1]),
        lambda: h.gather_packed([0], i, i, i, off, [d[0].cpu()]),
        lambda: h.gather_packed([0], i, i, i, off, [d[0][:, ::2]]),
        lambda: h.gather_packed([0], i, i, i, off, d[:1], block_table=bt, page=0),
        lambda: h.gather_packed([0], i, i, i, off, d[:1], block_table=bt.long(), page=4),
        lambda: h.gather_packed([0], i, i, i, off, d[:1], block_table=bt[:2], page=4),
        lambda: h.gather_packed([0], i, i, i, off, d[:1], block_table=bt, page=1 << 31),
        lambda: h.gather_packed([0], i, i, i, off, d[:1], past=i),
        lambda: h.gather_packed([0], i, i, i, off, d[:1], block_table=bt, page=4, past=i[:1]),
        lambda: h.segment_lengths(i, i, i[:2], 0),
        lambda: h.segment_lengths(i, i, i, 7),
    ]
    for k, f in enumerate(bad):
        with pytest.raises(core.GearError) as e:
            f()
        assert e.value.code == N.ERR_INVALID, k
    h.gather_packed([0], i[:0], i[:0], i[:0], off[:1], d[:1])
    h.gather_packed([0], i, i, i, off, [d[0][:0]])


def test_from_a_draw_to_advantages(O):
    """The set as it is used: draw segments, lay them out without padding, gather, returns with gradients; and the
    same batch in pages holds the same rows."""
    rows, T, cap, L, B = [12, 4, 4], 60, 50, 25, 200
    t, img = make_table(rows, T, cap)
    rewards = np.random.default_rng(0).standard_normal(cap * T).astype(np.float32).reshape(cap, T)
    for i in range(cap):
        t.write(i * t.trajectory_stride + t.column_offset(1), rewards[i])
    h = core.StorageHandler(t)
    h.set([0, 1, 2], [core.SubscribePattern(0, L)] * 3)
    prio = torch.from_numpy(O.synth_lognormal(2, 0, cap * T)).to(DEV)
    sampler = core.PrioritySampler(cap * T)
    sampler.scan(prio)
    flat = sampler.search(torch.from_numpy(O.synth_u01(3, 0, B)).to(DEV), scale=True)
    idx, ts, ln = core.decode(flat, T)
    n = h.segment_lengths(idx, ts, ln, 1)
    page, pool = 8, 900
    table = torch.full((B, -(-L // page)), -1, dtype=torch.int32, device=DEV)
    used = torch.zeros(1, dtype=torch.int64, device=DEV)
    lay = layout.paged_layout(n, page, table, used, free_pages=torch.randperm(pool, device=DEV).to(torch.int32),
                              max_tokens=B * L)
    total = int(lay.offsets[-1])
    assert total == int(n.sum()) and int(lay.used) == int(((n + page - 1) // page).sum())
    packed = torch.zeros(B * L, 1, device=DEV)
    h.gather_packed([1], idx, ts, ln, lay.offsets, [packed])
    paged = torch.zeros(pool * page, 1, device=DEV)
    h.gather_packed([1], idx, ts, ln, lay.offsets, [paged], block_table=lay.block_table, page=page)
    assert torch.equal(paged[lay.slot_map[:total]], packed[:total])
    assert (lay.slot_map[total:] == -1).all()
    decay = torch.full((B * L, 1), 0.97, device=DEV, requires_grad=True)
    ret, _ = recurrence.linear_recurrence(packed, decay, offsets=lay.offsets, reverse=True, return_state=False)
    d, = torch.autograd.grad(ret.sum(), decay)
    gi, gt, go = (v.cpu().numpy() for v in (idx, ts, lay.offsets))
    for r in range(0, B, 7):
        seg = rewards[gi[r], gt[r]: gt[r] + L].astype(np.float64)
        want, acc = np.zeros(len(seg)), 0.0
        for k in range(len(seg) - 1, -1, -1):
            acc = float(np.float32(0.97)) * acc + seg[k]
            want[k] = acc
        got = ret[go[r]: go[r + 1], 0].detach().cpu().numpy()
        # at most 25 roundings of values below 25 * 5
        assert len(got) == len(seg) and np.abs(got - want).max() <= 25 * 2.0 ** -24 * 125
        # d sum / d decay_k = (sum over j <= k of decay^(k-j)) * ret_(k+1)
        gk = np.array([sum(0.97 ** j for j in range(k + 1)) * (want[k + 1] if k + 1 < len(seg) else 0.0)
                       for k in range(len(seg))])
        assert np.abs(d[go[r]: go[r + 1], 0].cpu().numpy() - gk).max() <= 1e-5 * max(1.0, np.abs(gk).max())
    assert (ret[total:] == 0).all() and (d[total:] == 0).all()


def test_refuses_pages_beyond_the_argument():
    t, _ = make_table([8], 20, 4)
    h = core.StorageHandler(t)
    h.set([0], [core.SubscribePattern(0, 20, 0)])
    z = torch.zeros(2, dtype=torch.int64, device=DEV)
    for page in (1 << 70, (1 << 64) + 16, -1):
        with pytest.raises(core.GearError) as e:
            h.gather_packed([0], z, z, z + 20, torch.tensor([0, 20, 40], device=DEV), [torch.zeros(64, 8, dtype=torch.uint8, device=DEV)],
                            block_table=torch.zeros(2, 2, dtype=torch.int32, device=DEV), page=page)
        assert e.value.code == N.ERR_INVALID


def test_destinations_beyond_32_bits():
    """Rows past 2^31 of a packed destination, pages past 2^31 rows of a pool; the same trajectory twice."""
    rows, T, cap = [4, 1], 40, 3
    t, img = make_table(rows, T, cap)
    h = core.StorageHandler(t)
    h.set([0, 1], [core.SubscribePattern(0, T, 0)] * 2)
    big = (1 << 31) + 200
    dsts = [torch.zeros(big, r, dtype=torch.uint8, device=DEV) for r in rows]
    idx = torch.tensor([2, 2], dtype=torch.int64, device=DEV)
    z = torch.zeros(2, dtype=torch.int64, device=DEV)
    off = torch.tensor([big - 80, big - 40, big], device=DEV)
    h.gather_packed([0, 1], idx, z, z + T, off, dsts)
    for c in (0, 1):
        base = 2 * t.trajectory_stride + t.column_offset(c)
        want = torch.from_numpy(img[base: base + T * rows[c]].reshape(T, rows[c]).copy()).to(DEV)
        assert torch.equal(dsts[c][big - 80: big - 40], want) and torch.equal(dsts[c][big - 40:], want)
        assert int(dsts[c][: big - 80].max()) == 0
        dsts[c].zero_()
    last = big // 8 - 5
    table = torch.arange(last, last - 10, -1, dtype=torch.int32, device=DEV).reshape(2, 5)
    h.gather_packed([0, 1], idx, z, z + T, off, dsts, block_table=table, page=8)
    for c in (0, 1):
        base = 2 * t.trajectory_stride + t.column_offset(c)
        want = torch.from_numpy(img[base: base + T * rows[c]].reshape(T, rows[c]).copy()).to(DEV)
        pages = dsts[c][: big // 8 * 8].reshape(big // 8, 8, rows[c])
        for r in range(2):
            assert torch.equal(pages[table[r].long()].reshape(T, rows[c]), want)
        assert int(dsts[c][: (last - 9) * 8].max()) == 0
    assert h.status() == 0


def test_layout_and_gather_captured_once_follow_their_inputs():
    """One graph from lengths to rows, replayed with other requests, beside the same graph on a second stream."""
    rows, T, cap, n, page = [12, 4], 60, 9, 50, 8
    t, img = make_table(rows, T, cap)
    rng = np.random.default_rng(4)
    blocks = -(-T // page)
    graphs = []
    for _ in range(2):
        h = core.StorageHandler(t)
        h.set([0, 1], [core.SubscribePattern(-3, T, 0)] * 2)
        inp = [torch.zeros(n, dtype=torch.int64, device=DEV) for _ in range(3)]
        used = torch.zeros(1, dtype=torch.int64, device=DEV)
        table = torch.full((n, blocks), -1, dtype=torch.int32, device=DEV)
        pools = [torch.zeros(n * blocks * page, r, dtype=torch.uint8, device=DEV) for r in rows]

        def step():
            lens = h.segment_lengths(*inp, 0)
            lay = layout.paged_layout(lens, page, table, used, num_pages=n * blocks, max_tokens=64)
            h.gather_packed([0, 1], *inp, lay.offsets, pools, block_table=table, page=page)
            return lens, lay
        step()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = step()
        graphs.append((g, inp, table, pools, res, torch.cuda.Stream(), h))
    for _ in range(3):
        wants = []
        for g, inp, table, pools, res, st, h in graphs:
            req = requests(rng, n, T, cap)
            for a, b in zip(inp, req):
                a.copy_(torch.from_numpy(b))
            for p in pools:
                p.zero_()
            start, count = clip(t, core.SubscribePattern(-3, T, 0), *req)
            wants.append((req, start, count))
        torch.cuda.synchronize()
        for g, _i, _t, _p, _r, st, _h in graphs:
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for (g, inp, table, pools, (lens, lay), st, h), (req, start, count) in zip(graphs, wants):
            offsets = np.concatenate([[0], np.cumsum(count)])
            assert np.array_equal(lens.cpu().numpy(), count) and np.array_equal(lay.offsets.cpu().numpy(), offsets)
            tab = table.cpu().numpy()
            for c in (0, 1):
                want = plain(t, img, c, start, count, req[0], offsets, np.zeros((n * blocks * page, rows[c]), np.uint8), tab, page)
                assert np.array_equal(pools[c].cpu().numpy(), want)


@pytest.mark.parametrize("page", [0, 8])
def test_offsets_that_fall_by_more_than_63_bits(page):
    """A request whose end lies in front of its start has no rows, however far in front."""
    rows, T, cap = [24, 5], 40, 5
    t, img = make_table(rows, T, cap)
    h = core.StorageHandler(t)
    h.set([0, 1], [core.SubscribePattern(0, 20)] * 2)
    idx, ts, ln = (np.full(3, v, np.int64) for v in (2, 3, 40))
    start, count = clip(t, core.SubscribePattern(0, 20), idx, ts, ln)
    for end in (-(1 << 63), -(1 << 63) + 5, -1, 0, 10):
        offsets = [0, 10, end, 30]
        table = np.arange(9, dtype=np.int32).reshape(3, 3) if page else None
        dsts = [np.full((80, r), 0xA5, np.uint8) for r in rows]
        ddst = [torch.from_numpy(d).to(DEV) for d in dsts]
        h.gather_packed([0, 1], *(torch.from_numpy(a).to(DEV) for a in (idx, ts, ln)), torch.tensor(offsets, device=DEV), ddst,
                        block_table=None if table is None else torch.from_numpy(table).to(DEV), page=page)
        torch.cuda.synchronize()
        # request 2 begins where `end` says: in front of row 0 it is refused as a whole
        own = [min(int(count[r]), max(0, offsets[r + 1] - offsets[r])) if offsets[r] >= 0 else 0 for r in range(3)]
        for c in (0, 1):
            want = plain(t, img, c, start, own, idx, [0, 10, max(end, 0), 30], dsts[c], table, page)
            if end < 10:                                  # `plain` takes what the offsets leave: nothing of request 1
                assert own[1] == 0
            assert np.array_equal(ddst[c].cpu().numpy(), want), (c, end)


@pytest.mark.parametrize("residency", [N.RES_HOST, N.RES_HOST | N.RES_HBM])
@pytest.mark.parametrize("page", [1, 8, 100])
def test_pages_filled_from_the_host(residency, page):
    rows, T, cap = [156, 24, 4, 1, 16], 50, 7
    t, img = make_table(rows, T, cap, residency)
    h = core.StorageHandler(t)
    pat = core.SubscribePattern(0, 30)
    cols = list(range(5))
    h.set(cols, [pat] * 5)
    rng = np.random.default_rng(3)
    idx, ts, ln = requests(rng, 60, T, cap)
    start, count = clip(t, pat, idx, ts, ln)
    offsets = np.concatenate([[0], np.cumsum(count)])
    past = rng.integers(0, 20, 60)
    m = -(-50 // page)
    table = rng.permutation(60 * m).astype(np.int32).reshape(60, m)
    dev = [torch.from_numpy(a).to(DEV) for a in (idx, ts, ln, offsets)]
    dsts = [np.full((60 * m * page, r), 0x5A, np.uint8) for r in rows]
    ddst = [torch.from_numpy(d).to(DEV) for d in dsts]
    h.gather_packed(cols, *dev[:3], dev[3], ddst, block_table=torch.from_numpy(table).to(DEV), page=page,
                    past=torch.from_numpy(past).to(DEV))
    for c in cols:
        want = plain(t, img, c, start, count, idx, offsets, dsts[c], table, page, past)
        assert np.array_equal(ddst[c].cpu().numpy(), want), c
