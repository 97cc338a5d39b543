"""Offsets, block tables and slot maps against a plain restatement; everything is whole numbers and must be equal."""
import numpy as np
import pytest
import torch

from gear_b200 import _native as N
from gear_b200 import core, layout

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def plain(lengths, past, page, table, used, free, num_pages, max_tokens):
    """(offsets, table, slots, used, flags)"""
    table, m = table.copy(), table.shape[1]
    offsets, slots, flags = [0], [], 0
    k = max(int(used), 0)
    for r, n in enumerate(lengths):
        room = m * page
        p = 0 if past is None else int(past[r])
        if p < 0 or p > room:
            p, flags = min(max(p, 0), room), flags | N.ST_LEN_CLAMPED
        n = int(n)
        if n < 0 or n > room - p:
            n, flags = min(max(n, 0), room - p), flags | N.ST_LEN_CLAMPED
        offsets.append(offsets[-1] + n)
        for b in range(-(-p // page), -(-(p + n) // page)):
            ok = k < num_pages
            flags |= 0 if ok else N.ST_NO_PAGE
            table[r, b] = (int(free[k]) if free is not None else k) if ok else -1
            k += 1
        for t in range(p, p + n):
            b = table[r, t // page]
            slots.append(int(b) * page + t % page if b >= 0 else -1)
    slots = (slots + [-1] * max_tokens)[:max_tokens]
    return np.array(offsets), table, np.array(slots, np.int64), min(k, max(num_pages, 0)), flags


def check(lengths, page, max_blocks, past=None, free=None, num_pages=None, used=0, max_tokens=None, seed=0, **kw):
    lengths = np.asarray(lengths, np.int64)
    past = None if past is None else np.asarray(past, np.int64)
    rng = np.random.default_rng(seed)
    table = rng.integers(0, 1000, (len(lengths), max_blocks)).astype(np.int32)   # what must be left alone shows
    pages = num_pages if num_pages is not None else len(free)
    mt = int(np.clip(lengths, 0, None).sum()) + 5 if max_tokens is None else max_tokens
    mt = min(mt, 1 << 22)
    want = plain(lengths, past, page, table, used, free, pages, mt)
    dev = lambda a: None if a is None else torch.from_numpy(np.ascontiguousarray(a)).to(DEV)
    status = torch.zeros(4, dtype=torch.int32, device=DEV)
    dt = dev(table)
    lay = layout.paged_layout(dev(lengths), page, dt, torch.tensor([used], device=DEV), free_pages=dev(free),
                              num_pages=num_pages, past=dev(past), max_tokens=mt, status=status, **kw)
    assert np.array_equal(lay.offsets.cpu().numpy(), want[0])
    assert lay.block_table is dt and np.array_equal(dt.cpu().numpy(), want[1])
    if mt:
        assert np.array_equal(lay.slot_map.cpu().numpy(), want[2])
    else:
        assert lay.slot_map is None
    assert int(lay.used) == want[3]
    assert int(status[0]) == want[4], (int(status[0]), want[4])
    return lay


@pytest.mark.parametrize("requests", [0, 1, 2, 31, 32, 33, 255, 1023, 1024, 1025, 2500, 9000])
@pytest.mark.parametrize("page", [1, 16, 48])
def test_fresh_batches(requests, page):
    rng = np.random.default_rng(requests + page)
    lengths = rng.integers(0, 40, requests)
    free = rng.permutation(requests * 41 + 3).astype(np.int32)
    check(lengths, page, -(-40 // page), free=free, seed=requests)


@pytest.mark.parametrize("requests,page", [(1, 1), (5, 16), (300, 16), (2100, 7)])
@pytest.mark.parametrize("one", [True, False])
def test_growing_requests(requests, page, one):
    rng = np.random.default_rng(requests)
    past = rng.integers(0, 70, requests)
    past[:: 3] = past[:: 3] // page * page            # pages that are exactly full
    lengths = np.ones(requests, np.int64) if one else rng.integers(0, 90, requests)
    m = -(-160 // page)
    free = rng.permutation(requests * m).astype(np.int32)
    check(lengths, page, m, past=past, free=free, used=11, seed=requests)


@pytest.mark.parametrize("lengths", [[0], [0] * 100, [1], [0, 5, 0, 0, 7, 0], [1000], [4096, 0, 1]])
def test_empty_and_single_requests(lengths):
    check(lengths, 16, 300, free=np.arange(2000, dtype=np.int32)[::-1].copy())
    check(lengths, 16, 300, num_pages=2000, used=3)
    check(lengths, 5000, 1, num_pages=2000)


def test_pool_runs_out_and_tables_are_full():
    check([20, 20, 20], 8, 4, num_pages=5)                       # the second request gets part of its pages
    check([20, 20, 20], 8, 4, num_pages=0)
    check([20, 20, 20], 8, 4, num_pages=7, used=9)
    check([20, 20, 20], 8, 2, num_pages=50)                      # 16 rows fit a table row
    check([-4, 20, 3], 8, 4, past=[3, 40, -2], num_pages=50)
    check([1 << 60, 7, -(1 << 60)], 8, 4, past=[1 << 60, 3, 0], num_pages=50)
    check([3, 4], 8, 4, num_pages=50, used=-5)


def test_slot_map_shorter_and_longer_than_the_batch():
    for mt in (0, 1, 9, 10, 11, 500):
        check([4, 0, 6], 4, 3, num_pages=50, max_tokens=mt)


def test_long_requests_and_slots_beyond_32_bits():
    lay = check([3_000_000, 1_000_000], 64, 50000, num_pages=1 << 20, max_tokens=4_000_100)
    assert int(lay.offsets[-1]) == 4_000_000
    # page * page size beyond 2^31: the last pages of a pool of 2^27 pages of 64 rows
    free = np.array([(1 << 27) - 1, (1 << 27) - 2], np.int32)
    lay = check([100], 64, 2, free=free, max_tokens=100)
    assert int(lay.slot_map[0]) == ((1 << 27) - 1) * 64


def test_counter_in_place_and_repeated_steps():
    """Decoding: every step adds one row to each request, the counter lives on the device."""
    r, page, m = 37, 4, 8
    table = torch.full((r, m), -1, dtype=torch.int32, device=DEV)
    free = torch.randperm(r * m, device=DEV).to(torch.int32)
    used = torch.zeros(1, dtype=torch.int64, device=DEV)
    past = torch.zeros(r, dtype=torch.int64, device=DEV)
    one = torch.ones(r, dtype=torch.int64, device=DEV)
    seen = []
    for _ in range(30):
        lay = layout.paged_layout(one, page, table, used, free_pages=free, past=past, max_tokens=r, used_out=used)
        assert lay.used is used
        seen.append(lay.slot_map.clone())
        past += 1
    assert int(used) == r * 8
    slots = torch.stack(seen, 1).cpu().numpy()
    assert len(np.unique(slots)) == slots.size                   # no slot twice
    t = table.cpu().numpy()
    assert np.array_equal(slots, np.array([[t[i, s // page] * page + s % page for s in range(30)] for i in range(r)]))


def test_graphs_streams_and_preallocated_outputs():
    rng = np.random.default_rng(5)
    lengths = torch.from_numpy(rng.integers(0, 60, 3000)).to(DEV)
    table = torch.full((3000, 4), -1, dtype=torch.int32, device=DEV)
    used = torch.zeros(1, dtype=torch.int64, device=DEV)
    out = dict(offsets=torch.empty(3001, dtype=torch.int64, device=DEV),
               slot_map=torch.empty(200000, dtype=torch.int64, device=DEV))
    want = layout.paged_layout(lengths, 16, table.clone(), used, num_pages=1 << 20, max_tokens=200000)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        o = {k: torch.empty_like(v) for k, v in out.items()}
        t = table.clone()
        with torch.cuda.graph(g):
            lay = layout.paged_layout(lengths, 16, t, used, num_pages=1 << 20, **o)
        graphs.append((g, lay))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        for (g, _l), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for _g, lay in graphs:
        for a, b in zip(lay, want):
            assert torch.equal(a, b)
    lay = layout.paged_layout(lengths, 16, table.clone(), used, num_pages=1 << 20, max_tokens=200000,
                              stream=torch.cuda.Stream())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(lay, want))


def test_refusals():
    L = torch.ones(4, dtype=torch.int64, device=DEV)
    T = torch.zeros(4, 2, dtype=torch.int32, device=DEV)
    U = torch.zeros(1, dtype=torch.int64, device=DEV)
    bad = [
        lambda: layout.paged_layout(L.int(), 16, T, U, num_pages=5),
        lambda: layout.paged_layout(L.cpu(), 16, T, U, num_pages=5),
        lambda: layout.paged_layout(L, 16, T.long(), U, num_pages=5),
        lambda: layout.paged_layout(L, 16, T[:3], U, num_pages=5),
        lambda: layout.paged_layout(L, 16, T.t().contiguous().t(), U, num_pages=5),
        lambda: layout.paged_layout(L, 16, torch.zeros(4, 0, dtype=torch.int32, device=DEV), U, num_pages=5),
        lambda: layout.paged_layout(L, 0, T, U, num_pages=5),
        lambda: layout.paged_layout(L, -1, T, U, num_pages=5),
        lambda: layout.paged_layout(L, 1 << 31, T, U, num_pages=5),
        lambda: layout.paged_layout(L, 16, T, U),
        lambda: layout.paged_layout(L, 16, T, U, num_pages=-1),
        lambda: layout.paged_layout(L, 16, T, U, num_pages=6, free_pages=torch.zeros(5, dtype=torch.int32, device=DEV)),
        lambda: layout.paged_layout(L, 16, T, U.int(), num_pages=5),
        lambda: layout.paged_layout(L, 16, T, U, num_pages=5, past=L[:2]),
        lambda: layout.paged_layout(L, 16, T, U, num_pages=5, max_tokens=-1),
        lambda: layout.paged_layout(L, 16, T, U, num_pages=5, max_tokens=3,
                                    slot_map=torch.zeros(4, dtype=torch.int64, device=DEV)),
        lambda: layout.paged_layout(L, 16, T, U, num_pages=5, offsets=torch.zeros(4, dtype=torch.int64, device=DEV)),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(core.GearError) as e:
            f()
        assert e.value.code == N.ERR_INVALID, i


def test_refuses_sizes_beyond_the_argument_block():
    L = torch.ones(4, dtype=torch.int64, device=DEV)
    T = torch.zeros(4, 2, dtype=torch.int32, device=DEV)
    U = torch.zeros(1, dtype=torch.int64, device=DEV)
    for kw in (dict(page=1 << 70, num_pages=5), dict(page=16, num_pages=1 << 70), dict(page=(1 << 64) + 16, num_pages=5),
               dict(page=16, num_pages=-(1 << 70))):
        with pytest.raises(core.GearError) as e:
            layout.paged_layout(L, block_table=T, used=U, **kw)
        assert e.value.code == N.ERR_INVALID


@pytest.mark.parametrize("requests,most", [(1024, 3), (1024, 30), (1025, 3), (1, 4096), (700, 5), (8192, 2), (8193, 2), (20000, 1)])
@pytest.mark.parametrize("room", [1, 4096, 4097])
def test_ways_of_the_scan_and_of_the_fill(requests, most, room):
    """Sizes on both sides of every choice: requests a thread, one launch or several, tokens a request."""
    rng = np.random.default_rng(requests + most)
    lengths = rng.integers(0, most + 1, requests)
    past = rng.integers(0, 20, requests)
    page, blocks = 8, -(-(most + 20) // 8)
    have = -(-past // page)
    table = np.full((requests, blocks), -1, np.int32)
    nxt = 0
    for r in range(requests):
        table[r, :have[r]] = np.arange(nxt, nxt + have[r])
        nxt += have[r]
    free = (nxt + np.random.default_rng(1).permutation(requests * blocks)).astype(np.int32)
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(DEV)
    used = torch.tensor([7], dtype=torch.int64, device=DEV)
    lay = layout.paged_layout(dev(lengths), page, dev(table), used, free_pages=dev(free), past=dev(past), max_tokens=room)
    want_table, at, slots = table.copy(), 7, []
    for r in range(requests):
        need = -(-(past[r] + lengths[r]) // page) - have[r]
        want_table[r, have[r]:have[r] + need] = free[at:at + need]
        at += need
        for t in range(past[r], past[r] + lengths[r]):
            slots.append(int(want_table[r, t // page]) * page + t % page)
    want_slots = np.full(room, -1, np.int64)
    want_slots[:min(room, len(slots))] = slots[:room]
    assert np.array_equal(lay.offsets.cpu().numpy(), np.concatenate([[0], np.cumsum(lengths)]))
    assert np.array_equal(lay.block_table.cpu().numpy(), want_table)
    assert int(lay.used) == at
    assert np.array_equal(lay.slot_map.cpu().numpy(), want_slots)


@pytest.mark.parametrize("requests", [3, 9000])
def test_counter_at_and_behind_the_end_of_the_pool(requests):
    """Nothing is needed, so nothing is missing; the counter comes back as the pool's size."""
    for used in (7, 8, 1 << 40):
        check([0] * requests, 8, 4, num_pages=7, used=used)
        check([5] * requests, 8, 4, past=[3] * requests, num_pages=7, used=used)     # in the page there is


@pytest.mark.parametrize("requests", [3, 9000])
def test_wild_counters(requests):
    """Page numbers that would pass 64 bits name no page."""
    free = np.arange(40, dtype=np.int32)
    for used in ((1 << 63) - 1, (1 << 63) - 2, -(1 << 63), 1 << 62):
        check([20] * requests, 8, 4, free=free, used=used)


@pytest.mark.parametrize("tokens,past", [((1 << 31) - 1, 0), ((1 << 31) - 130, 0), ((1 << 31) - 130, 129), ((1 << 31) - 4, 3)])
def test_requests_as_long_as_they_may_be(tokens, past):
    """Every slot of a request of some 2^31 tokens, and of the one behind it."""
    page, blocks = 64, 1 << 25
    table = torch.full((2, blocks), -1, dtype=torch.int32, device=DEV)
    have = -(-past // page)
    if have:
        table[0, :have] = torch.arange(have, device=DEV, dtype=torch.int32)
    free = torch.arange(have, blocks + 2, device=DEV, dtype=torch.int32)
    status = torch.zeros(4, dtype=torch.int32, device=DEV)
    lay = layout.paged_layout(torch.tensor([tokens, 5], device=DEV), page, table, torch.zeros(1, dtype=torch.int64, device=DEV),
                              free_pages=free, past=torch.tensor([past, 0], device=DEV), max_tokens=tokens + 7, status=status)
    pages = -(-(past + tokens) // page)
    assert lay.offsets.tolist() == [0, tokens, tokens + 5] and int(lay.used) == pages + 1 - have and int(status[0]) == 0
    assert torch.equal(table[0, :pages], torch.arange(pages, device=DEV, dtype=torch.int32)) and (table[0, pages:] == -1).all()
    assert int(table[1, 0]) == pages and (table[1, 1:] == -1).all()
    for t in range(0, tokens, 1 << 28):             # the pages follow one another, so do the slots
        part = lay.slot_map[t:min(t + (1 << 28), tokens)]
        assert torch.equal(part, torch.arange(t + past, t + past + part.numel(), device=DEV))
    assert lay.slot_map[tokens:].tolist() == [pages * page + t for t in range(5)] + [-1, -1]


@pytest.mark.parametrize("page", [64, 48, 1 << 20, 1 << 31])
def test_pages_of_requests_as_long_as_they_may_be(page):
    blocks = (1 << 31) // page
    room = blocks * page
    table = torch.full((2, blocks), -1, dtype=torch.int32, device=DEV)
    lay = layout.paged_layout(torch.tensor([room, room], device=DEV), page, table, torch.zeros(1, dtype=torch.int64, device=DEV),
                              num_pages=3 * blocks // 2)
    assert lay.offsets.tolist() == [0, room, 2 * room] and int(lay.used) == 3 * blocks // 2
    want = torch.arange(2 * blocks, device=DEV, dtype=torch.int32)
    want[3 * blocks // 2:] = -1
    assert torch.equal(table.reshape(-1), want)


@pytest.mark.parametrize("requests,page,room", [(1024, 4096, 64), (1024, 4099, 0), (9000, 4096, 64), (1, 64, 1000)])
def test_tokens_without_slots_cost_their_pages_only(requests, page, room):
    """Far more tokens than slots (every path of the fill): all pages, and in the time of the pages."""
    blocks = (1 << 24) // page
    tokens = torch.full((requests,), blocks * page - 5, dtype=torch.int64, device=DEV)
    past = torch.zeros(requests, dtype=torch.int64, device=DEV)
    past[::3] = 3 * page + 1
    tokens[::3] -= 3 * page + 1
    have = -(-past // page)
    table = torch.full((requests, blocks), -1, dtype=torch.int32, device=DEV)
    used = torch.zeros(1, dtype=torch.int64, device=DEV)

    def call(t):
        return layout.paged_layout(tokens, page, t, used, num_pages=1 << 31, past=past, max_tokens=room)

    call(table.clone())
    t0, t1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    t0.record()
    lay = call(table)
    t1.record()
    torch.cuda.synchronize()
    per = blocks - have
    start = torch.cumsum(per, 0) - per
    col = torch.arange(blocks, device=DEV)[None]
    want = torch.where(col < have[:, None], -1, start[:, None] + col - have[:, None])
    assert torch.equal(lay.block_table.long(), want) and int(lay.used) == int(per.sum())
    for t in range(0, room, 7):                 # the first request has them all
        pos = int(past[0]) + t
        at = int(want[0, pos // page])
        assert int(lay.slot_map[t]) == (at * page + pos % page if at >= 0 else -1)
    assert t0.elapsed_time(t1) < 50             # milliseconds; token by token it was hundreds
