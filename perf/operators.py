"""Measured cases of the operators that turn sampled trajectories into model inputs and targets.

Four operators, each in a plain form (elementary torch operations) and as a user of this framework
calls it:

* recurrence  h_t = a_t * h_(t-1) + x_t over dense, padded or packed sequences (discounted returns and
              advantages with one channel, recurrent model layers with many);
* train       the same with its backward pass: gradients of inputs, gates and initial states;
* layout      offsets, block tables and slot maps from request lengths (a batch's pages);
* gather      the sampled requests' rows out of the trajectory table into a packed or paged batch.

`own` selects the side that run() takes.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = {"f32": 4, "bf16": 2, "f16": 2}


# --------------------------------------------------------------------------- #
# cases
# --------------------------------------------------------------------------- #
def _rec(name, layout, batch, time, width, gates, dtype, gate_dtype, gate, reverse, state, train):
    return {"name": name, "op": "train" if train else "recurrence", "layout": layout, "batch": batch, "time": time,
            "width": width, "gates": gates, "dtype": dtype, "gate_dtype": gate_dtype, "gate": gate,
            "reverse": reverse, "state": state}


def listed():
    return [
        # one token for each of 256 running requests: a recurrent policy that answers step by step
        _rec("step", "dense", 256, 1, 1024, 1024, "bf16", "f32", "log", False, True, False),
        # returns-to-go of one sampled batch: 1024 padded segments of 64 steps, one reward column
        _rec("returns_batch", "padded", 1024, 64, 1, 1, "f32", "f32", "decay", True, False, False),
        # returns or advantages of a packed collection of whole trajectories of up to 1000 steps
        _rec("returns_packed", "packed", 16384, 1000, 1, 1, "f32", "f32", "decay", True, False, False),
        # a recurrent layer over two long contexts
        _rec("layer_long", "dense", 2, 16384, 2048, 2048, "bf16", "f32", "log", False, True, False),
        # a layer with one gate for each of eight heads over ragged packed sequences, an odd width
        _rec("layer_heads_packed", "packed", 64, 1999, 1000, 8, "bf16", "bf16", "log", False, True, False),
        # training step of a recurrent layer, a gate for each channel
        _rec("train_dense", "dense", 4, 4096, 2048, 2048, "bf16", "f32", "log", False, False, True),
        # training step of a layer with a gate for each head, packed ragged segments with initial states
        _rec("train_heads_packed", "packed", 37, 1000, 1024, 16, "f32", "f32", "decay", True, True, True),
        # one more token for each of 256 running requests: the bookkeeping of a decoding step
        {"name": "layout_step", "op": "layout", "requests": 256, "new": 1, "past": 4096, "page": 16},
        # pages for a batch of new trajectories of up to 1000 steps
        {"name": "layout_batch", "op": "layout", "requests": 4096, "new": 1000, "past": 0, "page": 16},
        # pages and slots of a whole replay table's worth of segments
        {"name": "layout_table", "op": "layout", "requests": 131072, "new": 1000, "past": 0, "page": 64},
        # a sampled batch of 64-step segments out of the decision-transformer table, packed without padding
        {"name": "gather_packed", "op": "gather", "requests": 1024, "length": 64, "steps": 1000, "trajectories": 4096,
         "page": 0, "rows": "156,24,4,4,1"},
        # whole trajectories into the pages of a batch pool
        {"name": "gather_paged", "op": "gather", "requests": 8192, "length": 1000, "steps": 1000,
         "trajectories": 4096, "page": 16, "rows": "156,24,4,4,1"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_any(rng):
    op = rng.choice(["recurrence", "recurrence", "train", "train", "layout", "gather"])
    if op in ("recurrence", "train"):
        kind = rng.choice(["dense", "padded", "packed"])
        batch, time = _log_int(rng, 1, 16384), _log_int(rng, 1, 32768)
        gates = rng.choice([1, 2, 5, 8, 16, 0, 0, 0])
        per = _log_int(rng, 1, 512)
        width = gates * per if gates else _log_int(rng, 1, 4096)
        dtype = rng.choice(["f32", "bf16", "f16"])
        return _rec("", kind, batch, time, width, gates or width, dtype, rng.choice(["f32", dtype]),
                    rng.choice(["log", "decay"]), rng.random() < 0.5, rng.random() < 0.5, op == "train")
    if op == "layout":
        return {"op": op, "requests": _log_int(rng, 1, 131072), "new": _log_int(rng, 1, 4000),
                "past": rng.choice([0, _log_int(rng, 1, 4096)]), "page": rng.choice([1, 8, 16, 48, 64, 128])}
    steps = _log_int(rng, 20, 1000)
    return {"op": op, "requests": _log_int(rng, 1, 8192), "length": _log_int(rng, 1, steps), "steps": steps,
            "trajectories": _log_int(rng, 1, 4096), "page": rng.choice([0, 0, 4, 16, 24, 64]),
            "rows": rng.choice(["156,24,4,4,1", "68,24,4,1", "4096,4,4", "3,7,13,1,2,5"])}


def _cost(case):
    if case["op"] in ("recurrence", "train"):  # the plain form walks over the elements once for each doubling
        return case["batch"] * case["time"] * case["width"] * (1 + math.log2(max(2, case["time"])))
    if case["op"] == "gather":
        row = sum(int(r) for r in case["rows"].split(","))
        return max(work(case)["bytes"], case["trajectories"] * case["steps"] * row * 2)
    return work(case)["bytes"] + 16 * case["requests"] * _pages_per_request(case)


def draw(rng):
    most = {}
    for c in listed():
        most[c["op"]] = max(most.get(c["op"], 0), _cost(c))
    least = {"recurrence": 1 << 14, "train": 1 << 14, "layout": 0, "gather": 0}
    while True:
        c = _draw_any(rng)
        c.pop("name", None)
        if least[c["op"]] <= _cost(c) <= most[c["op"]]:
            return c


def _pages_per_request(case):
    return (case["past"] + case["new"] + case["page"] - 1) // case["page"] + 1


def work(case):
    """Bytes read once and written once; the lengths are drawn evenly, so the mean stands for them."""
    if case["op"] in ("recurrence", "train"):
        rows = case["batch"] * case["time"]
        if case["layout"] != "dense":
            rows = rows * 0.5
        x, g = SIZES[case["dtype"]], SIZES[case["gate_dtype"]]
        per_row = 2 * case["width"] * x + case["gates"] * g
        flops = 2 * case["width"]
        if case["op"] == "train":
            per_row += 2 * case["width"] * x + case["gates"] * g
            flops += 5 * case["width"]
        state = 8 * case["batch"] * case["width"] if case["state"] else 0
        if case["op"] == "train":
            state *= 2
        return {"bytes": rows * per_row + state, "flops": rows * flops}
    if case["op"] == "layout":
        tokens = case["requests"] * (1 if case["new"] == 1 else case["new"] / 2)
        pages = tokens / case["page"]
        return {"bytes": 8 * tokens + 8 * case["requests"] * (2 + (case["past"] > 0)) + 8 * pages, "flops": 0}
    row = sum(int(r) for r in case["rows"].split(","))
    tokens = case["requests"] * _mean_rows(case["length"], case["steps"])
    return {"bytes": tokens * row * 2 + case["requests"] * 32 + (4 * tokens / case["page"] if case["page"] else 0),
            "flops": 0}


def _mean_rows(length, steps):
    """Mean of min(length, len - ts) for len in [ts, steps], ts in [0, steps): what _requests draws."""
    n = 0.0
    for i in range(64):
        for j in range(64):
            ts = (i + 0.5) / 64 * steps
            n += min(length, (j + 0.5) / 64 * (steps - ts))
    return n / 4096


# --------------------------------------------------------------------------- #
# inputs
# --------------------------------------------------------------------------- #
def _generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _room(count, most, mean):
    """Rows that a batch buffer holds for `count` sequences of up to `most` rows: their mean and six deviations."""
    return min(count * most, int(count * mean + 3.0 * most * math.sqrt(count))) + 7


def _lengths(case, g, most):
    return torch.randint(0, most + 1, (case["batch"],), generator=g, device=DEV)


def _offsets(lengths, room):
    return torch.cat([lengths.new_zeros(1), torch.cumsum(lengths, 0)]).clamp(max=room)


def _recurrence_inputs(case, seed):
    g = _generator(seed)
    b, t, d, k = case["batch"], case["time"], case["width"], case["gates"]
    s = {"lengths": None, "offsets": None, "h0": None}
    if case["layout"] == "packed":
        # a batch buffer has room for more rows than this batch fills
        lead = (_room(b, t, t / 2),)
        s["offsets"] = _offsets(_lengths(case, g, t), lead[0])
    else:
        if case["layout"] == "padded":
            s["lengths"] = _lengths(case, g, t)
        lead = (b, t)
    s["x"] = torch.randn(lead + (d,), generator=g, device=DEV).to(DTYPES[case["dtype"]])
    u = torch.rand(lead + (k,), generator=g, device=DEV)
    if d == 1:
        # gamma * lambda of an advantage estimate, zero after a terminal step
        a = torch.where(u < 0.01, 0.0, 0.99 * 0.95 + 0.0 * u)
    else:
        # memories between two steps and some thousands, evenly over the logarithm
        a = torch.exp(-torch.exp(u * 8.0 - 8.0))
    if case["gate"] == "log":
        a = torch.log(a)
    s["gate"] = a.to(DTYPES[case["gate_dtype"]])
    if case["state"]:
        s["h0"] = torch.randn((b, d), generator=g, device=DEV)
    if case["op"] == "train":
        s["dh"] = torch.randn(lead + (d,), generator=g, device=DEV).to(DTYPES[case["dtype"]])
        s["dstate"] = torch.randn((b, d), generator=g, device=DEV) if case["state"] else None
    return s


def _layout_inputs(case, seed):
    g = _generator(seed)
    r, p = case["requests"], case["page"]
    new = torch.ones(r, dtype=torch.int64, device=DEV) if case["new"] == 1 else \
        torch.randint(0, case["new"] + 1, (r,), generator=g, device=DEV)
    past = torch.randint(0, case["past"] + 1, (r,), generator=g, device=DEV) if case["past"] else None
    m = _pages_per_request(case)
    pages = r * m + 5
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((r, m), -1, dtype=torch.int32, device=DEV)
    used = torch.zeros(1, dtype=torch.int64, device=DEV)
    if past is not None:
        have = (past + p - 1) // p
        first = torch.cumsum(have, 0) - have
        col = torch.arange(m, device=DEV)
        at = first[:, None] + col
        table = torch.where(col < have[:, None], order[at.clamp(max=pages - 1)], table)
        used = have.sum().reshape(1)
    return {"lengths": new, "past": past, "page": p, "table": table, "free": order, "used": used,
            "max_tokens": _room(r, case["new"], 1 if case["new"] == 1 else case["new"] / 2)}


def _requests(case, g):
    n, t = case["requests"], case["steps"]
    idx = torch.randint(0, case["trajectories"], (n,), generator=g, device=DEV)
    ts = torch.randint(0, t, (n,), generator=g, device=DEV)
    u = torch.rand(n, generator=g, device=DEV)
    ln = ts + torch.floor(u * (t - ts + 1)).to(torch.int64)
    return idx, ts, torch.minimum(ln, torch.full_like(ln, t))


def _gather_inputs(case, seed):
    g = _generator(seed)
    rows = [int(r) for r in case["rows"].split(",")]
    stride = sum(rows) * case["steps"]
    table = torch.randint(0, 256, (case["trajectories"] * stride,), generator=g, device=DEV, dtype=torch.uint8)
    idx, ts, ln = _requests(case, g)
    room = _room(case["requests"], case["length"], _mean_rows(case["length"], case["steps"]))
    offsets = _offsets((torch.minimum(ts + case["length"], ln) - ts).clamp(min=0), room)
    count = offsets[1:] - offsets[:-1]
    s = {"rows": rows, "steps": case["steps"], "stride": stride, "length": case["length"], "table": table, "idx": idx,
         "ts": ts, "ln": ln, "offsets": offsets, "page": case["page"], "blocks": None, "max_tokens": room}
    slots = room
    if case["page"]:
        m = -(-case["length"] // case["page"])
        need = (count + case["page"] - 1) // case["page"]
        pages = room // case["page"] + case["requests"]
        order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
        col = torch.arange(m, device=DEV)
        at = (torch.cumsum(need, 0) - need)[:, None] + col
        s["blocks"] = torch.where(col < need[:, None], order[at.clamp(max=pages - 1)], -1).to(torch.int32)
        slots = pages * case["page"]
    # the plain form puts what is no row of the batch into the place behind the pool
    s["places"] = [torch.zeros((slots + 1, r), dtype=torch.uint8, device=DEV) for r in rows]
    s["pools"] = [p[:slots] for p in s["places"]]
    return s


def prepare(case, seed):
    if case["op"] in ("recurrence", "train"):
        s = _recurrence_inputs(case, seed)
        if case["op"] == "train":
            for k in ("x", "gate", "h0"):
                if s[k] is not None:
                    s[k].requires_grad_(True)
    elif case["op"] == "layout":
        s = _layout_inputs(case, seed)
    else:
        s = _gather_inputs(case, seed)
        if own:
            # the same bytes in the framework's own table, with the columns subscribed
            from gear_b200 import _native, core
            t = core.TrajectoryTable(s["rows"], case["steps"], case["trajectories"], residency=_native.RES_HBM)
            t.connect()
            core.device_view(t.device_ptr, t.nbytes, torch.uint8).copy_(s["table"])
            s["handler"] = core.StorageHandler(t)
            s["columns"] = list(range(len(s["rows"])))
            s["handler"].set(s["columns"], [core.SubscribePattern(0, case["length"])] * len(s["rows"]))
    s["case"] = case
    return s


# --------------------------------------------------------------------------- #
# plain forms
# --------------------------------------------------------------------------- #
def _rows_of(s):
    """(sequence, place, live, lengths, first row of each sequence) of every row, flattened."""
    x = s["x"]
    if s["offsets"] is not None:
        off = s["offsets"]
        row = torch.arange(x.shape[0], device=x.device)
        seq = torch.searchsorted(off[1:], row, right=True)
        live = seq < off.numel() - 1
        seq = seq.clamp(max=off.numel() - 2)
        return seq, row - off[seq], live, off[1:] - off[:-1], off[:-1]
    b, t = x.shape[:2]
    row = torch.arange(b * t, device=x.device)
    seq = row // t
    lengths = s["lengths"] if s["lengths"] is not None else torch.full((b,), t, device=x.device)
    return seq, row - seq * t, row - seq * t < lengths[seq], lengths, torch.arange(b, device=x.device) * t


def _scan(a, x, longest):
    """h_i = a_i * h_(i-1) + x_i along dim 0 in float32, by doubling."""
    k = 1
    while k < longest:
        h, p = x.clone(), a.clone()
        h[k:].addcmul_(a[k:], x[:-k])
        p[k:] *= a[:-k]
        a, x, k = p, h, 2 * k
    return x


def _spread(gate, width):
    return gate if gate.shape[-1] == width else torch.repeat_interleave(gate, width // gate.shape[-1], dim=-1)


def _plain_recurrence(s):
    case = s["case"]
    train = case["op"] == "train"
    x = s["x"].detach()
    d = x.shape[-1]
    seq, at, live, lengths, first = _rows_of(s)
    longest = case["time"]
    begin = (at == 0) & live
    last = (at == lengths[seq] - 1) & live
    end_row = first + lengths - 1
    if case["reverse"]:
        begin, last, end_row = last, begin, first
    g = s["gate"].detach().reshape(-1, case["gates"]).float()
    a = torch.exp(g) if case["gate"] == "log" else g
    a = _spread(a, d)
    turn = (lambda v: torch.flip(v, (0,))) if case["reverse"] else (lambda v: v)
    on = live[:, None]
    first_row = begin[:, None]
    h0 = s["h0"].detach() if s["h0"] is not None else None
    xs = torch.where(on, x.reshape(-1, d).float(), 0.0)
    if h0 is not None:
        xs = xs + torch.where(first_row, a * h0[seq], 0.0)
    keep = torch.where(on & ~first_row, a, 0.0)
    h = turn(_scan(turn(keep), turn(xs), longest))
    state = torch.where((lengths > 0)[:, None], h[end_row.clamp(0, max(0, h.shape[0] - 1))],
                        torch.zeros_like(h[:1]) if h0 is None else h0)
    out = {"h": h.reshape(x.shape).to(x.dtype), "state": state if case["state"] else None}
    if not train:
        return out
    before = torch.roll(h, -1 if case["reverse"] else 1, 0)
    before = torch.where(first_row, torch.zeros_like(h[:1]) if h0 is None else h0[seq], before)
    dh = torch.where(on, s["dh"].reshape(-1, d).float(), 0.0)
    if s["dstate"] is not None:
        dh = dh + torch.where(last[:, None], s["dstate"][seq], 0.0)
    back = (lambda v: v) if case["reverse"] else (lambda v: torch.flip(v, (0,)))
    follow = torch.where(on & ~last[:, None], torch.roll(a, 1 if case["reverse"] else -1, 0), 0.0)
    gr = back(_scan(back(follow), back(dh), longest))
    da = gr * before
    if case["gate"] == "log":
        da = da * a
    da = torch.where(on, da, 0.0).reshape(-1, case["gates"], d // case["gates"]).sum(-1)
    out["dx"] = gr.reshape(x.shape).to(x.dtype)
    out["dgate"] = da.reshape(s["gate"].shape).to(s["gate"].dtype)
    if h0 is not None:
        start = (first + lengths - 1 if case["reverse"] else first).clamp(0, max(0, h.shape[0] - 1))
        carried = s["dstate"] if s["dstate"] is not None else torch.zeros_like(h0)
        out["dh0"] = torch.where((lengths > 0)[:, None], a[start] * gr[start], carried)
    else:
        out["dh0"] = None
    return out


def _plain_layout(s):
    p, free, table = s["page"], s["free"], s["table"]
    new = s["lengths"]
    past = s["past"] if s["past"] is not None else torch.zeros_like(new)
    m = table.shape[1]
    have = (past + p - 1) // p
    need = (past + new + p - 1) // p - have
    offsets = torch.cat([new.new_zeros(1), torch.cumsum(new, 0)])
    first = s["used"] + torch.cumsum(need, 0) - need
    col = torch.arange(m, device=new.device)
    fresh = (col >= have[:, None]) & (col < (have + need)[:, None])
    page = (first[:, None] + col - have[:, None]).clamp(0, free.numel() - 1)
    table = torch.where(fresh, free[page], table)
    tok = torch.arange(s["max_tokens"], device=new.device)
    r = torch.searchsorted(offsets[1:], tok, right=True)
    valid = r < new.numel()
    r = r.clamp(max=new.numel() - 1)
    t = tok - offsets[r] + past[r]
    block = (t // p).clamp(max=m - 1)
    slots = torch.where(valid, table[r, block].to(torch.int64) * p + t % p, -1)
    return {"offsets": offsets, "slots": slots, "table": table, "used": s["used"] + need.sum()}


def _plain_gather(s):
    off, n = s["offsets"], s["max_tokens"]
    tok = torch.arange(n, device=off.device)
    r = torch.searchsorted(off[1:], tok, right=True)
    valid = r < off.numel() - 1
    r = r.clamp(max=off.numel() - 2)
    t = torch.where(valid, tok - off[r], 0)
    slot = tok
    if s["page"]:
        slot = s["blocks"][r, t // s["page"]].to(torch.int64) * s["page"] + t % s["page"]
    slot = torch.where(valid, slot, s["pools"][0].shape[0])
    who, step = s["idx"][r], s["ts"][r] + t
    count, done = s["table"].numel() // s["stride"], 0
    for row, pool in zip(s["rows"], s["places"]):
        column = s["table"].as_strided((count, s["steps"], row), (s["stride"], row, 1), done * s["steps"])
        pool[slot] = column[who, step]
        done += row
    return s["pools"]


# --------------------------------------------------------------------------- #
# one pass
# --------------------------------------------------------------------------- #
def run(state):
    op = state["case"]["op"]
    if not own:
        if op == "layout":
            return _plain_layout(state)
        return _plain_gather(state) if op == "gather" else _plain_recurrence(state)
    if op == "layout":
        from gear_b200 import layout
        lay = layout.paged_layout(state["lengths"], state["page"], state["table"], state["used"],
                                  free_pages=state["free"], past=state["past"], max_tokens=state["max_tokens"])
        return {"offsets": lay.offsets, "slots": lay.slot_map, "table": lay.block_table, "used": lay.used}
    if op == "gather":
        state["handler"].gather_packed(state["columns"], state["idx"], state["ts"], state["ln"], state["offsets"],
                                       state["pools"], block_table=state["blocks"], page=state["page"])
        return state["pools"]
    from gear_b200 import recurrence
    case = state["case"]
    h, last = recurrence.linear_recurrence(state["x"], state["gate"], h0=state["h0"], offsets=state["offsets"],
                                           lengths=state["lengths"], reverse=case["reverse"], gate_kind=case["gate"],
                                           return_state=case["state"])
    out = {"h": h.detach(), "state": last.detach() if case["state"] else None}
    if op == "recurrence":
        return out
    wrt = [state["x"], state["gate"]] + ([state["h0"]] if case["state"] else [])
    grads = torch.autograd.grad([h, last] if case["state"] else [h], wrt,
                                [state["dh"], state["dstate"]] if case["state"] else [state["dh"]])
    out["dx"], out["dgate"], out["dh0"] = grads[0], grads[1], grads[2] if case["state"] else None
    return out


# --------------------------------------------------------------------------- #
# the definition in 64 bits
# --------------------------------------------------------------------------- #
def exact(case, seed):
    """The recurrences step by step in float64; whole numbers and bytes have no such value."""
    if case["op"] not in ("recurrence", "train"):
        return None
    if case["time"] > 20000 or case["batch"] * case["time"] * case["width"] > 140_000_000:
        return None
    s = _recurrence_inputs(case, seed)
    d, k = case["width"], case["gates"]
    x = s["x"].reshape(-1, d).double()
    g = s["gate"].reshape(-1, k).double()
    a = g.exp() if case["gate"] == "log" else g
    n, b = x.shape[0], case["batch"]
    if s["offsets"] is not None:
        first, lengths = s["offsets"][:-1], s["offsets"][1:] - s["offsets"][:-1]
    else:
        first = torch.arange(b, device=x.device) * case["time"]
        lengths = s["lengths"] if s["lengths"] is not None else torch.full((b,), case["time"], device=x.device)
    longest = int(lengths.max())

    def rows(j):
        """Row of the j-th step of every sequence; n, the row of a scratch place, where there is none."""
        at = first + (lengths - 1 - j if case["reverse"] else j)
        return torch.where(j < lengths, at, n)

    per = d // k
    a = torch.cat([a, a.new_ones(1, k)])
    x = torch.cat([x, x.new_zeros(1, d)])
    h = torch.zeros_like(x)
    h0 = s["h0"].double() if s["h0"] is not None else x.new_zeros(b, d)
    cur = h0.clone()
    for j in range(longest):
        r = rows(j)
        cur = (a[r].unsqueeze(-1) * cur.view(b, k, per)).view(b, d) + x[r]
        h[r] = cur
    out = {"h": h[:n].reshape(s["x"].shape), "state": cur if case["state"] else None}
    if case["op"] == "recurrence":
        return out
    dh = torch.cat([s["dh"].reshape(-1, d).double(), x.new_zeros(1, d)])
    dx, da = torch.zeros_like(x), torch.zeros_like(a)
    carry = s["dstate"].double() if s["dstate"] is not None else x.new_zeros(b, d)
    h[n] = 0.0
    for j in reversed(range(longest)):
        r = rows(j)
        on = (j < lengths)[:, None]
        grad = dh[r] + carry
        prev = h0 if j == 0 else h[rows(j - 1)]
        dx[r] = grad
        da[r] = (grad * prev).view(b, k, per).sum(-1) * (a[r] if case["gate"] == "log" else 1.0)
        carry = torch.where(on, (a[r].unsqueeze(-1) * grad.view(b, k, per)).view(b, d), carry)
    out["dx"] = dx[:n].reshape(s["x"].shape)
    out["dgate"] = da[:n].reshape(s["gate"].shape)
    out["dh0"] = carry if case["state"] else None
    return out
