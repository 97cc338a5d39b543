"""The recurrences and their gradients in float64, one row after the other, with error bounds.

The bounds are those of float32 arithmetic on the same inputs.  One step h = a*h + x is one rounding of a value of at
most H_t = |a| H_(t-1) + |x|; a = exp(gate) is off by at most 2 units in the last place (4 half units); a state
carried over several rows as A*S + H rounds once for each product in A, like the steps it stands for, and once for
the sum.  So a row's own error is at most K half units of H_t with K = 1 + 4 + 2 (+ 1 to spare), and errors are
carried on by |a| like the values:  E_t = |a| E_(t-1) + K u H_t,  u = 2^-24.  The same holds for g.
A product g*h is off by |g| E_h + |h| E_g + u |g h| (twice u with log gates), a sum of n of them in any order by
n u of the sum of their magnitudes more.  Rounding to the output's type adds half a step of it.
"""
import numpy as np
import torch

U = 2.0 ** -24
K = 8.0
TINY = 1e-36   # below this float32 products may be flushed or subnormal

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SMALLEST = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def spans(rows, time, offsets, lengths):
    if offsets is not None:
        return [(int(a), int(b)) for a, b in zip(offsets[:-1], offsets[1:])]
    n = rows // time if time else 0
    ln = [time] * n if lengths is None else [int(v) for v in lengths]
    return [(b * time, b * time + v) for b, v in enumerate(ln)]


def reference(x, gate, seqs, h0=None, reverse=False, log=False, dh=None, dstate=None):
    """x [rows, D], gate [rows, G] float64 arrays -> dict of (value, bound) pairs, bounds before output rounding."""
    rows, d = x.shape
    g = gate.shape[1]
    per = d // g
    with np.errstate(all="ignore"):
        a = np.repeat(np.exp(gate) if log else gate, per, axis=1)
    aa = np.abs(a)
    h, eh = np.zeros((rows, d)), np.zeros((rows, d))
    prev, eprev = np.zeros((rows, d)), np.zeros((rows, d))
    out = {}
    ns = len(seqs)
    state, estate = np.zeros((ns, d)), np.zeros((ns, d))
    dx, edx = np.zeros((rows, d)), np.zeros((rows, d))
    dg, edg = np.zeros((rows, g)), np.zeros((rows, g))
    dh0, edh0 = np.zeros((ns, d)), np.zeros((ns, d))
    for s, (lo, hi) in enumerate(seqs):
        order = range(hi - 1, lo - 1, -1) if reverse else range(lo, hi)
        cur = np.zeros(d) if h0 is None else h0[s].copy()
        mag, err = np.abs(cur), np.zeros(d)
        first = True
        for r in order:
            prev[r], eprev[r] = cur, err
            if first and h0 is None:
                cur, mag, err = x[r].copy(), np.abs(x[r]), np.zeros(d)
            else:
                cur = a[r] * cur + x[r]
                mag = aa[r] * mag + np.abs(x[r])
                err = aa[r] * err + K * U * mag
            first = False
            h[r], eh[r] = cur, err
        state[s], estate[s] = cur, err
        if dh is None:
            continue
        c = np.zeros(d) if dstate is None else dstate[s].copy()
        cm, ce = np.abs(c), np.zeros(d)
        steps = list(order)
        for j in range(len(steps) - 1, -1, -1):
            r = steps[j]
            gr = dh[r] + c
            gm = np.abs(dh[r]) + cm
            ge = ce + K * U * gm
            dx[r], edx[r] = gr, ge
            if j > 0 or h0 is not None:
                f = a[r] if log else np.ones(d)
                v = gr * prev[r] * f
                e = (np.abs(gr) * eprev[r] + np.abs(prev[r]) * ge) * np.abs(f) + 8 * U * np.abs(v)
                dg[r] = v.reshape(g, per).sum(1)
                edg[r] = (e + per * U * np.abs(v)).reshape(g, per).sum(1)
            c, cm, ce = a[r] * gr, aa[r] * gm, aa[r] * ge + K * U * aa[r] * gm
        dh0[s], edh0[s] = c, ce
    out.update(h=(h, eh), state=(state, estate), dx=(dx, edx), dgate=(dg, edg), dh0=(dh0, edh0))
    return out


def check(got, want, dtype, what):
    """got (tensor) against (value, bound): the bound, half a step of the type, and its smallest values."""
    value, bound = want
    a = got.detach().double().cpu().numpy().reshape(value.shape)
    tol = bound * (1 + HALF_STEP[dtype]) + HALF_STEP[dtype] * np.abs(value) + SMALLEST[dtype] + TINY
    assert np.isfinite(a).all(), f"{what}: not finite"
    bad = np.abs(a - value) > tol
    if bad.any():
        i = np.unravel_index(np.argmax(np.where(bad, np.abs(a - value) / tol, 0)), bad.shape)
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.size} outside; at {i}: {a[i]} against {value[i]} "
                             f"(tolerance {tol[i]})")
