// Kernels of the recurrences for rows of many channels: one warp a row, V channels a lane.
//
// Three phases with a barrier between them.  Every warp forms (A, H) of its eight rows; then one thread per channel goes
// through the warps' pairs, publishes the tile's, learns the state before the tile and leaves the state before
// each warp; then every warp runs its rows from there.  These take what the streaming kernels cannot: rows that are not
// one matrix on 16-byte boundaries, odd widths, gates of up to 32 channels in the backward pass.  Bound by the latency
// of the phases: a CTA takes some 13 us for its tile, whatever its types, so what counts is how many fit an SM
// (2 to 5, by V) and how many bytes each has under way.  Where rows are not aligned for vectors a lane takes two
// channels 32 apart; with one channel a lane 650 x 64 x 1233 float16 with float32 gates took 235 us, now 148 (63 at
// the copy rate), 54 x 10733 x 43 221, now 156.  2 x 16384 x 2048 bf16 170 us (115 in the streaming kernels).
#pragma once

#include "recurrence.cuh"

namespace gearb {
namespace rec {

template <typename TA, int V, int kGate, bool kApart>
__device__ __forceinline__ void load_gate(const Params &P, const Place &pl, const TileRows &tr, int warp, int n,
                                          const Channels<V, kApart> &ch, float (&a)[kRows][kGate == kOne ? 1 : V]) {
  const TA *gate = static_cast<const TA *>(P.A.gate);
  auto one = [&](int g, bool on, int v) {  // gate g, for the lane's channel v
    const Channels<1, false> at(g, on ? g + 1 : g);
    Pack<TA, 1> raw[kRows];
    load_rows<TA>(gate, P, pl, tr, P.gate_period, P.A.gate_batch_stride, P.A.gate_row_stride, warp, n, at, raw);
#pragma unroll
    for (int k = 0; k < kRows; ++k) a[k][v] = to_f(raw[k].v[0]);
  };
  if constexpr (kGate == kTable) {
#pragma unroll
    for (int v = 0; v < V; ++v) one(ch.on(v) ? ch.at(v) / P.per : 0, ch.on(v), v);
  } else if constexpr (kGate == kOne) {
    one(static_cast<int>(pl.gate), ch.on(0), 0);
  } else {
    Pack<TA, V> raw[kRows];
    load_rows<TA>(gate, P, pl, tr, P.gate_period, P.A.gate_batch_stride, P.A.gate_row_stride, warp, n, ch, raw);
#pragma unroll
    for (int k = 0; k < kRows; ++k)
#pragma unroll
      for (int v = 0; v < V; ++v) a[k][v] = to_f(raw[k].v[v]);
  }
}

template <int kG>
__device__ __forceinline__ void exp_gate(float (&a)[kRows][kG]) {
#pragma unroll
  for (int k = 0; k < kRows; ++k)
#pragma unroll
    for (int v = 0; v < kG; ++v) a[k][v] = exp_of(a[k][v]);
}


// The tile's rows, and this warp's: looked up for the whole tile first, by each warp only where a sequence starts or
// ends in it.
struct SharedRows {
  TileRows t;
};
__device__ __forceinline__ TileRows rows_of_tile(const Params &P, const Place &pl) {
  if (!P.A.offsets) return tile_rows_dense(P, pl);
  TileRows t;
  t.bb = 0;
  t.tt = row_of(P, pl.i0);
  t.linear = true;
  t.interior = false;
  t.first_start = t.last_end = 0;
  return t;
}
__device__ __forceinline__ RowMap rows_of_warp(const Params &P, const Place &pl, TileRows &t, SharedRows &sm, int64_t i0, int n,
                                               int warp, int lane) {
  if (P.A.offsets) {
    if (warp == 0) {
      const TileRows found = tile_rows_packed(P, pl, lane);
      if (lane == 0) sm.t = found;
    }
    __syncthreads();
    t = sm.t;
  }
  if (!t.interior) return map_rows(P.A, P.rows, i0, n, lane);
  RowMap m;
  m.live = kAllRows;
  m.start = m.end = 0;
  m.seq = 0;
  m.first_start = t.first_start;
  m.last_end = t.last_end;
  return m;
}

// A float of every channel of [sequences][width], of the lane's channels of one sequence (the streaming kernels: of V
// consecutive ones).
template <int V>
__device__ __forceinline__ void state_load(const float *p, int seq, int64_t width, int64_t d, bool on, float (&r)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) r[v] = (p && on) ? p[static_cast<int64_t>(seq) * width + d + v] : 0.0f;
}
template <int V>
__device__ __forceinline__ void state_store(float *p, int seq, int64_t width, int64_t d, bool on, const float (&r)[V]) {
  if (p && on)
#pragma unroll
    for (int v = 0; v < V; ++v) p[static_cast<int64_t>(seq) * width + d + v] = r[v];
}
template <int V, bool kApart>
__device__ __forceinline__ void state_load(const float *p, int seq, int64_t width, const Channels<V, kApart> &ch, float (&r)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) r[v] = (p && ch.on(v)) ? p[static_cast<int64_t>(seq) * width + ch.at(v)] : 0.0f;
}
template <int V, bool kApart>
__device__ __forceinline__ void state_store(float *p, int seq, int64_t width, const Channels<V, kApart> &ch, const float (&r)[V]) {
  if (p)
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (ch.on(v)) p[static_cast<int64_t>(seq) * width + ch.at(v)] = r[v];
}

template <typename TX, typename TA, int V, int kGate, bool kApart>
__global__ void __launch_bounds__(kThreads, V == 4 ? 2 : V == 2 ? 3 : 5) forward_kernel(const __grid_constant__ Params P) {
  static_assert(kGate != kOne, "forward calls take a table of gates");
  constexpr int kW = 32 * V;  // channels of a block
  __shared__ float sa[kWarps][kW], sh[kWarps][kW];
  __shared__ int scut[kWarps];
  __shared__ unsigned sticket;
  __shared__ SharedRows srows;
  __shared__ int64_t sfirst;  // scan index at which the first row's sequence starts, or -1: nothing is needed from before
  const gearb_recurrence_args &A = P.A;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Place pl = take_place<V, kGate>(P, &sticket, false);
  const Channels<V, kApart> chans(pl, lane);
  const int64_t i0 = pl.i0 + warp * kRows;
  const int n = static_cast<int>(i0 >= pl.i1 ? 0 : (pl.i1 - i0 < kRows ? pl.i1 - i0 : kRows));

  Pack<TX, V> x[kRows];
  float a[kRows][V];
  TileRows tr = rows_of_tile(P, pl);
  load_rows<TX>(static_cast<const TX *>(A.x), P, pl, tr, P.x_period, A.x_batch_stride, A.x_row_stride, warp, n, chans, x);
  load_gate<TA, V, kGate>(P, pl, tr, warp, n, chans, a);
  const RowMap m = rows_of_warp(P, pl, tr, srows, i0, n, warp, lane);
  if (A.gate_log) exp_gate(a);
  const bool plain = m.live == kAllRows && (m.start | m.end) == 0;

  // (A, H) of this warp's rows; behind a start only H counts
  float ca[V], ch[V];
#pragma unroll
  for (int v = 0; v < V; ++v) { ca[v] = 1.0f; ch[v] = 0.0f; }
  if (plain) {
#pragma unroll
    for (int k = 0; k < kRows; ++k)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float av = a[k][v];
        ch[v] = fmaf(av, ch[v], to_f(x[k].v[v]));
        ca[v] *= av;
      }
  } else {
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      if (!(m.live >> k & 1u)) continue;
      const bool st = m.start >> k & 1u;
      float s[V];
      if (st) state_load<V>(A.h0, __shfl_sync(kAll, m.seq, k), A.width, chans, s);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float av = a[k][v], xv = to_f(x[k].v[v]);
        if (st) ch[v] = A.h0 ? fmaf(av, s[v], xv) : xv;
        else ch[v] = fmaf(av, ch[v], xv);
        ca[v] *= av;
      }
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) { sa[warp][chans.of(lane, v)] = ca[v]; sh[warp][chans.of(lane, v)] = ch[v]; }
  if (lane == 0) {
    scut[warp] = m.start != 0;
    if (warp == 0) sfirst = ((m.live & ~m.start) & 1u) ? m.first_start : -1;
  }
  __syncthreads();

  const int64_t ch2 = pl.d0 + threadIdx.x;
  if (threadIdx.x < kW && ch2 < pl.d1) {
    float ta = 1.0f, th = 0.0f;  // of the rows before warp q
    bool cut = false;
    float pa[kWarps], ph[kWarps];
#pragma unroll
    for (int q = 0; q < kWarps; ++q) {
      const float b = sa[q][threadIdx.x], h = sh[q][threadIdx.x];
      pa[q] = ta;
      ph[q] = th;
      th = scut[q] ? h : fmaf(b, th, h);
      ta *= b;
      cut |= scut[q] != 0;
    }
    float cin = 0.0f;
    if (P.chain) {
      publish_pair(P.agg + pl.tile * A.width + ch2, ta, th);
      const int64_t lo = sfirst >= 0 ? quotient(sfirst, P.tile_rows) : pl.tile;
      bool lost = false;
      cin = look_back<4, 0, int64_t>(P, pl.tile, lo, ch2, [&] { return make_float2(ta, th); }, cut, lost);
      if (lost && A.status) atomicOr(reinterpret_cast<unsigned *>(A.status), GEARB_ST_SCAN_ABORTED);
      if (lo < pl.tile && A.carry) A.carry[pl.tile * A.width + ch2] = cin;
    }
    cut = false;
#pragma unroll
    for (int q = 0; q < kWarps; ++q) {  // the state before warp q
      sh[q][threadIdx.x] = cut ? ph[q] : fmaf(pa[q], cin, ph[q]);
      cut |= scut[q] != 0;
    }
  }
  __syncthreads();

  if (n > 0) {
    float h[V];
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = sh[warp][chans.of(lane, v)];
    TX *out = static_cast<TX *>(A.out) + row_of(P, i0) * A.width;
    const int64_t step = A.reverse ? -A.width : A.width;
    if (plain) {
#pragma unroll
      for (int k = 0; k < kRows; ++k) {
#pragma unroll
        for (int v = 0; v < V; ++v) h[v] = fmaf(a[k][v], h[v], to_f(x[k].v[v]));
        chans.store(out + k * step, h);
      }
    } else {
#pragma unroll
      for (int k = 0; k < kRows; ++k) {
        if (k >= n) break;
        if (!(m.live >> k & 1u)) {
          if (A.zero_rest) {
            const float z[V] = {};
            chans.store(out + k * step, z);
          }
          continue;
        }
        const int seq = __shfl_sync(kAll, m.seq, k);
        if (m.start >> k & 1u) {
          float s[V];
          state_load<V>(A.h0, seq, A.width, chans, s);
#pragma unroll
          for (int v = 0; v < V; ++v) {
            const float xv = to_f(x[k].v[v]);
            h[v] = A.h0 ? fmaf(a[k][v], s[v], xv) : xv;
          }
        } else {
#pragma unroll
          for (int v = 0; v < V; ++v) h[v] = fmaf(a[k][v], h[v], to_f(x[k].v[v]));
        }
        chans.store(out + k * step, h);
        if (m.end >> k & 1u) state_store<V>(A.state_out, seq, A.width, chans, h);
      }
    }
  }
  empty_sequences(P, pl, kW, A.h0, A.state_out);
}

// Sums of kRows values over the 32 lanes, by halving: with every shuffle a lane gives away half of the values it still
// holds.  Lane l ends up with the sum of value row_of_lane(l); 7 + 2 shuffles for eight values instead of forty.
constexpr int kSpare = 32 / kRows;  // lanes that hold the same value in the end
__device__ __forceinline__ int row_of_lane(int lane) { return lane / kSpare; }
__device__ __forceinline__ float sum_rows(float (&v)[kRows], int lane) {
#pragma unroll
  for (int half = kRows / 2, m = 16; half > 0; half >>= 1, m >>= 1) {
    const bool up = lane & m;
#pragma unroll
    for (int j = 0; j < half; ++j) {
      const float give = up ? v[j] : v[j + half], keep = up ? v[j + half] : v[j];
      v[j] = keep + __shfl_xor_sync(kAll, give, m);
    }
  }
#pragma unroll
  for (int m = kSpare / 2; m > 0; m >>= 1) v[0] += __shfl_xor_sync(kAll, v[0], m);
  return v[0];
}

// Products are rounded (__fmul_rn) before they are added, as in the streaming kernels: left to the compiler, some would be
// fused with the addition in one kernel and not in the other.
template <typename TX, typename TA, int V, int kGate, bool kApart>
__global__ void __launch_bounds__(kThreads, V == 4 ? 2 : V == 2 ? 3 : 4) backward_kernel(const __grid_constant__ Params P) {
  constexpr int kG = kGate == kOne ? 1 : V;
  constexpr int kW = 32 * V;
  __shared__ float sa[kWarps][kW], sh[kWarps][kW], sc[kWarps][kW];
  __shared__ int scut[kWarps], send[kWarps];
  __shared__ unsigned sticket;
  __shared__ SharedRows srows;
  __shared__ int64_t slast;   // scan index at which the last row's sequence ends, or -1: nothing is needed from behind
  __shared__ int sopen;       // the first row continues a sequence of an earlier tile
  const gearb_recurrence_args &A = P.A;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Place pl = take_place<V, kGate>(P, &sticket, true);
  const Channels<V, kApart> chans(pl, lane);
  const int64_t i0 = pl.i0 + warp * kRows;
  const int n = static_cast<int>(i0 >= pl.i1 ? 0 : (pl.i1 - i0 < kRows ? pl.i1 - i0 : kRows));

  Pack<TX, V> x[kRows], dh[kRows];
  float a[kRows][kG];
  TileRows tr = rows_of_tile(P, pl);
  load_rows<TX>(static_cast<const TX *>(A.x), P, pl, tr, P.x_period, A.x_batch_stride, A.x_row_stride, warp, n, chans, x);
  load_gate<TA, V, kGate>(P, pl, tr, warp, n, chans, a);
  load_rows<TX>(static_cast<const TX *>(A.dout), P, pl, tr, P.dout_period, A.dout_batch_stride, A.dout_row_stride, warp, n,
                chans, dh);
  const RowMap m = rows_of_warp(P, pl, tr, srows, i0, n, warp, lane);
  if (A.gate_log) exp_gate(a);
  const bool plain = m.live == kAllRows && (m.start | m.end) == 0;

  // (A, H) of this warp's rows forward, (A, C) backward
  float ca[V], ch[V], cc[V];
#pragma unroll
  for (int v = 0; v < V; ++v) { ca[v] = 1.0f; ch[v] = 0.0f; cc[v] = 0.0f; }
  if (plain) {
#pragma unroll
    for (int k = 0; k < kRows; ++k)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float av = a[k][kGate == kOne ? 0 : v];
        ch[v] = fmaf(av, ch[v], to_f(x[k].v[v]));
        ca[v] *= av;
      }
#pragma unroll
    for (int k = kRows - 1; k >= 0; --k)
#pragma unroll
      for (int v = 0; v < V; ++v) cc[v] = __fmul_rn(a[k][kGate == kOne ? 0 : v], to_f(dh[k].v[v]) + cc[v]);
  } else {
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      if (!(m.live >> k & 1u)) continue;
      const bool st = m.start >> k & 1u;
      float s[V];
      if (st) state_load<V>(A.h0, __shfl_sync(kAll, m.seq, k), A.width, chans, s);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float av = a[k][kGate == kOne ? 0 : v], xv = to_f(x[k].v[v]);
        if (st) ch[v] = A.h0 ? fmaf(av, s[v], xv) : xv;
        else ch[v] = fmaf(av, ch[v], xv);
        ca[v] *= av;
      }
    }
#pragma unroll
    for (int k = kRows - 1; k >= 0; --k) {
      if (!(m.live >> k & 1u)) continue;
      if (m.end >> k & 1u) state_load<V>(A.dstate, __shfl_sync(kAll, m.seq, k), A.width, chans, cc);
#pragma unroll
      for (int v = 0; v < V; ++v) cc[v] = __fmul_rn(a[k][kGate == kOne ? 0 : v], to_f(dh[k].v[v]) + cc[v]);
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    sa[warp][chans.of(lane, v)] = ca[v];
    sh[warp][chans.of(lane, v)] = ch[v];
    sc[warp][chans.of(lane, v)] = cc[v];
  }
  if (lane == 0) {
    scut[warp] = m.start != 0;
    send[warp] = m.end != 0;
    if (warp == 0) sopen = ((m.live & ~m.start) & 1u) && quotient(m.first_start, P.tile_rows) < pl.tile;
    if (n > 0 && i0 + n == pl.i1) slast = ((m.live & ~m.end) >> (n - 1) & 1u) ? m.last_end : -1;
  }
  __syncthreads();

  // one thread per channel backward, another forward
  if (threadIdx.x < kW) {
    const int64_t ch2 = pl.d0 + threadIdx.x;
    if (ch2 < pl.d1) {
      const int64_t at = P.tiles - 1 - pl.tile;  // place of the tile in the order of the tickets
      float ta = 1.0f, tc = 0.0f;  // of the rows behind warp q
      bool cut = false;
      float pa[kWarps], pc[kWarps];
#pragma unroll
      for (int q = kWarps - 1; q >= 0; --q) {
        const float b = sa[q][threadIdx.x], c = sc[q][threadIdx.x];
        pa[q] = ta;
        pc[q] = tc;
        tc = send[q] ? c : fmaf(b, tc, c);
        ta *= b;
        cut |= send[q] != 0;
      }
      float cin = 0.0f;
      if (P.chain) {
        publish_pair(P.agg + at * A.width + ch2, ta, tc);
        const int64_t lo = slast >= 0 ? P.tiles - 1 - quotient(slast, P.tile_rows) : at;
        bool lost = false;
        cin = look_back<4, 0, int64_t>(P, at, lo < at ? lo : at, ch2, [&] { return make_float2(ta, tc); }, cut, lost);
        if (lost && A.status) atomicOr(reinterpret_cast<unsigned *>(A.status), GEARB_ST_SCAN_ABORTED);
      }
      cut = false;
#pragma unroll
      for (int q = kWarps - 1; q >= 0; --q) {
        sc[q][threadIdx.x] = cut ? pc[q] : fmaf(pa[q], cin, pc[q]);
        cut |= send[q] != 0;
      }
    }
  } else if (threadIdx.x < 2 * kW) {
    const int c0 = threadIdx.x - kW;
    const int64_t ch2 = pl.d0 + c0;
    if (ch2 < pl.d1) {
      const float hin = (P.chain && sopen) ? __ldg(A.carry + pl.tile * A.width + ch2) : 0.0f;
      float ta = 1.0f, th = 0.0f;
      bool cut = false;
#pragma unroll
      for (int q = 0; q < kWarps; ++q) {
        const float b = sa[q][c0], h = sh[q][c0];
        sh[q][c0] = cut ? th : fmaf(ta, hin, th);
        th = scut[q] ? h : fmaf(b, th, h);
        ta *= b;
        cut |= scut[q] != 0;
      }
    }
  }
  __syncthreads();

  if (n > 0) {
    float hp[kRows][V], h[V], c[V], part[kRows];  // hp: h_(t-1) of every row
#pragma unroll
    for (int v = 0; v < V; ++v) { h[v] = sh[warp][chans.of(lane, v)]; c[v] = sc[warp][chans.of(lane, v)]; }
    const int64_t row0 = row_of(P, i0), sign = A.reverse ? -1 : 1, xs = sign * A.width, gs = sign * A.gates;
    TX *dx = static_cast<TX *>(A.dx) + row0 * A.width;
    TA *dgate = static_cast<TA *>(A.dgate) + row0 * A.gates +
                (kGate == kOne ? pl.gate : kGate == kTable ? pl.d0 / P.per : 0);
    // Gates of a few channels each: a row's products through shared memory, a lane a gate (blocks hold whole gates).
    auto sum_gates = [&](int k, bool wanted, const float (&da)[V]) {
#pragma unroll
      for (int v = 0; v < V; ++v) sa[warp][chans.of(lane, v)] = da[v];
      __syncwarp();
      const int cols = static_cast<int>(pl.d1 - pl.d0);
      for (int j = lane; j * P.per < cols; j += 32) {
        float sum = 0.0f;
        for (int u = 0; u < P.per; ++u) sum += sa[warp][j * P.per + u];
        if (wanted) dgate[k * gs + j] = from_f<TA>(sum);
      }
      __syncwarp();
    };
    if (plain) {
#pragma unroll
      for (int k = 0; k < kRows; ++k)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          hp[k][v] = h[v];
          h[v] = fmaf(a[k][kGate == kOne ? 0 : v], h[v], to_f(x[k].v[v]));
        }
#pragma unroll
      for (int k = kRows - 1; k >= 0; --k) {
        float g[V], da[V];
        part[k] = 0.0f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float av = a[k][kGate == kOne ? 0 : v];
          g[v] = to_f(dh[k].v[v]) + c[v];
          c[v] = __fmul_rn(av, g[v]);
          da[v] = __fmul_rn(A.gate_log ? c[v] : g[v], hp[k][v]);
          part[k] += chans.on(v) ? da[v] : 0.0f;
        }
        chans.store(dx + k * xs, g);
        if constexpr (kGate == kOwn) chans.store(dgate + k * gs, da);
        if constexpr (kGate == kTable) sum_gates(k, true, da);
      }
    } else {
#pragma unroll
      for (int k = 0; k < kRows; ++k) {
        const bool st = m.start >> k & 1u, lv = m.live >> k & 1u;
        if (st) state_load<V>(A.h0, __shfl_sync(kAll, m.seq, k), A.width, chans, h);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float xv = to_f(x[k].v[v]);
          hp[k][v] = h[v];
          if (lv) h[v] = (st && !A.h0) ? xv : fmaf(a[k][kGate == kOne ? 0 : v], h[v], xv);
        }
      }
#pragma unroll
      for (int k = kRows - 1; k >= 0; --k) {
        part[k] = 0.0f;
        if (k >= n) continue;
        const bool lv = m.live >> k & 1u, st = m.start >> k & 1u;
        const int seq = __shfl_sync(kAll, m.seq, k);
        if (m.end >> k & 1u) state_load<V>(A.dstate, seq, A.width, chans, c);
        float g[V], da[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float av = a[k][kGate == kOne ? 0 : v];
          g[v] = lv ? to_f(dh[k].v[v]) + c[v] : 0.0f;
          if (lv) c[v] = __fmul_rn(av, g[v]);
          // the first row of a sequence without h0 is h = x: its gate plays no part
          da[v] = (lv && !(st && !A.h0)) ? __fmul_rn(A.gate_log ? c[v] : g[v], hp[k][v]) : 0.0f;
          part[k] += chans.on(v) ? da[v] : 0.0f;
        }
        if (lv || A.zero_rest) {
          chans.store(dx + k * xs, g);
          if constexpr (kGate == kOwn) chans.store(dgate + k * gs, da);
        }
        if constexpr (kGate == kTable) sum_gates(k, lv || A.zero_rest, da);
        if (st) state_store<V>(A.dh0, seq, A.width, chans, c);
      }
    }
    if constexpr (kGate == kOne) {
      const float sum = sum_rows(part, lane);
      const int k = row_of_lane(lane);
      if (lane % kSpare == 0 && k < n && ((m.live >> k & 1u) || A.zero_rest)) {
        if (P.blocks_per_gate == 1) dgate[k * gs] = from_f<TA>(sum);
        else P.gate_part[(pl.part * P.rows + row0 + k * sign) * A.gates + pl.gate] = sum;
      }
    }
  }
  empty_sequences(P, pl, kW, A.dstate, A.dh0);
}

template <typename TX, typename TA, int V, int kGate, bool kApart>
int launch_wide(Params &p, bool backward, cudaStream_t stream) {
  const gearb_recurrence_args &a = p.A;
  p.block = 32 * V;
  if (kGate == kTable && backward) {  // whole gates, and whole vectors
    const int unit = kApart || p.per % V == 0 ? p.per : (p.per % 2 == 0 && V == 4 ? 2 : V) * p.per;
    p.block = 32 * V / unit * unit;
  }
  p.blocks_per_gate = kGate == kOne ? (p.per + 32 * V - 1) / (32 * V) : 1;
  const int64_t ncol = kGate == kOne ? a.gates * p.blocks_per_gate : (a.width + p.block - 1) / p.block;
  GEARB_REQUIRE(p.tiles <= (int64_t(1) << 31) / ncol - 1, "recurrence: too many tiles for one launch");
  p.ncol = static_cast<int>(ncol);
  p.section_shift = section_shift_of(p);
  const unsigned grid = static_cast<unsigned>(p.tiles * ncol);
  if (p.chain) GEARB_CUDA(cudaMemsetAsync(p.ticket, 0xff, static_cast<size_t>(p.chain_bytes), stream));
  if (backward) backward_kernel<TX, TA, V, kGate, kApart><<<grid, kThreads, 0, stream>>>(p);
  else if constexpr (kGate != kOne) forward_kernel<TX, TA, V, kGate, kApart><<<grid, kThreads, 0, stream>>>(p);
  GEARB_CUDA(cudaGetLastError());
  return GEARB_OK;
}

template <typename TX, typename TA, int V, bool kApart>
int launch_wide_gate(Params &p, bool backward, cudaStream_t stream) {
  if (p.A.gates == p.A.width) return launch_wide<TX, TA, V, kOwn, kApart>(p, backward, stream);
  return p.by_gate ? launch_wide<TX, TA, V, kOne, kApart>(p, backward, stream) : launch_wide<TX, TA, V, kTable, kApart>(p, backward, stream);
}

template <typename TX, typename TA>
int launch_wide_any(Params &p, bool backward, cudaStream_t stream) {
  switch (p.V) {
    case 4: return launch_wide_gate<TX, TA, 4, false>(p, backward, stream);
    case 2:
      return p.apart ? launch_wide_gate<TX, TA, 2, true>(p, backward, stream)
                     : launch_wide_gate<TX, TA, 2, false>(p, backward, stream);
    default: return launch_wide_gate<TX, TA, 1, false>(p, backward, stream);
  }
}

}  // namespace rec
}  // namespace gearb
