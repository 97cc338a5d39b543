// Kernels of the recurrences for rows of few channels (returns, advantages): time goes over the lanes.
//
// A CTA takes a tile of some thousand rows into shared memory (reading and writing memory in order whatever the width),
// and a thread takes K consecutive rows of one channel there; the threads of a warp hold 32 / width such groups, the
// eight warps follow one another.  (A, H) of the groups are joined by a shuffle scan in the warp and one thread per
// channel across the warps; tiles hand their state on as in the other kernels.  Rows are laid out so that the threads
// of a warp, which read K rows apart, fall into different banks: a group's stride is the width modulo 32.
//
// 16384 packed sequences of up to 1000 rows of one channel, 8.6 M rows: 64 us (15 at the copy rate); a warp a row 2300,
// with loads one after the other 203, with the general code for one channel 142.  Issue slots are taken in 51 % of
// the cycles, mostly by the bookkeeping of rows (which start and end a sequence) rather than by the two
// multiply-adds a row; barriers between the phases are the first of the stalls.
#pragma once

#include "recurrence_wide.cuh"

namespace gearb {
namespace rec {

constexpr int kNarrowWidth = 16;

// Where the words of a tile's tensor of `w` values a row lie in shared memory.
struct NarrowLayout {
  int w, stride;  // values a row, floats from one group to the next
  __host__ __device__ constexpr NarrowLayout(int w_, int k)
      : w(w_), stride(w_ == 1 ? k + 1 : k * w_ + ((w_ - k * w_) % 32 + 32) % 32) {}
};
__host__ __device__ inline int narrow_groups(int width) { return 32 / width; }  // of a warp

// Live, start and end bits of K rows.
struct GroupRows {
  unsigned live, start, end;
};
template <int K>
__device__ __forceinline__ GroupRows group_rows_dense(const gearb_recurrence_args &A, int64_t i, int n) {
  GroupRows g = {0, 0, 0};
  if (n <= 0) return g;
  int64_t b = quotient(i, A.time), u = i - b * A.time;
  auto bounds = [&](int64_t &lo, int64_t &hi) {
    int64_t len = A.time;
    if (A.lengths) {
      len = __ldg(A.lengths + (A.reverse ? A.batch - 1 - b : b));
      len = len < 0 ? 0 : (len > A.time ? A.time : len);
    }
    lo = A.reverse ? A.time - len : 0;
    hi = lo + len;
  };
  int64_t lo, hi;
  bounds(lo, hi);
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if (k < n) {
      if (u >= lo && u < hi) g.live |= 1u << k;
      if (u == lo && hi > lo) g.start |= 1u << k;
      if (u == hi - 1 && hi > lo) g.end |= 1u << k;
      if (++u == A.time) {
        u = 0;
        ++b;
        if (k + 1 < n) bounds(lo, hi);
      }
    }
  }
  return g;
}

// The sequence of a live row.  Called where a sequence starts or ends and has a state; out of line, as it would stand in
// the code for every row a thread has.
static __device__ __noinline__ int64_t sequence_of(const gearb_recurrence_args &A, int64_t rows, int64_t i) {
  if (!A.offsets) {
    const int64_t b = quotient(i, A.time);
    return A.reverse ? A.batch - 1 - b : b;
  }
  const ScanOffsets so{A.offsets, rows, A.sequences, A.reverse};
  int64_t lo = 0, hi = A.sequences - 1;  // last sequence that starts at or before the row
  while (lo < hi) {
    const int64_t mid = (lo + hi + 1) >> 1;
    if (so.at(mid) <= i) lo = mid;
    else hi = mid - 1;
  }
  return A.reverse ? A.sequences - 1 - lo : lo;
}

constexpr int kMostNarrowRows = 32 * kWarps * 16;  // width 1, 16 rows a thread

struct NarrowShared {
  unsigned bits[kMostNarrowRows / 32 + 2];  // packed: bit r: a sequence starts (another ends) in front of row r of the tile
  float wa[kWarps][kNarrowWidth], wh[kWarps][kNarrowWidth], wb[kWarps][kNarrowWidth], wc[kWarps][kNarrowWidth];
  int wcut[kWarps], wend[kWarps];
  unsigned ticket;
  int64_t behind;  // packed: first offset behind the tile's first row
  int64_t first, last;  // see forward_kernel and backward_kernel
  int open;
};

// Marks the starts of the packed sequences that fall on the tile's rows or right behind them.  All threads.
__device__ __forceinline__ void mark_starts(const Params &P, NarrowShared &sm, int64_t i0, int64_t i1) {
  const gearb_recurrence_args &A = P.A;
  const ScanOffsets so{A.offsets, P.rows, A.sequences, A.reverse};
  const int n = static_cast<int>(i1 - i0);
  for (int w = threadIdx.x; w < n / 32 + 2; w += kThreads) sm.bits[w] = 0;
  if (threadIdx.x < 32) {
    int64_t s = A.sequences + 1;
    if (i0 < so.at(A.sequences)) s = warp_upper_bound<int64_t>(A.offsets, 0, A.sequences, i0, threadIdx.x, so);
    if (threadIdx.x == 0) sm.behind = s;
  }
  __syncthreads();
  const int64_t s0 = sm.behind;
  if (threadIdx.x == 0 && s0 >= 1 && s0 <= A.sequences && so.at(s0 - 1) == i0) atomicOr(&sm.bits[0], 1u);
  for (int64_t s = s0 + threadIdx.x; s <= A.sequences; s += kThreads) {
    const int64_t o = so.at(s);
    if (o > i1) break;
    if (o >= i0) atomicOr(&sm.bits[(o - i0) >> 5], 1u << ((o - i0) & 31));
  }
  __syncthreads();
}

template <int K>
__device__ __forceinline__ GroupRows group_rows_packed(const Params &P, const NarrowShared &sm, int64_t i0, int at, int n) {
  GroupRows g = {0, 0, 0};
  if (n <= 0) return g;
  const ScanOffsets so{P.A.offsets, P.rows, P.A.sequences, P.A.reverse};
  const int64_t first = so.at(0), total = so.at(P.A.sequences);
  const unsigned here = __funnelshift_r(sm.bits[at >> 5], sm.bits[(at >> 5) + 1], at & 31);  // bits of rows at ...
  const int next = at + 1;
  const unsigned follow = __funnelshift_r(sm.bits[next >> 5], sm.bits[(next >> 5) + 1], next & 31);
  const int64_t before = first - (i0 + at), after = total - (i0 + at);  // rows in front of the first and up to the last sequence
  const int lo = before < 0 ? 0 : (before < n ? static_cast<int>(before) : n);
  const int hi = after < 0 ? 0 : (after < n ? static_cast<int>(after) : n);
  if (hi > lo) g.live = ((1u << hi) - 1u) & ~((1u << lo) - 1u);
  g.start = here & g.live;
  g.end = follow & g.live;
  return g;
}

// Where the values of a tile's rows of one tensor lie, in memory order.
template <int K, bool kOne>
struct NarrowWalk {
  int n, w, stride, reverse;
  unsigned magic;  // e / w for e < 4096, w <= 16
  bool flat;       // one row stride
  int64_t row_low, base, period, sb, sr;
  __device__ __forceinline__ NarrowWalk(const Params &P, int64_t i0, int n_, const NarrowLayout &lay, int64_t period_,
                                        int64_t sb_, int64_t sr_)
      : n(n_), w(lay.w), stride(lay.stride), reverse(P.A.reverse), period(period_), sb(sb_), sr(sr_) {
    row_low = reverse ? P.rows - i0 - n : i0;  // matrix row of the first value
    magic = (0x10000u + w - 1) / w;
    const int64_t first = quotient(row_low, period);
    flat = row_low - first * period + n <= period;
    base = first * sb + (row_low - first * period) * sr;
  }
  // Value e: its word in shared memory, its row in scan order and its place in the row.
  __device__ __forceinline__ int word(int e, int &scan, int &c) const {
    if constexpr (kOne) {
      c = 0;
      scan = reverse ? n - 1 - e : e;
      return scan + scan / K;
    }
    const int r = static_cast<int>((static_cast<unsigned>(e) * magic) >> 16);
    c = e - r * w;
    scan = reverse ? n - 1 - r : r;
    const int g = scan / K;
    return g * stride + (scan - g * K) * w + c;
  }
  // Its element in memory.
  __device__ __forceinline__ int64_t element(int e) const {
    const int r = kOne ? e : static_cast<int>((static_cast<unsigned>(e) * magic) >> 16), c = e - r * w;
    if (flat) return base + r * sr + c;
    const int64_t b = quotient(row_low + r, period);
    return b * sb + (row_low + r - b * period) * sr + c;
  }
};

// Rows into shared memory: 16-byte (or 8-byte) loads where the values follow one another, several loads in flight.
template <typename T, int K, bool kOne, typename F>
__device__ __forceinline__ void load_values(const T *p, const NarrowWalk<K, kOne> &m, float *to, F f) {
  const int total = m.n * m.w;
  int scan, c;
  if (m.flat && m.sr == m.w && reinterpret_cast<uintptr_t>(p + m.base) % (4 * sizeof(T)) == 0) {
    for (int e0 = 4 * threadIdx.x; e0 < total; e0 += 4 * 4 * kThreads) {
      Pack<T, 4> v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (e0 + 4 * u * kThreads + 3 < total) v[u] = load_pack<T, 4>(p + m.base + e0 + 4 * u * kThreads);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int e = e0 + 4 * u * kThreads;
        if (e + 3 < total) {
#pragma unroll
          for (int q = 0; q < 4; ++q) to[m.word(e + q, scan, c)] = f(to_f(v[u].v[q]));
        } else {
          for (int q = e; q < total; ++q) to[m.word(q, scan, c)] = f(to_f(p[m.base + q]));
        }
      }
    }
    return;
  }
  for (int e0 = threadIdx.x; e0 < total; e0 += 8 * kThreads) {
    T v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (e0 + u * kThreads < total) v[u] = p[m.element(e0 + u * kThreads)];
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (e0 + u * kThreads < total) to[m.word(e0 + u * kThreads, scan, c)] = f(to_f(v[u]));
  }
}

// Composition of maps S -> A*S + H over the groups of a warp that are `w` lanes apart; `cut`: the state before plays no part.
struct Group {
  float a, h;
  int cut;
};
__device__ __forceinline__ Group join(const Group &before, const Group &g) {
  return Group{before.a * g.a, g.cut ? g.h : fmaf(g.a, before.h, g.h), g.cut | before.cut};
}

template <typename TX, typename TA, int K, bool kBackward, bool kOne>
__global__ void __launch_bounds__(kThreads, kBackward ? 3 : 4) narrow_kernel(const __grid_constant__ Params P) {
  extern __shared__ float values[];
  __shared__ NarrowShared sm;
  const gearb_recurrence_args &A = P.A;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int w = kOne ? 1 : static_cast<int>(A.width), gates = kOne ? 1 : static_cast<int>(A.gates), per = kOne ? 1 : P.per;
  const int gw = narrow_groups(w);
  using Walk = NarrowWalk<K, kOne>;
  const NarrowLayout xl(w, K), gl(gates, K);
  float *sx = values, *sg = sx + kWarps * gw * xl.stride, *sd = sg + kWarps * gw * gl.stride;

  int64_t tile = blockIdx.x;
  if (P.chain) {
    if (threadIdx.x == 0) sm.ticket = atomicAdd(P.ticket, 1u) + 1u;  // the counter starts at 0xffffffff
    __syncthreads();
    tile = sm.ticket;
  }
  const int64_t at_tile = tile;  // in the order of the tickets
  if (kBackward) tile = P.tiles - 1 - tile;
  const int64_t i0 = tile * P.tile_rows, i1 = i0 + P.tile_rows < P.rows ? i0 + P.tile_rows : P.rows;
  const int n = static_cast<int>(i1 - i0);

  auto same = [](float v) { return v; };
  load_values(static_cast<const TX *>(A.x), Walk(P, i0, n, xl, P.x_period, A.x_batch_stride, A.x_row_stride), sx, same);
  load_values(static_cast<const TA *>(A.gate), Walk(P, i0, n, gl, P.gate_period, A.gate_batch_stride, A.gate_row_stride),
              sg, [&](float v) { return A.gate_log ? exp_of(v) : v; });
  if (kBackward)
    load_values(static_cast<const TX *>(A.dout),
                Walk(P, i0, n, xl, P.dout_period, A.dout_batch_stride, A.dout_row_stride), sd, same);
  if (A.offsets) mark_starts(P, sm, i0, i1);

  // this thread's rows
  const int gi = lane / w, c = lane - gi * w, g = warp * gw + gi, at = g * K;
  const int mine = gi < gw ? (n - at < 0 ? 0 : (n - at < K ? n - at : K)) : 0;
  const GroupRows m = A.offsets ? group_rows_packed<K>(P, sm, i0, at, mine) : group_rows_dense<K>(A, i0 + at, mine);
  __syncthreads();

  const float *px = sx + g * xl.stride + c, *pg = sg + g * gl.stride + c / per;
  float *pd = sd + g * xl.stride + c;
  float h0v = 0.0f;  // of the last start looked at
  auto first_state = [&](const float *p, int k) { return p ? p[sequence_of(A, P.rows, i0 + at + k) * w + c] : 0.0f; };
  Group f{1.0f, 0.0f, m.start != 0}, b{1.0f, 0.0f, m.end != 0};
  // Without states of their own sequences start from nothing: no branches (0 * -0 + x is x, to the sign of a zero).  (What a row of no sequence leaves is not
  // used: the next row of one is its first.)
  const bool stateless = !A.h0 && !(kBackward ? A.dstate : nullptr);
  if (stateless && mine > 0) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const bool st = m.start >> k & 1u;
      const float a = pg[k * gates];
      f.h = fmaf(st ? 0.0f : a, st ? -0.0f : f.h, px[k * w]);
      f.a *= a;
    }
  } else {
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if (!(m.live >> k & 1u)) continue;
    const float a = pg[k * gates], x = px[k * w];
    if (m.start >> k & 1u) {
      h0v = first_state(A.h0, k);
      f.h = A.h0 ? fmaf(a, h0v, x) : x;
    } else {
      f.h = fmaf(a, f.h, x);
    }
    f.a *= a;
  }
  }
  if (kBackward) {
    b.a = f.a;
#pragma unroll
    for (int k = K - 1; k >= 0; --k) {
      if (!(m.live >> k & 1u)) continue;
      if (m.end >> k & 1u) b.h = first_state(A.dstate, k);
      b.h = pg[k * gates] * (pd[k * w] + b.h);
    }
  }
  // over the groups of the warp, then what lies before (backward: behind) this one in it
  Group fi = f, bi = b;
  for (int d = w; d < gw * w; d <<= 1) {
    Group u{__shfl_up_sync(kAll, fi.a, d), __shfl_up_sync(kAll, fi.h, d), __shfl_up_sync(kAll, fi.cut, d)};
    if (lane >= d) fi = join(u, fi);
    if (kBackward) {
      Group v{__shfl_down_sync(kAll, bi.a, d), __shfl_down_sync(kAll, bi.h, d), __shfl_down_sync(kAll, bi.cut, d)};
      if (lane + d < gw * w) bi = join(v, bi);
    }
  }
  Group fx{__shfl_up_sync(kAll, fi.a, w), __shfl_up_sync(kAll, fi.h, w), __shfl_up_sync(kAll, fi.cut, w)};
  Group bx{__shfl_down_sync(kAll, bi.a, w), __shfl_down_sync(kAll, bi.h, w), __shfl_down_sync(kAll, bi.cut, w)};
  if (gi == 0) fx = Group{1.0f, 0.0f, 0};
  if (gi == gw - 1) bx = Group{1.0f, 0.0f, 0};
  if (gi == gw - 1) {
    sm.wa[warp][c] = fi.a;
    sm.wh[warp][c] = fi.h;
    if (c == 0) sm.wcut[warp] = fi.cut;
  }
  if (kBackward && gi == 0) {
    sm.wb[warp][c] = bi.a;
    sm.wc[warp][c] = bi.h;
    if (c == 0) sm.wend[warp] = bi.cut;
  }
  // whether the tile's first and last row belong to sequences that go on elsewhere, and how far
  if (threadIdx.x == 0) {
    int64_t from = -1;
    if (m.live & ~m.start & 1u) {
      if (A.offsets) {
        const ScanOffsets so{A.offsets, P.rows, A.sequences, A.reverse};
        from = so.at(sm.behind - 1);
      } else {
        const int64_t q = quotient(i0, A.time);
        from = q * A.time;
        if (A.lengths && A.reverse) {
          const int64_t len = __ldg(A.lengths + (A.batch - 1 - q));
          from += A.time - (len > A.time ? A.time : len);
        }
      }
    }
    sm.first = from < 0 || from > i0 ? -1 : from;
    sm.open = sm.first >= 0 && quotient(sm.first, P.tile_rows) < tile;
  }
  if (kBackward && mine > 0 && at + mine == n && c == 0) {
    int64_t to = -1;
    if ((m.live & ~m.end) >> (mine - 1) & 1u) {
      const int64_t i = i1 - 1;
      if (A.offsets) {
        const ScanOffsets so{A.offsets, P.rows, A.sequences, 0};
        const int64_t s = sequence_of(A, P.rows, i);
        to = A.reverse ? P.rows - so.at(s) - 1 : so.at(s + 1) - 1;
      } else {
        const int64_t q = quotient(i, A.time);
        to = (q + 1) * A.time - 1;
        if (A.lengths && !A.reverse) {
          const int64_t len = __ldg(A.lengths + q);
          to = q * A.time + (len > A.time ? A.time : len) - 1;
        }
      }
    }
    sm.last = to < i1 || to >= P.rows ? -1 : to;
  }
  __syncthreads();

  // across the warps: one thread per channel, backward ones from thread 32 on
  if (threadIdx.x < w) {
    const int ch = threadIdx.x;
    float pa[kWarps], ph[kWarps], in = 0.0f;
    int cut[kWarps];
    Group t{1.0f, 0.0f, 0};
#pragma unroll
    for (int q = 0; q < kWarps; ++q) {
      pa[q] = t.a;
      ph[q] = t.h;
      cut[q] = t.cut;
      t = join(t, Group{sm.wa[q][ch], sm.wh[q][ch], sm.wcut[q]});
    }
    if (P.chain) {
      if (!kBackward) {
        publish_pair(P.agg + tile * w + ch, t.a, t.h);
        bool lost = false;
        in = look_back<4, 0, int64_t>(P, tile, sm.open ? quotient(sm.first, P.tile_rows) : tile, ch,
                                   [&] { return make_float2(t.a, t.h); }, t.cut != 0, lost);
        if (lost && A.status) atomicOr(reinterpret_cast<unsigned *>(A.status), GEARB_ST_SCAN_ABORTED);
        if (sm.open && A.carry) A.carry[tile * w + ch] = in;
      } else if (sm.open) {
        in = __ldg(A.carry + tile * w + ch);
      }
    }
#pragma unroll
    for (int q = 0; q < kWarps; ++q) sm.wh[q][ch] = cut[q] ? ph[q] : fmaf(pa[q], in, ph[q]);
  }
  if (kBackward && threadIdx.x >= 32 && threadIdx.x < 32 + w) {
    const int ch = threadIdx.x - 32;
    float pa[kWarps], ph[kWarps], in = 0.0f;
    int cut[kWarps];
    Group t{1.0f, 0.0f, 0};
#pragma unroll
    for (int q = kWarps - 1; q >= 0; --q) {
      pa[q] = t.a;
      ph[q] = t.h;
      cut[q] = t.cut;
      t = join(t, Group{sm.wb[q][ch], sm.wc[q][ch], sm.wend[q]});
    }
    if (P.chain) {
      publish_pair(P.agg + at_tile * w + ch, t.a, t.h);
      const int64_t lo = sm.last >= 0 ? P.tiles - 1 - quotient(sm.last, P.tile_rows) : at_tile;
      bool lost = false;
      in = look_back<4, 0, int64_t>(P, at_tile, lo < at_tile ? lo : at_tile, ch, [&] { return make_float2(t.a, t.h); },
                                 t.cut != 0, lost);
      if (lost && A.status) atomicOr(reinterpret_cast<unsigned *>(A.status), GEARB_ST_SCAN_ABORTED);
    }
#pragma unroll
    for (int q = 0; q < kWarps; ++q) sm.wc[q][ch] = cut[q] ? ph[q] : fmaf(pa[q], in, ph[q]);
  }
  __syncthreads();

  // this thread's rows again
  if (mine > 0) {
    float h = fx.cut ? fx.h : fmaf(fx.a, sm.wh[warp][c], fx.h);
    float *ox = sx + g * xl.stride + c;
    if (!kBackward && stateless && !A.state_out) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const bool st = m.start >> k & 1u;
        h = fmaf(st ? 0.0f : pg[k * gates], st ? -0.0f : h, px[k * w]);
        ox[k * w] = (m.live >> k & 1u) ? h : 0.0f;
      }
    } else if (!kBackward) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const float a = pg[k * gates], x = px[k * w];
        const bool st = m.start >> k & 1u;
        if (st && A.h0) h0v = first_state(A.h0, k);
        if (m.live >> k & 1u) h = st ? (A.h0 ? fmaf(a, h0v, x) : x) : fmaf(a, h, x);
        if (k < mine) ox[k * w] = (m.live >> k & 1u) ? h : 0.0f;
        if ((m.end >> k & 1u) && A.state_out) A.state_out[sequence_of(A, P.rows, i0 + at + k) * w + c] = h;
      }
    } else {
      float hp[K], cb = bx.cut ? bx.h : fmaf(bx.a, sm.wc[warp][c], bx.h);
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const float a = pg[k * gates], x = px[k * w];
        const bool st = m.start >> k & 1u;
        if (st) h = first_state(A.h0, k);
        hp[k] = (st && !A.h0) ? 0.0f : h;
        if (m.live >> k & 1u) h = (st && !A.h0) ? x : fmaf(a, h, x);
      }
#pragma unroll
      for (int k = K - 1; k >= 0; --k) {
        const float a = pg[k * gates];
        const bool lv = m.live >> k & 1u, st = m.start >> k & 1u;
        if (m.end >> k & 1u) cb = first_state(A.dstate, k);
        const float gr = lv ? pd[k * w] + cb : 0.0f;
        if (lv) cb = a * gr;
        if (k < mine) {
          pd[k * w] = gr;
          // the first row of a sequence without h0 is h = x: its gate plays no part
          ox[k * w] = (lv && !(st && !A.h0)) ? (A.gate_log ? cb : gr) * hp[k] : 0.0f;
        }
        if (st && A.dh0) A.dh0[sequence_of(A, P.rows, i0 + at + k) * w + c] = cb;
      }
    }
  }
  __syncthreads();

  // out in memory order; rows of no sequence hold zeros, or are left as they are
  auto owned = [&](int scan) {
    const int64_t i = i0 + scan;
    if (A.offsets) {
      const ScanOffsets so{A.offsets, P.rows, A.sequences, A.reverse};
      return i >= so.at(0) && i < so.at(A.sequences);
    }
    if (!A.lengths) return true;
    const int64_t row = row_of(P, i), b0 = quotient(row, A.time);
    return row - b0 * A.time < __ldg(A.lengths + b0);
  };
  const Walk xw(P, i0, n, xl, P.rows, 0, w), gwalk(P, i0, n, gl, P.rows, 0, gates);
  TX *to = static_cast<TX *>(kBackward ? A.dx : A.out) + xw.base;
  const float *from = kBackward ? sd : sx;
  int scan, ch;
#pragma unroll 4
  for (int e = threadIdx.x; e < n * w; e += kThreads) {
    const float v = from[xw.word(e, scan, ch)];
    if (A.zero_rest || owned(scan)) to[e] = from_f<TX>(v);
  }
  if (kBackward) {
    TA *dg = static_cast<TA *>(A.dgate) + gwalk.base;
    for (int e = threadIdx.x; e < n * gates; e += kThreads) {
      gwalk.word(e, scan, ch);
      if (!A.zero_rest && !owned(scan)) continue;
      const int gg = scan / K;
      const float *p = sx + gg * xl.stride + (scan - gg * K) * w + ch * per;
      float sum = 0.0f;
      for (int v = 0; v < per; ++v) sum += p[v];
      dg[e] = from_f<TA>(sum);
    }
  }
  empty_sequences(P, Place{tile, i0, i1, 0, 0, w, 0}, w, kBackward ? A.dstate : A.h0, kBackward ? A.dh0 : A.state_out);
}

template <typename TX, typename TA, int K>
int launch_narrow(Params &p, bool backward, cudaStream_t stream) {
  const int w = static_cast<int>(p.A.width), groups = kWarps * narrow_groups(w);
  const NarrowLayout xl(w, K), gl(static_cast<int>(p.A.gates), K);
  const int smem = groups * ((backward ? 2 : 1) * xl.stride + gl.stride) * 4;
  GEARB_REQUIRE(p.tiles < (int64_t(1) << 31), "recurrence: too many tiles for one launch");
  p.ncol = 1;
  p.section_shift = section_shift_of(p);
  p.blocks_per_gate = 1;
  if (p.chain) GEARB_CUDA(cudaMemsetAsync(p.ticket, 0xff, static_cast<size_t>(p.chain_bytes), stream));
  void (*kernel)(Params);
  if (w == 1) kernel = backward ? narrow_kernel<TX, TA, K, true, true> : narrow_kernel<TX, TA, K, false, true>;
  else kernel = backward ? narrow_kernel<TX, TA, K, true, false> : narrow_kernel<TX, TA, K, false, false>;
  if (smem > 40 * 1024) GEARB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  kernel<<<static_cast<unsigned>(p.tiles), kThreads, smem, stream>>>(p);
  GEARB_CUDA(cudaGetLastError());
  return GEARB_OK;
}

}  // namespace rec
}  // namespace gearb
