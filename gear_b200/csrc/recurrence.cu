// Linear recurrences over sequences, forward and backward.
//
//   h_t = a_t * h_(t-1) + x_t                      h_(-1) = h0
//   g_t = dh_t + a_(t+1) * g_(t+1)                 g_last = dh_last + dstate
//   dx_t = g_t,  da_t = sum over the gate's channels of g_t * h_(t-1),  dh0 = a_0 * g_0
//
// with a_t = gate, or exp(gate) (then dgate = da * a).
//
// Any run of rows maps the state before it to the state behind it as S -> A*S + H (A the product of its a_t,
// H its own result from zero), and such maps compose, so rows can be worked on in parallel: all rows of a call,
// sequence after sequence, are cut into tiles of 64; a CTA takes one tile and one block of channels, keeps
// gate and x in registers (8 rows a warp, one channel or a few a lane), forms (A, H), learns the state before
// its tile, and runs its rows again from there.  Every input is read once and every output written once.
//
// The state before a tile.  Tiles publish their (A, H); 16 consecutive tiles form a superblock, and the last
// tile of one publishes the state behind it.  A tile composes the tiles before it in its superblock, in
// order, onto the state in front of the superblock: the same operations whatever the timing, so results are the
// same bits every time, and the chain of waiting CTAs has one link per 1024 rows.  A tile needs nothing from
// before the start of the sequence its first row belongs to.  Tiles are handed out by a counter in scan order,
// so a CTA only ever waits for CTAs that are already running; every wait has a limit, after which the
// launch goes on with NaN and says so in the status word.  Published words are 32 bits that read
// 0xffffffff until they are written (a value of those bits is published as another NaN), so no flags and
// fences are needed beside them.
//
// Backward.  In terms of c_t = a_t * g_t the gradients obey c_t = a_t * c_(t+1) + a_t * dh_t, the same
// recurrence from the last row to the first, over the same tiles.  h_(t-1) is not read back (it was rounded to
// x's type) but formed again in float32 from x, gate and the state before the tile, which the forward
// pass leaves in `carry`.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.h"
#include "warp_search.cuh"

namespace gearb {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kRows = 8;                     // rows a warp keeps in registers
constexpr int kTile = kWarps * kRows;        // rows per tile
constexpr int kSuper = 16;                   // tiles per superblock
constexpr unsigned kAll = 0xffffffffu;
constexpr unsigned kUnset = 0xffffffffu;     // a published word that has not been written
constexpr int kPollLimit = 1 << 20;          // polls of one word, the better part of a second

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f(float v) { return v; }
template <> __device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f(float v) { return v; }
template <> __device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }

// V consecutive values of T, loaded and stored as one access.
template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
  T v[V];
};
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T *p) {
  constexpr int kBytes = sizeof(T) * V;
  Pack<T, V> r;
  if constexpr (kBytes == 16) {
    *reinterpret_cast<uint4 *>(&r) = __ldcs(reinterpret_cast<const uint4 *>(p));
  } else if constexpr (kBytes == 8) {
    *reinterpret_cast<uint2 *>(&r) = __ldcs(reinterpret_cast<const uint2 *>(p));
  } else if constexpr (kBytes == 4) {
    *reinterpret_cast<unsigned *>(&r) = __ldcs(reinterpret_cast<const unsigned *>(p));
  } else {
    *reinterpret_cast<unsigned short *>(&r) = __ldcs(reinterpret_cast<const unsigned short *>(p));
  }
  return r;
}
template <typename T, int V>
__device__ __forceinline__ void store_pack(T *p, const float (&f)[V]) {
  Pack<T, V> r;
#pragma unroll
  for (int v = 0; v < V; ++v) r.v[v] = from_f<T>(f[v]);
  *reinterpret_cast<Pack<T, V> *>(p) = r;
}

// What the kernels need beyond the caller's arguments.
struct Params {
  gearb_recurrence_args A;
  int64_t rows;
  int64_t tiles;
  int tile_rows;         // kTile, or the largest multiple of `time` below it when tiles then need nothing from each other
  int chain;             // tiles publish to each other
  int per;               // channels per gate
  int blocks_per_gate;   // column blocks of a gate's channels (shared gates)
  int ncol;              // column blocks
  // Address periods: rows per batch entry, or all rows where one row stride covers the whole batch.
  int64_t x_period, gate_period, dout_period;
  unsigned *ticket;
  float2 *agg;           // [tiles][width]: (A, H) of every tile
  float *super;          // [superblocks][width]: state in front of every superblock
  float *gate_part;      // [blocks_per_gate][rows][gates], when a gate's channels span several column blocks
};

__device__ __forceinline__ unsigned poll_word(const unsigned *p, bool &lost) {
  unsigned v;
  for (int n = 0;; ++n) {
    asm volatile("ld.relaxed.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    if (v != kUnset) return v;
    if (lost || n == kPollLimit) break;
    __nanosleep(20);
  }
  lost = true;
  return 0x7fffffffu;  // NaN
}
__device__ __forceinline__ float2 poll_pair(const float2 *p, bool &lost) {
  unsigned a, h;
  for (int n = 0;; ++n) {
    asm volatile("ld.relaxed.gpu.global.v2.u32 {%0,%1}, [%2];" : "=r"(a), "=r"(h) : "l"(p) : "memory");
    if (a != kUnset && h != kUnset) return make_float2(__uint_as_float(a), __uint_as_float(h));
    if (lost || n == kPollLimit) break;
    __nanosleep(20);
  }
  lost = true;
  return make_float2(__uint_as_float(0x7fffffffu), __uint_as_float(0x7fffffffu));
}
__device__ __forceinline__ unsigned word_of(float v) {
  const unsigned u = __float_as_uint(v);
  return u == kUnset ? 0x7fffffffu : u;
}
__device__ __forceinline__ void publish_pair(float2 *p, float a, float h) {
  asm volatile("st.relaxed.gpu.global.v2.u32 [%0], {%1,%2};" ::"l"(p), "r"(word_of(a)), "r"(word_of(h)) : "memory");
}
__device__ __forceinline__ void publish_word(float *p, float v) {
  asm volatile("st.relaxed.gpu.global.u32 [%0], %1;" ::"l"(p), "r"(word_of(v)) : "memory");
}

// Offset s of the packed sequences in scan order: as given, or mirrored for a reverse call.  Kept inside the rows.
struct ScanOffsets {
  const int64_t *off;
  int64_t rows, n;
  int reverse;
  __device__ __forceinline__ int64_t at(int64_t s) const {
    int64_t v = __ldg(off + (reverse ? n - s : s));
    v = v < 0 ? 0 : (v > rows ? rows : v);
    return reverse ? rows - v : v;
  }
  // For warp_upper_bound, which walks a pointer.
  __device__ __forceinline__ int64_t operator()(const int64_t *p) const { return at(p - off); }
};

// Rows [i0, i0 + n) of the scan as one warp sees them; row k is bit k.  Lane k holds the sequence of row k.
struct RowMap {
  unsigned live, start, end;
  int seq;
  int64_t first_start;  // scan index at which the sequence of row i0 starts
  int64_t last_end;     // scan index at which the sequence of row i0 + n - 1 ends
};

__device__ __forceinline__ RowMap map_rows(const gearb_recurrence_args &A, int64_t rows, int64_t i0, int n, int lane) {
  RowMap m;
  m.seq = 0;
  m.first_start = m.last_end = 0;
  const int64_t i = i0 + lane;
  bool live = lane < n, start = false, end = false;
  if (!A.offsets) {
    int64_t s0 = 0, s1 = 0;
    if (live) {
      const int64_t b = i / A.time, u = i - b * A.time;
      const int64_t seq = A.reverse ? A.batch - 1 - b : b;
      int64_t len = A.time;
      if (A.lengths) {
        len = __ldg(A.lengths + seq);
        len = len < 0 ? 0 : (len > A.time ? A.time : len);
      }
      const int64_t lo = A.reverse ? A.time - len : 0;  // first live row of this batch entry, in scan order
      live = u >= lo && u < lo + len;
      start = live && u == lo;
      end = live && u == lo + len - 1;
      m.seq = static_cast<int>(seq);
      s0 = i - u + lo;
      s1 = s0 + len - 1;
    }
    m.first_start = __shfl_sync(kAll, s0, 0);
    m.last_end = __shfl_sync(kAll, s1, n > 0 ? n - 1 : 0);
  } else {
    const ScanOffsets so{A.offsets, rows, A.sequences, A.reverse};
    const int64_t total = so.at(A.sequences);
    live = live && i < total;
    int64_t my_seq = -1, my_start = 0, my_end = 0;
    if (n > 0 && i0 < total) {
      int64_t s = warp_upper_bound<int64_t>(A.offsets, 0, A.sequences, i0, lane, so);  // first offset behind row i0
      int64_t before = s > 0 ? so.at(s - 1) : -1;  // the offset in front of the window; -1: rows of no sequence
      bool settled = lane >= n;
      for (;;) {  // 32 offsets at a time: one round unless many sequences end within these rows
        const int64_t b = s + lane <= A.sequences ? so.at(s + lane) : rows + 1;
        int count = 0;  // offsets of the window at or before this lane's row
        for (int k = 0; k < n; ++k) {
          const unsigned c = __ballot_sync(kAll, b <= i0 + k);
          if (lane == k) count = __popc(c);
        }
        const int64_t st = __shfl_sync(kAll, b, count > 0 ? count - 1 : 0);
        const int64_t nx = __shfl_sync(kAll, b, count < 32 ? count : 31);
        if (!settled && count < 32) {
          settled = true;
          my_seq = s + count - 1;
          my_start = count > 0 ? st : before;
          my_end = nx;
        }
        if (__all_sync(kAll, settled)) break;
        before = __shfl_sync(kAll, b, 31);
        s += 32;
      }
    }
    live = live && my_seq >= 0;
    start = live && my_start == i;
    end = live && my_end == i + 1;
    // offsets that do not ascend give nonsense, but nothing outside the rows
    if (my_start > i || my_start < 0) my_start = i;
    if (my_end <= i || my_end > rows) my_end = i + 1;
    m.seq = live ? static_cast<int>(A.reverse ? A.sequences - 1 - my_seq : my_seq) : 0;
    m.first_start = __shfl_sync(kAll, my_start, 0);
    m.last_end = __shfl_sync(kAll, my_end - 1, n > 0 ? n - 1 : 0);
  }
  m.live = __ballot_sync(kAll, live);
  m.start = __ballot_sync(kAll, start && live);
  m.end = __ballot_sync(kAll, end && live);
  return m;
}

// Element offset of consecutive rows of the scan in one tensor.
struct RowWalk {
  int64_t off, t, period, step, wrap;
  int reverse;
  __device__ __forceinline__ RowWalk(int64_t row, int64_t period_, int64_t sb, int64_t sr, int reverse_)
      : period(period_), reverse(reverse_) {
    const int64_t b = row / period;
    t = row - b * period;
    off = b * sb + t * sr;
    step = reverse ? -sr : sr;
    wrap = reverse ? period * sr - sb : sb - period * sr;
  }
  __device__ __forceinline__ void next() {
    off += step;
    if (reverse) {
      if (t-- == 0) {
        t = period - 1;
        off += wrap;
      }
    } else if (++t == period) {
      t = 0;
      off += wrap;
    }
  }
};

__device__ __forceinline__ int64_t row_of(const Params &P, int64_t i) { return P.A.reverse ? P.rows - 1 - i : i; }

// The CTA's tile and column block.
struct Place {
  int64_t tile;
  int64_t i0, i1;  // rows of the scan
  int64_t gate;    // shared gates: the gate of this column block
  int64_t d0, d1;  // channels
  int part;        // which column block of the gate
};

template <int V, bool kShared>
__device__ __forceinline__ Place take_place(const Params &P, unsigned *smem_ticket, bool backward) {
  int64_t item;
  if (P.chain) {
    if (threadIdx.x == 0) *smem_ticket = atomicAdd(P.ticket, 1u) + 1u;  // the counter starts at 0xffffffff
    __syncthreads();
    item = *smem_ticket;
  } else {
    item = blockIdx.x;
  }
  Place p;
  const int64_t t = item / P.ncol;
  const int c = static_cast<int>(item - t * P.ncol);
  p.tile = backward ? P.tiles - 1 - t : t;
  p.i0 = p.tile * P.tile_rows;
  p.i1 = p.i0 + P.tile_rows < P.rows ? p.i0 + P.tile_rows : P.rows;
  if (kShared) {
    p.gate = c / P.blocks_per_gate;
    p.part = c - static_cast<int>(p.gate) * P.blocks_per_gate;
    p.d0 = p.gate * P.per + static_cast<int64_t>(p.part) * 32 * V;
    p.d1 = (p.gate + 1) * P.per;
  } else {
    p.gate = 0;
    p.part = 0;
    p.d0 = static_cast<int64_t>(c) * 32 * V;
    p.d1 = P.A.width;
  }
  return p;
}

// gate of 8 rows, as a_t, for this lane's channels: one value a row when it is shared by them.
template <typename TA, int V, bool kShared>
__device__ __forceinline__ void load_gate(const Params &P, const Place &pl, int64_t i0, int n, int64_t d, bool on,
                                          float (&a)[kRows][kShared ? 1 : V]) {
  constexpr int kG = kShared ? 1 : V;
  const TA *gate = static_cast<const TA *>(P.A.gate) + (kShared ? pl.gate : d);
  if (n > 0) {
    RowWalk w(row_of(P, i0), P.gate_period, P.A.gate_batch_stride, P.A.gate_row_stride, P.A.reverse);
    Pack<TA, kG> raw[kRows];
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      if (k < n && (kShared || on)) raw[k] = load_pack<TA, kG>(gate + w.off);
      w.next();
    }
#pragma unroll
    for (int k = 0; k < kRows; ++k)
#pragma unroll
      for (int v = 0; v < kG; ++v) a[k][v] = (k < n && (kShared || on)) ? to_f(raw[k].v[v]) : 0.0f;
  } else {
#pragma unroll
    for (int k = 0; k < kRows; ++k)
#pragma unroll
      for (int v = 0; v < kG; ++v) a[k][v] = 0.0f;
  }
}

template <typename T, int V>
__device__ __forceinline__ void load_rows(const T *base, int64_t row0, int64_t period, int64_t sb, int64_t sr, int reverse,
                                          int n, int64_t d, bool on, Pack<T, V> (&r)[kRows]) {
  RowWalk w(row0, period, sb, sr, reverse);
#pragma unroll
  for (int k = 0; k < kRows; ++k) {
    if (k < n && on) r[k] = load_pack<T, V>(base + w.off + d);
    else
#pragma unroll
      for (int v = 0; v < V; ++v) r[k].v[v] = from_f<T>(0.0f);
    w.next();
  }
}

// The state in front of the tile, from what the tiles before it (in scan order, or behind it in a backward pass:
// `at` counts them in the order of their tickets) have published.  lo: the first of them that matters.
template <int V>
struct Carry {
  float pa[kSuper][32 * V], ph[kSuper][32 * V], ps[32 * V];
};
template <int V>
__device__ __forceinline__ void look_back(const Params &P, Carry<V> &sm, int64_t at, int64_t lo, int64_t d, bool on, int lane,
                                          int warp, float (&cin)[V], bool &lost) {
  const int64_t sb = at / kSuper, sb0 = sb * kSuper;
  const bool need_super = lo < sb0;
  const int64_t j0 = need_super ? sb0 : lo;
  if (on) {
    for (int64_t j = j0 + warp; j < at; j += kWarps) {
      const float2 *p = P.agg + j * P.A.width + d;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float2 q = poll_pair(p + v, lost);
        sm.pa[j - j0][lane * V + v] = q.x;
        sm.ph[j - j0][lane * V + v] = q.y;
      }
    }
    if (need_super && warp == kWarps - 1) {
#pragma unroll
      for (int v = 0; v < V; ++v)
        sm.ps[lane * V + v] = __uint_as_float(
            poll_word(reinterpret_cast<const unsigned *>(P.super + sb * P.A.width + d + v), lost));
    }
  }
  __syncthreads();
#pragma unroll
  for (int v = 0; v < V; ++v) {
    float s = need_super ? sm.ps[lane * V + v] : sm.ph[0][lane * V + v];
    for (int64_t j = need_super ? j0 : j0 + 1; j < at; ++j)
      s = fmaf(sm.pa[j - j0][lane * V + v], s, sm.ph[j - j0][lane * V + v]);
    cin[v] = s;
  }
}

// Hands a sequence without rows its state (forward) or its gradient (backward): the CTAs of a launch share the
// sequences among them.
template <int V>
__device__ __forceinline__ void empty_sequences(const Params &P, const Place &pl, const float *from, float *to) {
  const gearb_recurrence_args &A = P.A;
  if (!to) return;
  const int64_t step = P.tiles * kThreads;
  for (int64_t s = pl.tile * kThreads + threadIdx.x; s < A.sequences; s += step) {
    int64_t n;
    if (A.offsets) {
      const ScanOffsets so{A.offsets, P.rows, A.sequences, 0};
      n = so.at(s + 1) - so.at(s);
    } else {
      n = A.lengths ? __ldg(A.lengths + s) : A.time;
    }
    if (n > 0) continue;
    const int64_t d1 = pl.d0 + 32 * V < pl.d1 ? pl.d0 + 32 * V : pl.d1;
    for (int64_t d = pl.d0; d < d1; ++d) to[s * A.width + d] = from ? from[s * A.width + d] : 0.0f;
  }
}

template <typename TX, typename TA, int V, bool kShared>
__global__ void __launch_bounds__(kThreads) forward_kernel(const __grid_constant__ Params P) {
  constexpr int kG = kShared ? 1 : V;
  __shared__ float sa[kWarps][32 * V], sh[kWarps][32 * V];
  __shared__ int scut[kWarps];
  __shared__ unsigned sticket;
  __shared__ int64_t sfirst;  // scan index at which the first row's sequence starts, or -1: nothing is needed from before
  __shared__ Carry<V> scarry;
  const gearb_recurrence_args &A = P.A;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Place pl = take_place<V, kShared>(P, &sticket, false);
  const int64_t d = pl.d0 + lane * V;
  const bool on = d < pl.d1;
  const int64_t i0 = pl.i0 + warp * kRows;
  const int n = static_cast<int>(i0 >= pl.i1 ? 0 : (pl.i1 - i0 < kRows ? pl.i1 - i0 : kRows));

  Pack<TX, V> x[kRows];
  float a[kRows][kG];
  if (n > 0)
    load_rows<TX, V>(static_cast<const TX *>(A.x), row_of(P, i0), P.x_period, A.x_batch_stride, A.x_row_stride, A.reverse, n,
                     d, on, x);
  load_gate<TA, V, kShared>(P, pl, i0, n, d, on, a);
  const RowMap m = map_rows(A, P.rows, i0, n, lane);
  if (A.gate_log) {
#pragma unroll
    for (int k = 0; k < kRows; ++k)
#pragma unroll
      for (int v = 0; v < kG; ++v) a[k][v] = expf(a[k][v]);
  }

  // (A, H) of this warp's rows; behind a start only H counts
  float ca[V], ch[V], first[V];  // first: h of the last start row, see below
#pragma unroll
  for (int v = 0; v < V; ++v) { ca[v] = 1.0f; ch[v] = first[v] = 0.0f; }
#pragma unroll
  for (int k = 0; k < kRows; ++k) {
    if (!(m.live >> k & 1u)) continue;
    if (m.start >> k & 1u) {
      const int seq = __shfl_sync(kAll, m.seq, k);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float xv = to_f(x[k].v[v]);
        ch[v] = first[v] = (A.h0 && on) ? fmaf(a[k][kShared ? 0 : v], A.h0[static_cast<int64_t>(seq) * A.width + d + v], xv) : xv;
      }
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float av = a[k][kShared ? 0 : v];
        ch[v] = fmaf(av, ch[v], to_f(x[k].v[v]));
        ca[v] *= av;
      }
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) { sa[warp][lane * V + v] = ca[v]; sh[warp][lane * V + v] = ch[v]; }
  if (lane == 0) {
    scut[warp] = m.start != 0;
    if (warp == 0) sfirst = ((m.live & ~m.start) & 1u) ? m.first_start : -1;
  }
  __syncthreads();

  // of the warps before this one
  float pa[V], ph[V];
  bool cut = false;
#pragma unroll
  for (int v = 0; v < V; ++v) { pa[v] = 1.0f; ph[v] = 0.0f; }
  for (int q = 0; q < warp; ++q) {
    const bool c = scut[q];
    cut |= c;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float h = sh[q][lane * V + v], b = sa[q][lane * V + v];
      ph[v] = c ? h : fmaf(b, ph[v], h);
      pa[v] *= b;
    }
  }
  float ta[V], th[V];  // of the whole tile (last warp)
  const bool tcut = cut || m.start != 0;
  if (P.chain && warp == kWarps - 1) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      th[v] = m.start != 0 ? ch[v] : fmaf(ca[v], ph[v], ch[v]);
      ta[v] = pa[v] * ca[v];
      if (on) publish_pair(P.agg + pl.tile * A.width + d + v, ta[v], th[v]);
    }
  }
  float cin[V];
#pragma unroll
  for (int v = 0; v < V; ++v) cin[v] = 0.0f;
  const int64_t lo = sfirst / P.tile_rows;
  if (P.chain && sfirst >= 0 && lo < pl.tile) {
    bool lost = false;
    look_back<V>(P, scarry, pl.tile, lo, d, on, lane, warp, cin, lost);
    if (lost && A.status) atomicOr(reinterpret_cast<unsigned *>(A.status), GEARB_ST_SCAN_ABORTED);
    if (A.carry && warp == 0 && on)
#pragma unroll
      for (int v = 0; v < V; ++v) A.carry[pl.tile * A.width + d + v] = cin[v];
  }
  if (P.chain && warp == kWarps - 1 && pl.tile % kSuper == kSuper - 1 && pl.tile + 1 < P.tiles && on) {
#pragma unroll
    for (int v = 0; v < V; ++v)
      publish_word(P.super + (pl.tile / kSuper + 1) * A.width + d + v, tcut ? th[v] : fmaf(ta[v], cin[v], th[v]));
  }

  if (n > 0) {
    float h[V];
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = cut ? ph[v] : fmaf(pa[v], cin[v], ph[v]);
    TX *out = static_cast<TX *>(A.out) + d;
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      if (k >= n) break;
      const int64_t row = row_of(P, i0 + k);
      if (!(m.live >> k & 1u)) {
        if (A.zero_rest && on) {
          const float z[V] = {};
          store_pack<TX, V>(out + row * A.width, z);
        }
        continue;
      }
      const int seq = __shfl_sync(kAll, m.seq, k);
      if (m.start >> k == 1u) {
        // The sequence may end in another warp or tile, which may by now have put its state where h0 was
        // (state_out may be h0): h of this row is kept from the first look at it.
#pragma unroll
        for (int v = 0; v < V; ++v) h[v] = first[v];
      } else if (m.start >> k & 1u) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float xv = to_f(x[k].v[v]);
          h[v] = (A.h0 && on) ? fmaf(a[k][kShared ? 0 : v], A.h0[static_cast<int64_t>(seq) * A.width + d + v], xv) : xv;
        }
      } else {
#pragma unroll
        for (int v = 0; v < V; ++v) h[v] = fmaf(a[k][kShared ? 0 : v], h[v], to_f(x[k].v[v]));
      }
      if (on) store_pack<TX, V>(out + row * A.width, h);
      if ((m.end >> k & 1u) && A.state_out && on)
#pragma unroll
        for (int v = 0; v < V; ++v) A.state_out[static_cast<int64_t>(seq) * A.width + d + v] = h[v];
    }
  }
  empty_sequences<V>(P, pl, A.h0, A.state_out);
}

// Sums of eight values over the 32 lanes: lane l with l % 4 == 0 ends up with the sum of value
// (l >> 4 & 1) * 4 + (l >> 3 & 1) * 2 + (l >> 2 & 1).  Nine shuffles instead of forty.
__device__ __forceinline__ float sum_rows(float (&v)[kRows], int lane) {
  static_assert(kRows == 8, "three halvings");
#pragma unroll
  for (int half = 4, m = 16; half > 0; half >>= 1, m >>= 1) {
    const bool up = lane & m;
#pragma unroll
    for (int j = 0; j < half; ++j) {
      const float give = up ? v[j] : v[j + half], keep = up ? v[j + half] : v[j];
      v[j] = keep + __shfl_xor_sync(kAll, give, m);
    }
  }
  v[0] += __shfl_xor_sync(kAll, v[0], 2);
  v[0] += __shfl_xor_sync(kAll, v[0], 1);
  return v[0];
}

template <typename TX, typename TA, int V, bool kShared>
__global__ void __launch_bounds__(kThreads) backward_kernel(const __grid_constant__ Params P) {
  constexpr int kG = kShared ? 1 : V;
  __shared__ float sa[kWarps][32 * V], sh[kWarps][32 * V], sc[kWarps][32 * V];
  __shared__ int scut[kWarps], send[kWarps];
  __shared__ unsigned sticket;
  __shared__ int64_t slast;   // scan index at which the last row's sequence ends, or -1: nothing is needed from behind
  __shared__ int sopen;       // the first row continues a sequence of an earlier tile
  __shared__ Carry<V> scarry;
  const gearb_recurrence_args &A = P.A;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Place pl = take_place<V, kShared>(P, &sticket, true);
  const int64_t d = pl.d0 + lane * V;
  const bool on = d < pl.d1;
  const int64_t i0 = pl.i0 + warp * kRows;
  const int n = static_cast<int>(i0 >= pl.i1 ? 0 : (pl.i1 - i0 < kRows ? pl.i1 - i0 : kRows));

  Pack<TX, V> x[kRows], dh[kRows];
  float a[kRows][kG];
  if (n > 0) {
    load_rows<TX, V>(static_cast<const TX *>(A.x), row_of(P, i0), P.x_period, A.x_batch_stride, A.x_row_stride, A.reverse, n,
                     d, on, x);
    load_rows<TX, V>(static_cast<const TX *>(A.dout), row_of(P, i0), P.dout_period, A.dout_batch_stride,
                     A.dout_row_stride, A.reverse, n, d, on, dh);
  }
  load_gate<TA, V, kShared>(P, pl, i0, n, d, on, a);
  const RowMap m = map_rows(A, P.rows, i0, n, lane);
  if (A.gate_log) {
#pragma unroll
    for (int k = 0; k < kRows; ++k)
#pragma unroll
      for (int v = 0; v < kG; ++v) a[k][v] = expf(a[k][v]);
  }

  // (A, H) of this warp's rows forward, (A, C) backward
  float ca[V], ch[V], cc[V];
#pragma unroll
  for (int v = 0; v < V; ++v) { ca[v] = 1.0f; ch[v] = 0.0f; cc[v] = 0.0f; }
#pragma unroll
  for (int k = 0; k < kRows; ++k) {
    if (!(m.live >> k & 1u)) continue;
    const bool st = m.start >> k & 1u;
    const int seq = __shfl_sync(kAll, m.seq, k);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float av = a[k][kShared ? 0 : v], xv = to_f(x[k].v[v]);
      if (st) ch[v] = (A.h0 && on) ? fmaf(av, A.h0[static_cast<int64_t>(seq) * A.width + d + v], xv) : xv;
      else ch[v] = fmaf(av, ch[v], xv);
      ca[v] *= av;
    }
  }
#pragma unroll
  for (int k = kRows - 1; k >= 0; --k) {
    if (!(m.live >> k & 1u)) continue;
    const bool en = m.end >> k & 1u;
    const int seq = __shfl_sync(kAll, m.seq, k);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if (en) cc[v] = (A.dstate && on) ? A.dstate[static_cast<int64_t>(seq) * A.width + d + v] : 0.0f;
      cc[v] = a[k][kShared ? 0 : v] * (to_f(dh[k].v[v]) + cc[v]);
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    sa[warp][lane * V + v] = ca[v];
    sh[warp][lane * V + v] = ch[v];
    sc[warp][lane * V + v] = cc[v];
  }
  if (lane == 0) {
    scut[warp] = m.start != 0;
    send[warp] = m.end != 0;
    if (warp == 0) sopen = ((m.live & ~m.start) & 1u) && m.first_start / P.tile_rows < pl.tile;
    if (n > 0 && i0 + n == pl.i1) slast = ((m.live & ~m.end) >> (n - 1) & 1u) ? m.last_end : -1;
  }
  __syncthreads();

  // of the warps before this one, forward, and of the warps behind it, backward
  float pa[V], ph[V], ba[V], bc[V];
  bool cut = false, bcut = false;
#pragma unroll
  for (int v = 0; v < V; ++v) { pa[v] = ba[v] = 1.0f; ph[v] = bc[v] = 0.0f; }
  for (int q = 0; q < warp; ++q) {
    const bool c = scut[q];
    cut |= c;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float h = sh[q][lane * V + v], b = sa[q][lane * V + v];
      ph[v] = c ? h : fmaf(b, ph[v], h);
      pa[v] *= b;
    }
  }
  for (int q = kWarps - 1; q > warp; --q) {
    const bool c = send[q];
    bcut |= c;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float h = sc[q][lane * V + v], b = sa[q][lane * V + v];
      bc[v] = c ? h : fmaf(b, bc[v], h);
      ba[v] *= b;
    }
  }
  const int64_t at = P.tiles - 1 - pl.tile;  // place of the tile in the order of the tickets
  float ta[V], tc[V];                        // of the whole tile (first warp)
  const bool tcut = bcut || m.end != 0;
  if (P.chain && warp == 0) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      tc[v] = m.end != 0 ? cc[v] : fmaf(ca[v], bc[v], cc[v]);
      ta[v] = ba[v] * ca[v];
      if (on) publish_pair(P.agg + at * A.width + d + v, ta[v], tc[v]);
    }
  }
  float hin[V], cin[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    cin[v] = 0.0f;
    hin[v] = (P.chain && sopen && on) ? A.carry[pl.tile * A.width + d + v] : 0.0f;
  }
  const int64_t lo = P.tiles - 1 - slast / P.tile_rows;
  if (P.chain && slast >= 0 && lo < at) {
    bool lost = false;
    look_back<V>(P, scarry, at, lo, d, on, lane, warp, cin, lost);
    if (lost && A.status) atomicOr(reinterpret_cast<unsigned *>(A.status), GEARB_ST_SCAN_ABORTED);
  }
  if (P.chain && warp == 0 && at % kSuper == kSuper - 1 && at + 1 < P.tiles && on) {
#pragma unroll
    for (int v = 0; v < V; ++v)
      publish_word(P.super + (at / kSuper + 1) * A.width + d + v, tcut ? tc[v] : fmaf(ta[v], cin[v], tc[v]));
  }

  if (n > 0) {
    // h_(t-1) of every row
    float hp[kRows][V], h[V];
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = cut ? ph[v] : fmaf(pa[v], hin[v], ph[v]);
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      const bool st = m.start >> k & 1u, lv = m.live >> k & 1u;
      const int seq = __shfl_sync(kAll, m.seq, k);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float xv = to_f(x[k].v[v]);
        if (st) h[v] = (A.h0 && on) ? A.h0[static_cast<int64_t>(seq) * A.width + d + v] : 0.0f;
        hp[k][v] = h[v];
        if (lv) h[v] = (st && !A.h0) ? xv : fmaf(a[k][kShared ? 0 : v], h[v], xv);
      }
    }
    float c[V], part[kRows];
#pragma unroll
    for (int v = 0; v < V; ++v) c[v] = bcut ? bc[v] : fmaf(ba[v], cin[v], bc[v]);
    TX *dx = static_cast<TX *>(A.dx) + d;
    TA *dgate = static_cast<TA *>(A.dgate);
#pragma unroll
    for (int k = kRows - 1; k >= 0; --k) {
      part[k] = 0.0f;
      if (k >= n) continue;
      const int64_t row = row_of(P, i0 + k);
      const bool lv = m.live >> k & 1u, st = m.start >> k & 1u, en = m.end >> k & 1u;
      const int seq = __shfl_sync(kAll, m.seq, k);
      float g[V], da[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float av = a[k][kShared ? 0 : v];
        if (en) c[v] = (A.dstate && on) ? A.dstate[static_cast<int64_t>(seq) * A.width + d + v] : 0.0f;
        g[v] = lv ? to_f(dh[k].v[v]) + c[v] : 0.0f;
        da[v] = (lv && !(st && !A.h0)) ? g[v] * hp[k][v] : 0.0f;
        if (A.gate_log && lv) da[v] = (st && !A.h0) ? 0.0f : da[v] * av;
        if (lv) c[v] = av * g[v];
        part[k] += on ? da[v] : 0.0f;
      }
      if (on && (lv || A.zero_rest)) {
        store_pack<TX, V>(dx + row * A.width, g);
        if constexpr (!kShared) store_pack<TA, V>(dgate + row * A.gates + d, da);
      }
      if (st && A.dh0 && on)
#pragma unroll
        for (int v = 0; v < V; ++v) A.dh0[static_cast<int64_t>(seq) * A.width + d + v] = c[v];
    }
    if constexpr (kShared) {
      const float sum = sum_rows(part, lane);
      const int k = (lane >> 4 & 1) * 4 + (lane >> 3 & 1) * 2 + (lane >> 2 & 1);
      if ((lane & 3) == 0 && k < n && ((m.live >> k & 1u) || A.zero_rest)) {
        const int64_t at_gate = row_of(P, i0 + k) * A.gates + pl.gate;
        if (P.blocks_per_gate == 1) dgate[at_gate] = from_f<TA>(sum);
        else P.gate_part[pl.part * P.rows * A.gates + at_gate] = sum;
      }
    }
  }
  empty_sequences<V>(P, pl, A.dstate, A.dh0);
}

// Joins the column blocks' sums of a gate whose channels span several of them, in order.  Rows of no
// sequence hold zeros when zero_rest is set; otherwise they are left as they are.
template <typename TA>
__global__ void __launch_bounds__(kThreads) gate_sum_kernel(const __grid_constant__ Params P) {
  const gearb_recurrence_args &A = P.A;
  const int64_t n = P.rows * A.gates;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < n;
       i += static_cast<int64_t>(gridDim.x) * kThreads) {
    if (!A.zero_rest) {
      const int64_t row = i / A.gates;
      bool live;
      if (A.offsets) live = row >= __ldg(A.offsets) && row < __ldg(A.offsets + A.sequences);
      else live = !A.lengths || row % A.time < __ldg(A.lengths + row / A.time);
      if (!live) continue;
    }
    float sum = P.gate_part[i];
    for (int b = 1; b < P.blocks_per_gate; ++b) sum += P.gate_part[b * n + i];
    static_cast<TA *>(A.dgate)[i] = from_f<TA>(sum);
  }
}

// States of sequences of a call without rows.
__global__ void states_kernel(const float *from, float *to, int64_t n) {
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < n;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x)
    to[i] = from ? from[i] : 0.0f;
}

// ---- host -------------------------------------------------------------------
int64_t up256(int64_t v) { return (v + 255) / 256 * 256; }

// Tiling of a call: rows per tile, and whether tiles need anything from each other.
void tiling(const gearb_recurrence_args &a, int64_t *rows, int *tile_rows, int64_t *tiles, int *chain) {
  *rows = a.batch * a.time;
  *tile_rows = kTile;
  *chain = *rows > kTile;
  if (!a.offsets && a.time > 0 && a.time <= kTile) {  // whole sequences per tile
    *tile_rows = static_cast<int>(kTile / a.time * a.time);
    *chain = 0;
  }
  *tiles = (*rows + *tile_rows - 1) / *tile_rows;
}

struct Scratch {
  int64_t agg, super, part, chain_bytes, total;
};
Scratch scratch_of(const gearb_recurrence_args &a, bool backward) {
  int64_t rows, tiles;
  int tile_rows, chain;
  tiling(a, &rows, &tile_rows, &tiles, &chain);
  Scratch s = {};
  if (chain) {
    s.agg = 256;
    s.super = s.agg + up256(tiles * a.width * 8);
    s.chain_bytes = s.super + up256((tiles / kSuper + 1) * a.width * 4);
  }
  s.part = s.chain_bytes;
  s.total = s.part;
  const int64_t per = a.width / a.gates;
  if (backward && a.gates < a.width && per > 32) s.total += up256((per + 31) / 32 * rows * a.gates * 4);
  return s;
}

bool vector_ok(const void *p, int64_t sb, int64_t sr, int size, int v) {
  return reinterpret_cast<uintptr_t>(p) % (size * v) == 0 && sb % v == 0 && sr % v == 0;
}

int check_sizes(const gearb_recurrence_args *a) {
  GEARB_REQUIRE(a, "recurrence: null argument");
  GEARB_REQUIRE(a->batch >= 0 && a->time >= 0 && a->width > 0 && a->gates > 0 && a->sequences >= 0,
                "recurrence: sizes must not be negative, width and gates positive");
  GEARB_REQUIRE(a->width % a->gates == 0, "recurrence: %lld channels cannot be shared by %lld gates",
                (long long)a->width, (long long)a->gates);
  GEARB_REQUIRE(a->width <= (int64_t(1) << 24) && a->batch < (int64_t(1) << 31) && a->sequences < (int64_t(1) << 31) &&
                    (a->batch == 0 || a->time <= (int64_t(1) << 40) / a->batch),
                "recurrence: width is limited to 2^24, batch and sequences to 2^31, rows to 2^40");
  GEARB_REQUIRE(a->x_dtype == GEARB_DT_F32 || a->x_dtype == GEARB_DT_F16 || a->x_dtype == GEARB_DT_BF16,
                "recurrence: x must be float32, float16 or bfloat16");
  GEARB_REQUIRE(a->gate_dtype == GEARB_DT_F32 || a->gate_dtype == a->x_dtype,
                "recurrence: gate must be float32 or of x's type");
  GEARB_REQUIRE(!(a->offsets && a->lengths), "recurrence: offsets and lengths exclude each other");
  GEARB_REQUIRE(a->offsets ? a->batch == 1 : a->sequences == a->batch,
                "recurrence: packed rows are one batch entry; otherwise there is one sequence per batch entry");
  return GEARB_OK;
}

int check_pointers(const gearb_recurrence_args *a, bool backward) {
  const bool rows = a->batch > 0 && a->time > 0;
  GEARB_REQUIRE(!rows || (a->x && a->gate), "recurrence: null argument");
  if (backward)
    GEARB_REQUIRE(!rows || (a->dout && a->dx && a->dgate), "recurrence: null argument");
  else
    GEARB_REQUIRE(!rows || a->out, "recurrence: null argument");
  return GEARB_OK;
}

template <typename TX, typename TA, int V, bool kShared>
int launch_v(Params &p, bool backward, cudaStream_t stream) {
  const gearb_recurrence_args &a = p.A;
  p.blocks_per_gate = kShared ? (p.per + 32 * V - 1) / (32 * V) : 1;
  const int64_t ncol = kShared ? a.gates * p.blocks_per_gate : (a.width + 32 * V - 1) / (32 * V);
  GEARB_REQUIRE(p.tiles <= (int64_t(1) << 31) / ncol - 1, "recurrence: too many tiles for one launch");
  p.ncol = static_cast<int>(ncol);
  const unsigned grid = static_cast<unsigned>(p.tiles * ncol);
  if (!backward) {
    forward_kernel<TX, TA, V, kShared><<<grid, kThreads, 0, stream>>>(p);
  } else {
    backward_kernel<TX, TA, V, kShared><<<grid, kThreads, 0, stream>>>(p);
    if (kShared && p.blocks_per_gate > 1) {
      const int64_t blocks = (p.rows * a.gates + kThreads - 1) / kThreads, most = static_cast<int64_t>(sm_count()) * 8;
      gate_sum_kernel<TA><<<static_cast<unsigned>(blocks < most ? blocks : most), kThreads, 0, stream>>>(p);
    }
  }
  GEARB_CUDA(cudaGetLastError());
  return GEARB_OK;
}

template <typename TX, typename TA>
int launch(const gearb_recurrence_args &a, bool backward, cudaStream_t stream) {
  Params p = {};
  p.A = a;
  tiling(a, &p.rows, &p.tile_rows, &p.tiles, &p.chain);
  if (p.rows == 0) {
    const float *from = backward ? a.dstate : a.h0;
    float *to = backward ? a.dh0 : a.state_out;
    const int64_t n = a.sequences * a.width;
    if (to && n > 0 && from != to) {
      states_kernel<<<static_cast<unsigned>((n + 255) / 256 < 4096 ? (n + 255) / 256 : 4096), 256, 0, stream>>>(from, to, n);
      GEARB_CUDA(cudaGetLastError());
    }
    return GEARB_OK;
  }
  p.per = static_cast<int>(a.width / a.gates);
  const Scratch s = scratch_of(a, backward);
  if (p.chain) {
    char *base = static_cast<char *>(a.scratch);
    p.ticket = reinterpret_cast<unsigned *>(base);
    p.agg = reinterpret_cast<float2 *>(base + s.agg);
    p.super = reinterpret_cast<float *>(base + s.super);
    GEARB_CUDA(cudaMemsetAsync(base, 0xff, static_cast<size_t>(s.chain_bytes), stream));
  }
  p.gate_part = reinterpret_cast<float *>(static_cast<char *>(a.scratch) + s.part);
  auto period = [&](int64_t sb, int64_t sr) { return sb == a.time * sr || a.batch == 1 ? p.rows : a.time; };
  p.x_period = period(a.x_batch_stride, a.x_row_stride);
  p.gate_period = period(a.gate_batch_stride, a.gate_row_stride);
  p.dout_period = period(a.dout_batch_stride, a.dout_row_stride);
  // Eight bytes of x a lane where everything is aligned for it, one channel a lane otherwise.
  constexpr int V = 8 / sizeof(TX);
  const bool shared = a.gates < a.width;
  const int64_t unit = shared ? p.per : a.width;
  bool vec = unit % V == 0 && a.width % V == 0 && vector_ok(a.x, a.x_batch_stride, a.x_row_stride, sizeof(TX), V) &&
             (shared || vector_ok(a.gate, a.gate_batch_stride, a.gate_row_stride, sizeof(TA), V));
  if (backward)
    vec = vec && vector_ok(a.dout, a.dout_batch_stride, a.dout_row_stride, sizeof(TX), V) &&
          vector_ok(a.dx, 0, 0, sizeof(TX), V) && (shared || vector_ok(a.dgate, 0, 0, sizeof(TA), V));
  else
    vec = vec && vector_ok(a.out, 0, 0, sizeof(TX), V);
  if (vec)
    return shared ? launch_v<TX, TA, V, true>(p, backward, stream) : launch_v<TX, TA, V, false>(p, backward, stream);
  return shared ? launch_v<TX, TA, 1, true>(p, backward, stream) : launch_v<TX, TA, 1, false>(p, backward, stream);
}

int dispatch(const gearb_recurrence_args &a, bool backward, cudaStream_t stream) {
  const bool wide_gate = a.gate_dtype == GEARB_DT_F32;
  switch (a.x_dtype) {
    case GEARB_DT_F32: return launch<float, float>(a, backward, stream);
    case GEARB_DT_F16:
      return wide_gate ? launch<__half, float>(a, backward, stream) : launch<__half, __half>(a, backward, stream);
    default:
      return wide_gate ? launch<__nv_bfloat16, float>(a, backward, stream)
                       : launch<__nv_bfloat16, __nv_bfloat16>(a, backward, stream);
  }
}

int run(const gearb_recurrence_args *args, bool backward, void *stream) {
  int64_t scratch = 0, carry = 0;
  int rc = gearb_recurrence_bytes(args, backward, &scratch, &carry);
  if (rc == GEARB_OK) rc = check_pointers(args, backward);
  if (rc != GEARB_OK) return rc;
  GEARB_REQUIRE(args->scratch_bytes >= scratch && (scratch == 0 || args->scratch),
                "recurrence: scratch of %lld bytes needed", (long long)scratch);
  GEARB_REQUIRE(!backward || carry == 0 || args->carry, "recurrence: the backward pass needs the forward pass's carry");
  return dispatch(*args, backward, as_stream(stream));
}

}  // namespace
}  // namespace gearb

using namespace gearb;

extern "C" {

int gearb_recurrence_bytes(const gearb_recurrence_args *args, int backward, int64_t *scratch_bytes,
                           int64_t *carry_bytes) {
  GEARB_REQUIRE(scratch_bytes && carry_bytes, "recurrence_bytes: null argument");
  const int rc = check_sizes(args);
  if (rc != GEARB_OK) return rc;
  int64_t rows, tiles;
  int tile_rows, chain;
  tiling(*args, &rows, &tile_rows, &tiles, &chain);
  *scratch_bytes = scratch_of(*args, backward != 0).total;
  *carry_bytes = chain ? tiles * args->width * 4 : 0;
  return GEARB_OK;
}

int gearb_recurrence_forward(const gearb_recurrence_args *args, void *stream) {
  TraceRange trace("gearb:recurrence");
  return run(args, false, stream);
}

int gearb_recurrence_backward(const gearb_recurrence_args *args, void *stream) {
  TraceRange trace("gearb:recurrence_backward");
  return run(args, true, stream);
}

}  // extern "C"
