// Linear recurrences over sequences, forward and backward.
//
//   h_t = a_t * h_(t-1) + x_t                      h_(-1) = h0
//   g_t = dh_t + a_(t+1) * g_(t+1)                 g_last = dh_last + dstate
//   dx_t = g_t,  da_t = sum over the gate's channels of g_t * h_(t-1),  dh0 = a_0 * g_0
//
// with a_t = gate, or exp(gate) (then dgate = da * a).  This file has what the kernels share.
//
// Any run of rows maps the state before it to the state behind it as S -> A*S + H (A the product of its a_t,
// H its own result from zero), and such maps compose, so rows can be worked on in parallel: all rows of a call,
// sequence after sequence, are cut into tiles of 64; a CTA takes one tile and one block of channels, keeps
// gate and x in registers (eight rows a warp, up to four channels a lane), forms (A, H), learns the state before
// its tile, and runs its rows again from there.  Every input is read once and every output written once.
//
// The state before a tile.  Tiles publish their (A, H).  8 consecutive tiles form a superblock, whose last tile
// publishes the superblock's (A, H); 8 superblocks form a section, whose last tile publishes the state behind it.  A tile
// applies the superblocks before it in its section to the state in front of the section, in order, and composes the
// tiles before it in its superblock onto that: the same operations whatever the timing, so results are the same bits
// every time, and the chain of CTAs that wait for one another has one link (0.5 to 0.65 us) per 4096 rows.  Where
// there are more than 512 channels, so that 512 rows of all of them take longer than a link, or few rows a sequence, a
// superblock is a section by itself: one thing less to wait for.  Measured, short sections and long:
// 54 x 10752 x 48 float32 630 and 362 us, 1 x 580000 x 16 158 and 109, 4 x 65536 x 512 bf16 (4 blocks) 376 and 328,
// 4 x 32768 x 768 (6 blocks) 217 and 229, 1 x 32768 x 2048 (16 blocks) 113 and 124, 3000 x 300 x 64 171 and 235.
// A tile needs nothing from before the start of the sequence its first row belongs to.  Tiles are handed out by a counter
// in scan order, so a CTA only ever waits for CTAs that are already running; every wait has a limit, after which the
// launch says so in the status word and the rows concerned, their states and what depends on them are NaN.  Published words are 32 bits that read 0xffffffff until they
// are written (a value of those bits is published as another NaN), so no flags and fences are needed beside them.
//
// Backward.  In terms of c_t = a_t * g_t the gradients obey c_t = a_t * c_(t+1) + a_t * dh_t, the same
// recurrence from the last row to the first, over the same tiles.  h_(t-1) is not read back (it was rounded to
// x's type) but formed again in float32 from x, gate and the state before the tile, which the forward
// pass leaves in `carry`.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.h"
#include "warp_search.cuh"

namespace gearb {
namespace rec {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kRows = 8;                     // rows a warp keeps in registers
constexpr int kTile = kWarps * kRows;        // rows per tile
constexpr int kSuper = 8;                    // tiles per superblock
constexpr int kShortSection = 3, kLongSection = 6;  // tiles per section (powers of two): one superblock, or eight
constexpr int kLongWidth = 512;              // most channels with long sections,
constexpr int kLongRows = 2048;              // and fewest rows a sequence
constexpr unsigned kAll = 0xffffffffu;
constexpr unsigned kAllRows = (1u << kRows) - 1u;
constexpr unsigned kUnset = 0xffffffffu;     // a published word that has not been written
constexpr int kPollLimit = 1 << 20;          // polls of one word, the better part of a second
constexpr unsigned kWaitLimit = 1u << 20;    // polls of an mbarrier, 4 s

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
  if constexpr (kBytes == 32) {
    reinterpret_cast<uint4 *>(&r)[0] = __ldcs(reinterpret_cast<const uint4 *>(p));
    reinterpret_cast<uint4 *>(&r)[1] = __ldcs(reinterpret_cast<const uint4 *>(p) + 1);
  } else if constexpr (kBytes == 16) {
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

// How a block of channels gets its gates: a gate each; one for the whole block; or any that it spans, each lane finding
// its own (in the streaming kernel, from a table of a few).
enum { kOwn = 0, kOne = 1, kTable = 2 };

// The rows of a tile among the sequences, for the streaming kernels.
struct alignas(16) TileRec {
  unsigned char live[kWarps], start[kWarps], end[kWarps];  // bits: rows of each warp
  unsigned starts, ends;  // bit w: a sequence starts (ends) in warp w's rows
  unsigned cut;           // bit w: a sequence starts in rows of the tile before warp w's (bit kWarps: anywhere in it)
  unsigned bcut;          // bit w: a sequence ends in rows of the tile behind warp w's (bit kWarps: anywhere in it)
  int dead;               // no row of the tile belongs to a sequence
  int plain;              // one sequence goes through the whole tile: no row of it is its first or last
  int open;               // the first row continues a sequence of an earlier tile
  int lo, lo_back;        // look back as far as this tile, counted in the order of the tickets; -1: nothing is needed
  int seq[kTile];         // sequence of each row (unless plain)
};

// What the kernels need beyond the caller's arguments.
struct Params {
  gearb_recurrence_args A;
  int64_t rows;
  int64_t tiles;
  int tile_rows;         // kTile (narrow_kernel: more), or the largest multiple of `time` below it when tiles then need
                         // nothing from each other
  int backward;
  int narrow_rows;       // rows a thread takes in narrow_kernel; 0: another kernel
  int chain;             // tiles publish to each other
  int section_shift;     // kShortSection or kLongSection
  int per;               // channels per gate
  int blocks_per_gate;   // column blocks of a gate's channels (shared gates)
  int by_gate;           // shared gates: column blocks inside one gate each (wide kernels)
  int block;             // channels of a column block where gates are not one per block
  int ncol;              // column blocks
  int flat;              // every tensor's rows lie one stride apart over the whole batch
  // Address periods: rows per batch entry, or all rows where one row stride covers the whole batch.
  int64_t x_period, gate_period, dout_period;
  unsigned *ticket;
  float2 *agg;           // [tiles][width]: (A, H) of every tile
  float2 *super;         // [superblocks][width]: (A, H) of every superblock, in long sections
  float *section;        // [sections][width]: state in front of every section
  int V;                 // channels a lane, by alignment and width
  int apart;             // with V = 2: channels 32 apart, where vectors are not aligned (wide kernels)
  TileRec *recs;         // [tiles]
  int64_t chain_bytes;   // at `ticket`: to be set to 0xff before tiles publish
  float *gate_part;      // [blocks_per_gate][rows][gates], when a gate's channels span several column blocks
  int poll_limit;        // polls of a published word before the wait is given up
  int no_waits;          // the roles of a streaming kernel give up at once
};

__device__ __forceinline__ unsigned poll_word(const unsigned *p, int limit, bool &lost) {
  unsigned v;
  for (int n = 0;; ++n) {
    asm volatile("ld.relaxed.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    if (v != kUnset) return v;
    if (lost || n == limit) break;
    __nanosleep(20);
  }
  lost = true;
  return 0x7fffffffu;  // NaN
}
__device__ __forceinline__ float2 peek_pair(const float2 *p) {
  unsigned a, h;
  asm volatile("ld.relaxed.gpu.global.v2.u32 {%0,%1}, [%2];" : "=r"(a), "=r"(h) : "l"(p) : "memory");
  return make_float2(__uint_as_float(a), __uint_as_float(h));
}
__device__ __forceinline__ float2 poll_pair(const float2 *p, int limit, bool &lost) {
  unsigned a, h;
  for (int n = 0;; ++n) {
    asm volatile("ld.relaxed.gpu.global.v2.u32 {%0,%1}, [%2];" : "=r"(a), "=r"(h) : "l"(p) : "memory");
    if (a != kUnset && h != kUnset) return make_float2(__uint_as_float(a), __uint_as_float(h));
    if (lost || n == limit) break;
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

// a / b of non-negative numbers, in 32 bits where both have no more (the usual case by far).
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  if (((a | b) >> 32) == 0) return static_cast<unsigned>(a) / static_cast<unsigned>(b);
  return a / b;
}

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
      const int64_t b = quotient(i, A.time), u = i - b * A.time;
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
      const int64_t behind = so.at(s);
      if (behind > i0 + n) {  // no sequence starts or ends behind the first row: nearly always
        settled = true;
        my_seq = s - 1;
        my_start = before;
        my_end = behind;
      }
      while (!__all_sync(kAll, settled)) {  // 32 offsets at a time: one round unless many sequences end within these rows
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
    const int64_t b = quotient(row, period);
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

template <int V, int kGate>
__device__ __forceinline__ Place take_place(const Params &P, unsigned *smem_ticket, bool backward) {
  unsigned item;
  if (P.chain) {
    if (threadIdx.x == 0) *smem_ticket = atomicAdd(P.ticket, 1u) + 1u;  // the counter starts at 0xffffffff
    __syncthreads();
    item = *smem_ticket;
  } else {
    item = blockIdx.x;
  }
  Place p;
  const unsigned t = item / static_cast<unsigned>(P.ncol);
  const int c = static_cast<int>(item - t * static_cast<unsigned>(P.ncol));
  p.tile = backward ? P.tiles - 1 - t : t;
  p.i0 = p.tile * P.tile_rows;
  p.i1 = p.i0 + P.tile_rows < P.rows ? p.i0 + P.tile_rows : P.rows;
  if (kGate == kOne) {
    p.gate = c / P.blocks_per_gate;
    p.part = c - static_cast<int>(p.gate) * P.blocks_per_gate;
    p.d0 = p.gate * P.per + static_cast<int64_t>(p.part) * 32 * V;
    p.d1 = (p.gate + 1) * P.per;
  } else {
    p.gate = 0;
    p.part = 0;
    p.d0 = static_cast<int64_t>(c) * P.block;
    p.d1 = p.d0 + P.block < P.A.width ? p.d0 + P.block : P.A.width;
  }
  return p;
}

// How the rows of a tile lie: what is the same for all of its warps.
struct TileRows {
  int64_t bb, tt;  // batch entry and row in it of the tile's first row
  bool linear;     // the tile's rows lie one row stride apart in every tensor
  bool interior;   // one sequence goes through the whole tile: no row of it is its first or last
  int64_t first_start, last_end;  // with interior: scan indexes of that sequence's first and last row
};

// Dense and padded rows, from the tile's place alone.
__device__ __forceinline__ TileRows tile_rows_dense(const Params &P, const Place &pl) {
  const gearb_recurrence_args &A = P.A;
  const int64_t b = quotient(pl.i0, A.time), u = pl.i0 - b * A.time, n = pl.i1 - pl.i0;
  TileRows t;
  t.bb = A.reverse ? A.batch - 1 - b : b;
  t.tt = A.reverse ? A.time - 1 - u : u;
  t.linear = P.flat || u + n <= A.time;
  int64_t lo = 0, hi = A.time;  // rows of the sequence, in scan order within the batch entry
  if (A.lengths) {
    int64_t len = __ldg(A.lengths + t.bb);
    len = len < 0 ? 0 : (len > A.time ? A.time : len);
    if (A.reverse) lo = A.time - len;
    else hi = len;
  }
  t.interior = u > lo && u + n < hi;
  t.first_start = pl.i0 - u + lo;
  t.last_end = pl.i0 - u + hi - 1;
  return t;
}

// Packed rows: one warp looks the tile's place up in the offsets.
__device__ __forceinline__ TileRows tile_rows_packed(const Params &P, const Place &pl, int lane) {
  const gearb_recurrence_args &A = P.A;
  TileRows t;
  t.bb = 0;
  t.tt = row_of(P, pl.i0);
  t.linear = true;
  t.interior = false;
  t.first_start = t.last_end = 0;
  const ScanOffsets so{A.offsets, P.rows, A.sequences, A.reverse};
  if (pl.i0 < so.at(A.sequences)) {
    const int64_t s = warp_upper_bound<int64_t>(A.offsets, 0, A.sequences, pl.i0, lane, so);
    if (s > 0) {
      t.first_start = so.at(s - 1);
      const int64_t behind = so.at(s);
      t.last_end = behind - 1;
      t.interior = t.first_start < pl.i0 && behind > pl.i1 && behind <= P.rows;
    }
  }
  return t;
}

// Tiles with rows of sequences, [first, end): packed sequences may leave rows in front of the first and behind the last.
struct LiveTiles {
  int64_t first, end;
};
__device__ __forceinline__ LiveTiles live_tiles(const Params &P) {
  if (!P.A.offsets) return {0, P.tiles};
  const ScanOffsets so{P.A.offsets, P.rows, P.A.sequences, P.A.reverse};
  const int64_t lo = so.at(0), hi = so.at(P.A.sequences);
  LiveTiles t;
  t.first = quotient(lo, P.tile_rows);
  t.end = quotient(hi + P.tile_rows - 1, P.tile_rows);
  if (hi <= lo) t.end = t.first;
  return t;
}

// V channels a lane of a warp's n rows of the scan (zeros where there is no row or channel): consecutive ones from d on, or,
// with kApart, every 32nd.  Where vectors are not aligned, two channels apart a lane are as many bytes in flight as
// vectors of two, and read memory in order.
template <int V, bool kApart>
struct Channels {
  int d, end;  // the lane's first channel, the block's end
  __device__ __forceinline__ Channels(int d_, int end_) : d(d_), end(end_) {}
  __device__ __forceinline__ Channels(const Place &pl, int lane)
      : d(static_cast<int>(pl.d0) + (kApart ? lane : lane * V)), end(static_cast<int>(pl.d1)) {}
  __device__ __forceinline__ static int of(int lane, int v) { return kApart ? lane + 32 * v : lane * V + v; }  // in the block
  __device__ __forceinline__ int at(int v) const { return d + (kApart ? 32 * v : v); }
  __device__ __forceinline__ bool on(int v) const { return at(v) < end; }
  template <typename T>
  __device__ __forceinline__ Pack<T, V> load(const T *row) const {
    Pack<T, V> r;
    if constexpr (kApart) {
#pragma unroll
      for (int v = 0; v < V; ++v) r.v[v] = on(v) ? load_pack<T, 1>(row + at(v)).v[0] : from_f<T>(0.0f);
    } else {
      if (on(0)) return load_pack<T, V>(row + d);
#pragma unroll
      for (int v = 0; v < V; ++v) r.v[v] = from_f<T>(0.0f);
    }
    return r;
  }
  template <typename T>
  __device__ __forceinline__ void store(T *row, const float (&f)[V]) const {
    if constexpr (kApart) {
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (on(v)) row[at(v)] = from_f<T>(f[v]);
    } else {
      if (on(0)) store_pack<T, V>(row + d, f);
    }
  }
};
template <typename T, int V, bool kApart>
__device__ __forceinline__ void load_rows(const T *base, const Params &P, const Place &pl, const TileRows &tr, int64_t period,
                                          int64_t sb, int64_t sr, int warp, int n, const Channels<V, kApart> &ch,
                                          Pack<T, V> (&r)[kRows]) {
  if (n == kRows && tr.linear) {
    const int64_t step = P.A.reverse ? -sr : sr;
    const T *p = base + (tr.bb * sb + tr.tt * sr + warp * kRows * step);
#pragma unroll
    for (int k = 0; k < kRows; ++k) r[k] = ch.load(p + k * step);
    return;
  }
#pragma unroll
  for (int k = 0; k < kRows; ++k)
#pragma unroll
    for (int v = 0; v < V; ++v) r[k].v[v] = from_f<T>(0.0f);
  if (n == 0) return;
  RowWalk w(row_of(P, pl.i0 + warp * kRows), period, sb, sr, P.A.reverse);
#pragma unroll
  for (int k = 0; k < kRows; ++k) {
    if (k < n) r[k] = ch.load(base + w.off);
    w.next();
  }
}

// The state of channel d in front of tile `at` (in the order of the tickets), from what the tiles before it published;
// the last tile of a superblock publishes for it on the way, that of a section too.  lo: the first tile that matters
// (`at`: none).  own() gives the tile's own (A, H), asked for by such last tiles only; cut: a sequence starts in the tile.
// kAhead pairs are asked for at a time: all seven by warps that have nothing else to hold in registers.  kShift: the
// section's shift where it is known in advance, or 0.
template <int kAhead, int kShift, typename Index, typename Own>
__device__ __forceinline__ float look_back(const Params &P, Index at, Index lo, Index d, Own &&own, bool cut,
                                           bool &lost) {
  const int shift = kShift > 0 ? kShift : P.section_shift;
  const int64_t width = P.A.width;
  const Index sb = at / kSuper, sec = at >> shift, sec0 = sec << shift;
  const bool by_super = lo < sb * kSuper, by_section = lo < sec0;
  const Index t0 = by_super ? sb * kSuper : lo, s0 = (by_section ? sec0 : lo) / kSuper;
  const int tiles = static_cast<int>(at - t0), supers = kShift != kShortSection && by_super ? static_cast<int>(sb - s0) : 0;
  const float2 *tp = P.agg + t0 * width + d, *sp = P.super + s0 * width + d;
  constexpr bool kAll7 = kAhead == kSuper - 1;
  float2 t[kAhead], s[kAhead];
  auto peek = [&](float2(&q)[kAhead], const float2 *p, int from, int n) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (from + u < n) q[u] = peek_pair(p + (from + u) * width);
  };
  auto settle = [&](float2 &q, const float2 *p) {
    if (__float_as_uint(q.x) == kUnset || __float_as_uint(q.y) == kUnset) q = poll_pair(p, P.poll_limit, lost);
  };
  unsigned word = 0;
  peek(t, tp, 0, tiles);
  if (kAll7) peek(s, sp, 0, supers);
  if (by_section) asm volatile("ld.relaxed.gpu.global.u32 %0, [%1];" : "=r"(word) : "l"(P.section + sec * width + d) : "memory");

  float pa = 1.0f, ph = 0.0f;  // of the tiles before this one in its superblock
  for (int j = 0; j < tiles; j += kAhead) {
    if (j > 0) peek(t, tp, j, tiles);
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (j + u < tiles) {
        settle(t[u], tp + (j + u) * width);
        // nothing in front of the sequence's start counts
        ph = (j + u == 0 && !by_super) ? t[u].y : fmaf(t[u].x, ph, t[u].y);
        pa *= t[u].x;
      }
  }
  const bool last = at % kSuper == kSuper - 1 && at + 1 < static_cast<Index>(P.tiles);
  const bool very_last = last && at + 1 == (sec + 1) << shift;
  if (last && !very_last) {
    const float2 t = own();
    publish_pair(P.super + sb * width + d, t.x * pa, cut ? t.y : fmaf(t.x, ph, t.y));
  }
  float in = ph;
  if (by_super) {
    float h = 0.0f;
    if (by_section) {
      if (word == kUnset) word = poll_word(reinterpret_cast<const unsigned *>(P.section + sec * width + d), P.poll_limit, lost);
      h = __uint_as_float(word);
    }
    for (int j = 0; j < supers; j += kAhead) {
      if (!kAll7) peek(s, sp, j, supers);
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (j + u < supers) {
          settle(s[u], sp + (j + u) * width);
          h = (j + u == 0 && !by_section) ? s[u].y : fmaf(s[u].x, h, s[u].y);
        }
    }
    in = fmaf(pa, h, ph);
  }
  if (very_last) {
    const float2 t = own();
    publish_word(P.section + (sec + 1) * width + d, cut ? t.y : fmaf(t.x, in, t.y));
  }
  return in;
}

// e^x in float32 from 2^t (one instruction, 2 units in the last place): with t = x / ln 2 rounded, e^x = 2^t * e^r for
// the r = x - t ln 2 that the rounding left, and e^r = 1 + r to 2^-30 for x above -150, below which e^x is 0.
constexpr float kLog2E = 1.4426950408889634f;
constexpr float kLn2Hi = 0.693147180559945309f;                       // rounded to float32
constexpr float kLn2Lo = static_cast<float>(0.693147180559945309 - static_cast<double>(kLn2Hi));
__device__ __forceinline__ float exp_of(float x) {
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(x) : "f"(x), "f"(-150.0f));
  const float t = x * kLog2E;
  const float r = fmaf(-t, kLn2Lo, fmaf(-t, kLn2Hi, x));
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
  return fmaf(e, r, e);
}

// Hands a sequence without rows its state (forward) or its gradient (backward): the CTAs of a launch share the
// sequences among them.
__device__ __forceinline__ void empty_sequences(const Params &P, const Place &pl, int64_t block, const float *from, float *to) {
  const gearb_recurrence_args &A = P.A;
  if (!to) return;
  for (int64_t s = pl.tile * kThreads + threadIdx.x; s < A.sequences; s += P.tiles * kThreads) {
    int64_t n;
    if (A.offsets) {
      const ScanOffsets so{A.offsets, P.rows, A.sequences, 0};
      n = so.at(s + 1) - so.at(s);
    } else if (!A.lengths) {
      return;
    } else {
      n = __ldg(A.lengths + s);
    }
    if (n > 0) continue;
    const int64_t d1 = pl.d0 + block < pl.d1 ? pl.d0 + block : pl.d1;
    for (int64_t d = pl.d0; d < d1; ++d) to[s * A.width + d] = from ? from[s * A.width + d] : 0.0f;
  }
}

// Whether rows can be read or written v values at a time.
inline bool vector_ok(const void *p, int64_t sb, int64_t sr, int size, int v) {
  return reinterpret_cast<uintptr_t>(p) % (size * v) == 0 && sb % v == 0 && sr % v == 0;
}

// Long sections where the chain would take longer than the work, and sequences are long enough to feel it.  By the sizes
// alone: the section decides how a state is rounded, and every kernel gives the same bits.
inline int section_shift_of(const Params &p) {
  return p.A.width <= kLongWidth && p.rows / kLongRows >= p.A.sequences ? kLongSection : kShortSection;
}

// In front of a streaming kernel: finds out about the tiles' rows, and clears what they publish in.
int launch_prepare(const Params &p, cudaStream_t stream);
int launch_f32(Params &p, bool backward, cudaStream_t stream);
int launch_f16(Params &p, bool backward, cudaStream_t stream);
int launch_bf16(Params &p, bool backward, cudaStream_t stream);

}  // namespace rec
}  // namespace gearb
