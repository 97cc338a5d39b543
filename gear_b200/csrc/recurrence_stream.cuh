// Kernels of the recurrences for long calls whose rows lie in one TMA-addressable matrix.
//
// The tiles are those of recurrence_wide.cuh, but the CTAs stay, one per SM, and their warps have roles, so that
// nothing waits in line:
//   issuer      takes the next tile's number from the counter and starts its copies (one tensor copy per input)
//   recorders   fetch what the launch before found out about the tile's rows (which start or end a sequence: once for all
//               column blocks), and shared gates
//   compute     first look at tile m: (A, H) of each warp's rows; then, tile m - 2 again: its rows from the state
//               before them, and out
//   publishers  one thread per channel: turn the warps' pairs into those of all rows before each warp, publish the
//               tile's
//   finishers   one thread per channel: the state in front of the tile from what the tiles before published
// They meet at mbarriers only, and once more when they end: where a wait ran into its limit, abandon() leaves NaN.
// 2 x 16384 x 2048 bf16 with float32 log gates takes 115 us, 4.67 TB/s of 6.55 (82 us); the backward pass of
// 4 x 4096 x 2048 118 us, beside 62 us forward.  What bounds it now: 19 warps of one CTA issue in 52 % of the cycles (the
// two looks at every element, exponentials and conversions), and the rest is the latency of what they hand each other
// (long scoreboard 3.8 of 8 stall cycles an issue); two CTAs an SM do not fit the registers.  Measured on the way:
// a CTA per tile 170 us whatever the types; CTAs that stay but finish a tile before they begin the next: every tile
// spent 6700 of 11000 cycles looking back; one bulk copy per row: an SM starts one about every 35 cycles, 180 us;
// every warp finding its rows' place itself: 600 of 1000 instructions; both phases' rows in registers: spills, 234 us;
// the issuer looking the rows up in the offsets: 4 us a tile; several tiles' numbers taken at once: tiles wait for
// others far back in another CTA's queue, 250 to 600 us; two CTA barriers a tile in place of the roles: 136 us.
#pragma once

#include <cuda.h>

#include "recurrence_narrow.cuh"
#include "recurrence_wide.cuh"
#include "ring.h"

namespace gearb {
namespace rec {

constexpr int kStreamThreads = kThreads + 11 * 32;  // compute, 4 publishers, 4 finishers, issuer, 2 recorders
constexpr int kSmemMost = 227 * 1024;
constexpr unsigned kLag = 2;  // tiles that compute warps begin before they come back to one (1: 124 us in place of 110)
constexpr unsigned kRing = kLag + 1;
constexpr int kMostStages = 6;
constexpr int kRecorders = 2;  // one takes 3 us a tile: two dependent trips to L2
constexpr int kTableGates = 8;

constexpr unsigned kNoItem = 0xffffffffu;

__device__ __forceinline__ uint32_t smem_addr(const void *p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void mbar_expect(uint64_t *bar, unsigned bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_addr(bar)), "r"(bytes) : "memory");
}
// Every try waits up to 4 us by itself; with a hint it may wait as long as the hint says, and 2^20 times that is no limit.  The
// limit is a constant: as a parameter of the launch it made packed heads 5 % slower.
__device__ __forceinline__ bool mbar_wait(uint64_t *bar, unsigned parity) {
#pragma unroll 1
  for (unsigned n = 0; n < kWaitLimit; ++n) {
    unsigned ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_addr(bar)), "r"(parity)
        : "memory");
    if (ok) return true;
  }
  return false;
}
// Box (channels c.., rows r..) of a matrix into shared memory; what lies outside the matrix arrives as zeros.
__device__ __forceinline__ void tensor_load(void *dst, const CUtensorMap *map, int c, int r, uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
          smem_addr(dst)),
      "l"(map), "r"(c), "r"(r), "r"(smem_addr(bar))
      : "memory");
}
int encode_map(CUtensorMap *map, CUtensorMapDataType type, void *base, int64_t width, int64_t rows, int64_t row_bytes, int box_w,
               int box_h);
struct Maps {
  CUtensorMap x, gate, dout;
};

// Two multiply-adds in one instruction.
__device__ __forceinline__ void fma2(float &d0, float &d1, float a0, float a1, float b0, float b1, float c0, float c1) {
  asm("{\n\t.reg .b64 a, b, c, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\t"
      "mov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d0), "=f"(d1)
      : "f"(a0), "f"(a1), "f"(b0), "f"(b1), "f"(c0), "f"(c1));
}
__device__ __forceinline__ void mul2(float &d0, float &d1, float a0, float a1, float b0, float b1) {
  asm("{\n\t.reg .b64 a, b, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "mul.rn.f32x2 d, a, b;\n\t"
      "mov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d0), "=f"(d1)
      : "f"(a0), "f"(a1), "f"(b0), "f"(b1));
}
// d = a * b + c, channel by channel.
template <int V, int kG>
__device__ __forceinline__ void fma_v(float (&d)[V], const float (&a)[kG], const float (&b)[V], const float (&c)[V]) {
  if constexpr (V == 1) {
    d[0] = fmaf(a[0], b[0], c[0]);
  } else {
#pragma unroll
    for (int v = 0; v < V; v += 2)
      fma2(d[v], d[v + 1], a[kG == 1 ? 0 : v], a[kG == 1 ? 0 : v + 1], b[v], b[v + 1], c[v], c[v + 1]);
  }
}
template <int V, int kG>
__device__ __forceinline__ void mul_v(float (&d)[V], const float (&a)[kG], const float (&b)[V]) {
  if constexpr (V == 1) {
    d[0] = a[0] * b[0];
  } else {
#pragma unroll
    for (int v = 0; v < V; v += 2) mul2(d[v], d[v + 1], a[kG == 1 ? 0 : v], a[kG == 1 ? 0 : v + 1], b[v], b[v + 1]);
  }
}
template <typename T, int V>
__device__ __forceinline__ void unpack(const Pack<T, V> &p, float (&f)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) f[v] = to_f(p.v[v]);
}

__device__ __forceinline__ bool warp_wait(uint64_t *bar, unsigned parity) {
  return __all_sync(kAll, mbar_wait(bar, parity));
}
__device__ __forceinline__ void mbar_init_count(uint64_t *bar, unsigned n) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(bar)), "r"(n));
}
__device__ __forceinline__ void mbar_arrive(uint64_t *bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}

// Shared memory of one stage.  A tensor copy writes to 128-byte boundaries.
template <typename TX, typename TA, int V, int kGate, bool kBackward>
struct Stage {
  alignas(128) TX x[kTile][32 * V];
  alignas(128) TX dout[kBackward ? kTile : 1][kBackward ? 32 * V : 8];
  alignas(128) TA gate[kGate != kOwn ? 1 : kTile][kGate != kOwn ? 8 : 32 * V];
  static constexpr unsigned kBytes = sizeof(TX) * 32 * V * kTile * (kBackward ? 2 : 1) +
                                     (kGate != kOwn ? 0 : sizeof(TA) * 32 * V * kTile);
};

// What the warps need to know about a tile: what prepare_kernel found out about its rows, and its place.  Rows are
// counted in 32 bits here (the entry point sends longer calls elsewhere).
struct Plan {
  TileRec rec;
  int valid;
  int tile, rows;  // rows of the scan in it
  int row0;        // matrix row of the first of them; the others follow it, or precede it in a reverse call
  int d0, cols;    // first channel, channels
  int gate, part;  // shared gates: the gate, and which block of its channels
};
template <int kGate>
struct GateRows {  // a of each row, for gates that are not copied with the rows
  float a[kGate == kOwn ? 1 : kTile][kGate == kTable ? kTableGates : 1];
};

template <int V, bool kBackward>
struct Pairs {  // of the warps of one tile; then of all rows before (backward: behind) each warp's
  alignas(16) float a[kWarps][32 * V];
  alignas(16) float h[kWarps][32 * V];
  alignas(16) float b[kBackward ? kWarps : 1][kBackward ? 32 * V : 4];
  alignas(16) float c[kBackward ? kWarps : 1][kBackward ? 32 * V : 4];
};
template <int V, bool kBackward>
struct Edge {  // of one tile: its own pair, and the state that enters it (backward: from behind, and from in front)
  alignas(16) float a[32 * V];
  alignas(16) float h[32 * V];
  alignas(16) float in[32 * V];
  alignas(16) float front[kBackward ? 32 * V : 4];
};

template <typename TX, typename TA, int V, int kGate, bool kBackward>
struct StreamShared {
  using StageT = Stage<TX, TA, V, kGate, kBackward>;
  static constexpr int kEach = static_cast<int>(sizeof(StageT) + sizeof(Edge<V, kBackward>) + sizeof(Plan) + sizeof(GateRows<kGate>)) + 64;
  static constexpr int kFit = (kSmemMost - static_cast<int>(kRing * sizeof(Pairs<V, kBackward>)) - 256) / kEach;
  static constexpr unsigned kStages = kFit > kMostStages ? kMostStages : kFit;
  static_assert(kStages >= kLag + 2, "the tiles in work and one on its way");
  StageT stage[kStages];
  Pairs<V, kBackward> pairs[kRing];
  Edge<V, kBackward> edge[kStages];
  Plan plan[kStages];
  GateRows<kGate> gates[kStages];
  uint64_t full[kStages], empty[kStages];  // the tile's rows and plan are there; the tile is done with
  uint64_t issued[kStages];                // item is there
  unsigned item[kStages];
  uint64_t entered[kStages];               // edge.in is there
  uint64_t paired[kRing], ready[kRing], read[kRing];   // the warps' pairs; turned and edge.a, edge.h there; read again
  // How far the roles have come when they end, for abandon(): tiles issued, the item behind them, tiles that each compute warp
  // has done with, the turn of the first tile that each recorder has not recorded.
  unsigned issued_tiles, next, done[kWarps];
  Turn<kStages> recorded[kRecorders];
};

// Short sections: what the tiles before one (in the order of the tickets) published, asked for at once.
struct Peek {
  float2 q[kSuper - 1];
  float s;
};
__device__ __forceinline__ void peek_back(const Params &P, int at, int lo, int d, Peek &k) {
  const int sb = at / kSuper, sb0 = sb * kSuper;
  const bool need_section = lo < sb0;
  const int j0 = need_section ? sb0 : lo, count = at - j0;
  const float2 *p = P.agg + j0 * P.A.width + d;
#pragma unroll
  for (int u = 0; u < kSuper - 1; ++u)
    if (u < count) k.q[u] = peek_pair(p + u * P.A.width);
  if (need_section) {
    unsigned w;
    asm volatile("ld.relaxed.gpu.global.u32 %0, [%1];" : "=r"(w) : "l"(P.section + sb * P.A.width + d) : "memory");
    k.s = __uint_as_float(w);
  }
}
// The state in front of tile `at`: as look_back, from what was peeked at, waiting for what was not there yet.
__device__ __forceinline__ float settle_back(const Params &P, int at, int lo, int d, Peek &k, bool &lost) {
  const int sb = at / kSuper, sb0 = sb * kSuper;
  const bool need_section = lo < sb0;
  const int j0 = need_section ? sb0 : lo, count = at - j0;
  const float2 *p = P.agg + j0 * P.A.width + d;
  float pa = 1.0f, ph = 0.0f;
#pragma unroll
  for (int u = 0; u < kSuper - 1; ++u)
    if (u < count) {
      if (__float_as_uint(k.q[u].x) == kUnset || __float_as_uint(k.q[u].y) == kUnset)
        k.q[u] = poll_pair(p + u * P.A.width, P.poll_limit, lost);
      ph = (u == 0 && !need_section) ? k.q[u].y : fmaf(k.q[u].x, ph, k.q[u].y);
      pa *= k.q[u].x;
    }
  if (!need_section) return ph;
  if (__float_as_uint(k.s) == kUnset)
    k.s = __uint_as_float(poll_word(reinterpret_cast<const unsigned *>(P.section + sb * P.A.width + d), P.poll_limit, lost));
  return fmaf(pa, k.s, ph);
}

// Where an item lies.
template <int V, int kGate, bool kBackward>
__device__ __forceinline__ Place place_of_item(const Params &P, unsigned item) {
  Place at;
  const unsigned t = item / static_cast<unsigned>(P.ncol);
  const int c = static_cast<int>(item - t * static_cast<unsigned>(P.ncol));
  at.tile = kBackward ? P.tiles - 1 - t : t;
  at.i0 = at.tile * P.tile_rows;
  at.i1 = at.i0 + P.tile_rows < P.rows ? at.i0 + P.tile_rows : P.rows;
  at.gate = kGate == kOne ? c / P.blocks_per_gate : 0;
  at.part = kGate == kOne ? c - static_cast<int>(at.gate) * P.blocks_per_gate : 0;
  at.d0 = kGate == kOne ? at.gate * P.per + at.part * 32 * V : c * 32 * V;
  at.d1 = kGate == kOne ? (at.gate + 1) * P.per : P.A.width;
  return at;
}

// The items of a call: tiles without sequences are none, the launch before has zeroed their rows.  (Taken through the
// pipeline, the 43 % of a packed batch's room that no sequence filled cost a quarter of the time.)
struct Items {
  unsigned base, end;
};
template <bool kBackward>
__device__ __forceinline__ Items items_of(const Params &P) {
  const LiveTiles live = live_tiles(P);
  Items t;
  t.base = static_cast<unsigned>((kBackward ? P.tiles - live.end : live.first) * P.ncol);
  t.end = t.base + static_cast<unsigned>((live.end - live.first) * P.ncol);
  return t;
}
// The item behind `item` for this CTA.
__device__ __forceinline__ unsigned item_behind(const Params &P, const Items &items, unsigned item) {
  return P.chain ? items.base + atomicAdd(P.ticket, 1u) + 1u : item + gridDim.x;  // the counter starts at 0xffffffff
}

// The issuing warp (one lane of it): numbers and copies.
template <typename TX, typename TA, int V, int kGate, bool kBackward>
__device__ __forceinline__ bool issue_tiles(const Params &P, const Maps &maps, StreamShared<TX, TA, V, kGate, kBackward> &sm) {
  using Shared = StreamShared<TX, TA, V, kGate, kBackward>;
  const gearb_recurrence_args &A = P.A;
  const Items items = items_of<kBackward>(P);
  // One number at a time from the start: CTAs that took several at once would come to tiles much later than others come to
  // the tiles behind them, and those would wait.
  unsigned next = P.chain ? item_behind(P, items, 0) : items.base + blockIdx.x;
  Turn<Shared::kStages> now;
  bool lost = false;
  for (unsigned m = 0;; ++m, now.next()) {
    lost = m >= Shared::kStages && (P.no_waits || !mbar_wait(&sm.empty[now.i], now.parity ^ 1u));
    if (lost || next >= items.end) {
      sm.issued_tiles = m;
      sm.next = next;
      if (lost) return true;
    }
    const unsigned item = next;
    sm.item[now.i] = item < items.end ? item : kNoItem;
    if (item >= items.end) {
      mbar_arrive(&sm.full[now.i]);
      for (int r = 0; r < kRecorders; ++r) {  // every recorder has to learn that there are no more
        mbar_arrive(&sm.issued[now.i]);
        now.next();
        if (r + 1 < kRecorders) {
          ++m;
          if (m >= Shared::kStages && (P.no_waits || !mbar_wait(&sm.empty[now.i], now.parity ^ 1u))) return true;
          sm.item[now.i] = kNoItem;
        }
      }
      return false;
    }
    const Place at = place_of_item<V, kGate, kBackward>(P, item);
    uint64_t *full = &sm.full[now.i];
    // a reverse call's tile ends at row_of(i0): its box begins kTile - 1 rows before, if need be in front of the matrix
    const int row0 = static_cast<int>(row_of(P, at.i0)), c = static_cast<int>(at.d0), r = A.reverse ? row0 - (kTile - 1) : row0;
    mbar_expect(full, Shared::StageT::kBytes);
    tensor_load(sm.stage[now.i].x, &maps.x, c, r, full);
    if constexpr (kGate == kOwn) tensor_load(sm.stage[now.i].gate, &maps.gate, c, r, full);
    if constexpr (kBackward) tensor_load(sm.stage[now.i].dout, &maps.dout, c, r, full);
    mbar_arrive(&sm.issued[now.i]);
    next = item_behind(P, items, item);  // needed a tile later
  }
}

// The recording warps, every kRecorders-th tile each: what is known about a tile's rows, and gates that are not copied.
template <typename TX, typename TA, int V, int kGate, bool kBackward>
__device__ __forceinline__ bool record_tiles(const Params &P, StreamShared<TX, TA, V, kGate, kBackward> &sm, int which, int lane) {
  using Shared = StreamShared<TX, TA, V, kGate, kBackward>;
  const gearb_recurrence_args &A = P.A;
  Turn<Shared::kStages> now;
  for (int k = 0; k < which; ++k) now.next();
  for (;;) {
    if (!warp_wait(&sm.issued[now.i], now.parity)) {
      if (lane == 0) sm.recorded[which] = now;
      return true;
    }
    const unsigned item = sm.item[now.i];
    Plan &pl = sm.plan[now.i];
    if (item == kNoItem) {
      if (lane == 0) {
        pl.valid = 0;
        sm.recorded[which] = now;
        mbar_arrive(&sm.full[now.i]);
      }
      return false;
    }
    const Place at = place_of_item<V, kGate, kBackward>(P, item);
    const int n = static_cast<int>(at.i1 - at.i0), row0 = static_cast<int>(row_of(P, at.i0));
    constexpr int kWords = static_cast<int>(sizeof(TileRec) / 4), kEach = (kWords + 31) / 32;
    const int *from = reinterpret_cast<const int *>(P.recs + at.tile);
    int word[kEach];
#pragma unroll
    for (int w = 0; w < kEach; ++w) word[w] = w * 32 + lane < kWords ? __ldg(from + w * 32 + lane) : 0;
    // gates: all 64 rows of one, or of eight (lane l: gate l % 8 of rows l / 8, l / 8 + 4, ...)
    constexpr int kLooks = kGate == kOwn ? 1 : (kGate == kOne ? kTile / 32 : kTile / 4);
    float own[kLooks];
    if constexpr (kGate != kOwn) {
      const int g = kGate == kOne ? static_cast<int>(at.gate) : static_cast<int>(at.d0) / P.per + (lane & 7);
      const bool wanted = g < A.gates && (kGate == kOne || static_cast<int64_t>(g) * P.per < at.d0 + 32 * V);
#pragma unroll
      for (int u = 0; u < kLooks; ++u) {
        const int k = kGate == kOne ? lane + 32 * u : (lane >> 3) + 4 * u;
        own[u] = 0.0f;
        if (k < n && wanted)
          own[u] = to_f(static_cast<const TA *>(A.gate)[(A.reverse ? row0 - k : row0 + k) * A.gate_row_stride + g]);
      }
    }
#pragma unroll
    for (int w = 0; w < kEach; ++w)
      if (w * 32 + lane < kWords) reinterpret_cast<int *>(&pl.rec)[w * 32 + lane] = word[w];
    if constexpr (kGate != kOwn) {
#pragma unroll
      for (int u = 0; u < kLooks; ++u) {
        const float a = A.gate_log ? exp_of(own[u]) : own[u];
        if constexpr (kGate == kOne) sm.gates[now.i].a[lane + 32 * u][0] = a;
        else sm.gates[now.i].a[(lane >> 3) + 4 * u][lane & 7] = a;
      }
    }
    if (lane == 0) {
      pl.valid = 1;
      pl.tile = static_cast<int>(at.tile);
      pl.rows = n;
      pl.row0 = row0;
      pl.d0 = static_cast<int>(at.d0);
      pl.cols = static_cast<int>(at.d1 - at.d0 < 32 * V ? at.d1 - at.d0 : 32 * V);
      pl.gate = static_cast<int>(at.gate);
      pl.part = at.part;
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&sm.full[now.i]);
    for (int k = 0; k < kRecorders; ++k) now.next();
  }
}

// A warp's rows of a tile in its stage: row k of the warp (in scan order) at k * step.
template <typename TX, typename TA, int V, int kGate, bool kBackward>
struct WarpRows {
  static constexpr int kW = 32 * V, kG = kGate == kOne ? 1 : V;
  TX *x, *dout;
  TA *gate;
  const float *table;
  int step, column[kGate == kTable ? V : 1];
  __device__ __forceinline__ WarpRows(const Params &P, const Plan &pl, StreamShared<TX, TA, V, kGate, kBackward> &sm,
                                      unsigned stage, int warp, int lane) {
    auto &st = sm.stage[stage];
    const int k0 = P.A.reverse ? kTile - 1 - warp * kRows : warp * kRows, at = k0 * kW + lane * V;
    step = P.A.reverse ? -kW : kW;
    x = st.x[0] + at;
    dout = st.dout[0] + (kBackward ? at : 0);
    gate = st.gate[0] + (kGate != kOwn ? 0 : at);
    table = sm.gates[stage].a[kGate == kOwn ? 0 : warp * kRows];
    if constexpr (kGate == kTable) {
      const int d = pl.d0 + lane * V, g0 = pl.d0 / P.per;
#pragma unroll
      for (int v = 0; v < V; ++v) column[v] = min((d + v) / P.per - g0, kTableGates - 1);  // channels beyond the width too
    }
  }
  __device__ __forceinline__ void get_x(int k, float (&f)[V]) const {
    unpack(*reinterpret_cast<const Pack<TX, V> *>(x + k * step), f);
  }
  __device__ __forceinline__ void get_dout(int k, float (&f)[V]) const {
    unpack(*reinterpret_cast<const Pack<TX, V> *>(dout + k * step), f);
  }
  // a of row k.  The first look turns a float32 log gate into a where it lies; a 16-bit one is turned at every look.
  __device__ __forceinline__ void get_a(int k, int log, bool first, float (&a)[kG]) const {
    if constexpr (kGate == kOne) {
      a[0] = table[k];
    } else if constexpr (kGate == kTable) {
#pragma unroll
      for (int v = 0; v < V; ++v) a[v] = table[k * kTableGates + column[v]];
    } else {
      unpack(*reinterpret_cast<const Pack<TA, V> *>(gate + k * step), a);
      if (log && (first || sizeof(TA) == 2)) {
#pragma unroll
        for (int v = 0; v < V; ++v) a[v] = exp_of(a[v]);
        if constexpr (sizeof(TA) == 4)
          if (first) store_pack<TA, V>(gate + k * step, a);
      }
    }
  }
};

// h = a * h + x for one row.  At a sequence's first row h comes from h0, or the row is h = x.  What a row of no
// sequence leaves is never used: the next row of one is its first.
template <int V, int kG>
__device__ __forceinline__ void step_row(const gearb_recurrence_args &A, const Plan &pl, unsigned start, int k, int row, int d,
                                         bool on, float (&a)[kG], const float (&x)[V], float (&h)[V]) {
  if (start >> k & 1u) {
    if (A.h0) {
      state_load<V>(A.h0, pl.rec.seq[row], A.width, d, on, h);
    } else {  // 0 * -0 + x is x, to the sign of a zero
#pragma unroll
      for (int v = 0; v < V; ++v) h[v] = -0.0f;
#pragma unroll
      for (int v = 0; v < kG; ++v) a[v] = 0.0f;
    }
  }
  fma_v(h, a, h, x);
}

// Finishers: the state in front of every tile (backward: behind it), and what its superblock and section publish.
template <typename TX, typename TA, int V, int kGate, bool kBackward, bool kLong>
__device__ __forceinline__ bool finish_tiles(const Params &P, StreamShared<TX, TA, V, kGate, kBackward> &sm, int c, int lane) {
  using Shared = StreamShared<TX, TA, V, kGate, kBackward>;
  const gearb_recurrence_args &A = P.A;
  bool lost = false;
  unsigned stage = 0, parity = 0;
  Follower<kRing> ready;
  for (;;) {
    if (!warp_wait(&sm.full[stage], parity)) return true;
    const Plan &pl = sm.plan[stage];
    if (!pl.valid) return lost;
    const int tile = kBackward ? static_cast<int>(P.tiles) - 1 - pl.tile : pl.tile, lo = kBackward ? pl.rec.lo_back : pl.rec.lo, d = pl.d0 + c;
    const bool on = c < pl.cols;
    float in = 0.0f;
    const bool cut = (kBackward ? pl.rec.bcut : pl.rec.cut) >> kWarps & 1u;
    if constexpr (!kLong) {
      if (on && lo >= 0) {
        Peek peek;
        peek_back(P, tile, lo, d, peek);
        in = settle_back(P, tile, lo, d, peek, lost);
        if (!kBackward && A.carry) A.carry[pl.tile * A.width + d] = in;
      }
    } else if (on && (lo >= 0 || (P.chain && tile % kSuper == kSuper - 1))) {
      auto own = [&] {
        if (mbar_wait(&sm.ready[ready.turn.i], ready.turn.parity))
          return make_float2(sm.edge[stage].a[c], sm.edge[stage].h[c]);
        lost = true;
        return make_float2(__uint_as_float(0x7fffffffu), __uint_as_float(0x7fffffffu));
      };
      in = look_back<kSuper - 1, kLongSection, int>(P, tile, lo >= 0 ? lo : tile, d, own, cut, lost);
      if (!kBackward && A.carry && lo >= 0) A.carry[pl.tile * A.width + d] = in;
    }
    // The tile's own pair, which the compute warps wait for as well.  Every tile's: see Follower.
    if (!ready.pass([&](unsigned i, unsigned p) { return warp_wait(&sm.ready[i], p); })) return true;
    if constexpr (!kLong) {
      if (on && P.chain && tile % kSuper == kSuper - 1 && tile + 1 < P.tiles) {
        const float h = sm.edge[stage].h[c];
        publish_word(P.section + ((tile / kSuper + 1) * A.width + d), cut ? h : fmaf(sm.edge[stage].a[c], in, h));
      }
    }
    if (c < 32 * V) {
      sm.edge[stage].in[c] = in;
      if constexpr (kBackward) sm.edge[stage].front[c] = (on && pl.rec.open) ? __ldg(A.carry + (pl.tile * A.width + d)) : 0.0f;
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&sm.entered[stage]);
    if (++stage == Shared::kStages) {
      stage = 0;
      parity ^= 1u;
    }
  }
}

// Publishers.  In place of its own pair every warp finds that of all rows before it in the tile (h: forward) and, going
// backward, that of all rows behind it (c).
template <typename TX, typename TA, int V, int kGate, bool kBackward>
__device__ __forceinline__ bool publish_tiles(const Params &P, StreamShared<TX, TA, V, kGate, kBackward> &sm, int c, int lane) {
  using Shared = StreamShared<TX, TA, V, kGate, kBackward>;
  Turn<Shared::kStages> now;
  Turn<kRing> pair;
  for (;; pair.next(), now.next()) {
    if (!warp_wait(&sm.full[now.i], now.parity)) return true;
    const Plan &pl = sm.plan[now.i];
    if (!pl.valid) return false;
    if (!warp_wait(&sm.paired[pair.i], pair.parity)) return true;
    if (c < pl.cols) {
      auto &pr = sm.pairs[pair.i];
      const unsigned starts = pl.rec.starts;
      float a[kWarps], h[kWarps], ta = 1.0f, th = 0.0f;
#pragma unroll
      for (int q = 0; q < kWarps; ++q) { a[q] = pr.a[q][c]; h[q] = pr.h[q][c]; }
#pragma unroll
      for (int q = 0; q < kWarps; ++q) {
        pr.a[q][c] = ta;
        pr.h[q][c] = th;
        th = (starts >> q & 1u) ? h[q] : fmaf(a[q], th, h[q]);
        ta *= a[q];
      }
      int at = pl.tile;
      if constexpr (kBackward) {
        const unsigned ends = pl.rec.ends;
        at = static_cast<int>(P.tiles) - 1 - at;
#pragma unroll
        for (int q = 0; q < kWarps; ++q) h[q] = pr.c[q][c];
        ta = 1.0f;
        th = 0.0f;
#pragma unroll
        for (int q = kWarps - 1; q >= 0; --q) {
          pr.b[q][c] = ta;
          pr.c[q][c] = th;
          th = (ends >> q & 1u) ? h[q] : fmaf(a[q], th, h[q]);
          ta *= a[q];
        }
      }
      if (P.chain) publish_pair(P.agg + (at * P.A.width + pl.d0 + c), ta, th);
      sm.edge[now.i].a[c] = ta;
      sm.edge[now.i].h[c] = th;
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&sm.ready[pair.i]);
  }
}

template <typename TX, typename TA, int V, int kGate>
__device__ __forceinline__ bool compute_forward(const Params &P, StreamShared<TX, TA, V, kGate, false> &sm, unsigned &m,
                                                int warp, int lane) {
  using Shared = StreamShared<TX, TA, V, kGate, false>;
  static_assert(kGate != kOne, "forward calls take a table of gates");
  constexpr int kG = V, R = kRows;
  const gearb_recurrence_args &A = P.A;
  Turn<Shared::kStages> now, old;
  Turn<kRing> pair, opair;
  unsigned tiles = 0xffffffffu;  // of this CTA, known when the issuer has said that there are no more
  for (m = 0; m < kLag || m - kLag < tiles; ++m) {
    if (tiles == 0xffffffffu) {
      if (!warp_wait(&sm.full[now.i], now.parity)) return true;
      if (!sm.plan[now.i].valid) tiles = m;
    }
    if (m < tiles) {
      const unsigned stage = now.i;
      const Plan &pl = sm.plan[stage];
      const WarpRows<TX, TA, V, kGate, false> rows(P, pl, sm, stage, warp, lane);
      float a[kG], ca[V], ch[V], x[V];
#pragma unroll
      for (int v = 0; v < V; ++v) { ca[v] = 1.0f; ch[v] = 0.0f; }
      if (pl.rec.dead) {
      } else if (pl.rec.plain) {
#pragma unroll
        for (int k = 0; k < R; ++k) {
          rows.get_a(k, A.gate_log, true, a);
          rows.get_x(k, x);
          fma_v(ch, a, ch, x);
          mul_v(ca, a, ca);
        }
      } else {
        const unsigned start = pl.rec.start[warp];
        const int d = pl.d0 + lane * V;
        const bool on = lane * V < pl.cols;
        float as[R][kG], xs[R][V];
#pragma unroll
        for (int k = 0; k < R; ++k) {
          rows.get_a(k, A.gate_log, true, as[k]);
          rows.get_x(k, xs[k]);
        }
#pragma unroll
        for (int k = 0; k < R; ++k) {
          mul_v(ca, as[k], ca);
          step_row(A, pl, start, k, warp * R + k, d, on, as[k], xs[k], ch);
        }
      }
      if (m >= kRing && !warp_wait(&sm.read[pair.i], pair.parity ^ 1u)) return true;
      store_pack<float, V>(&sm.pairs[pair.i].a[warp][lane * V], ca);
      store_pack<float, V>(&sm.pairs[pair.i].h[warp][lane * V], ch);
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.paired[pair.i]);
      now.next();
      pair.next();
    }
    if (m >= kLag && m - kLag < tiles) {
      const unsigned ostage = old.i;
      const Plan &opl = sm.plan[ostage];
      const int n = opl.rows - warp * R, d = opl.d0 + lane * V;
      const bool on = lane * V < opl.cols;
      if (!warp_wait(&sm.ready[opair.i], opair.parity) || !warp_wait(&sm.entered[ostage], old.parity)) return true;
      float a[kG], h[V], x[V], in[V];
      unpack(*reinterpret_cast<const Pack<float, V> *>(&sm.pairs[opair.i].h[warp][lane * V]), h);
      if (!(opl.rec.cut >> warp & 1u)) {
        float pa[V];
        unpack(*reinterpret_cast<const Pack<float, V> *>(&sm.pairs[opair.i].a[warp][lane * V]), pa);
        unpack(*reinterpret_cast<const Pack<float, V> *>(&sm.edge[ostage].in[lane * V]), in);
        fma_v(h, pa, in, h);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.read[opair.i]);
      if (n > 0) {
        const WarpRows<TX, TA, V, kGate, false> rows(P, opl, sm, ostage, warp, lane);
        const int64_t step = A.reverse ? -A.width : A.width;
        TX *out = static_cast<TX *>(A.out) + ((A.reverse ? opl.row0 - warp * R : opl.row0 + warp * R) * A.width + d);
        if (opl.rec.plain) {
#pragma unroll
          for (int k = 0; k < R; ++k) {
            rows.get_a(k, A.gate_log, false, a);
            rows.get_x(k, x);
            fma_v(h, a, h, x);
            if (on) store_pack<TX, V>(out, h);
            out += step;
          }
        } else {
          const unsigned live = opl.rec.live[warp], start = opl.rec.start[warp], end = opl.rec.end[warp];
          float as[R][kG], xs[R][V];
#pragma unroll
          for (int k = 0; k < R; ++k) {
            rows.get_a(k, A.gate_log, false, as[k]);
            rows.get_x(k, xs[k]);
          }
#pragma unroll
          for (int k = 0; k < R; ++k) {
            step_row(A, opl, start, k, warp * R + k, d, on, as[k], xs[k], h);
            const bool lv = live >> k & 1u;
            float o[V];
#pragma unroll
            for (int v = 0; v < V; ++v) o[v] = lv ? h[v] : 0.0f;
            if (on && (lv || (A.zero_rest && k < n))) store_pack<TX, V>(out, o);
            if (end >> k & 1u) state_store<V>(A.state_out, opl.rec.seq[warp * R + k], A.width, d, on, h);
            out += step;
          }
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // a was written where the next copy will write
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.empty[ostage]);
      old.next();
      opair.next();
    }
  }
  return false;
}

template <typename TX, typename TA, int V, int kGate>
__device__ __forceinline__ bool compute_backward(const Params &P, StreamShared<TX, TA, V, kGate, true> &sm, unsigned &m,
                                                 int warp, int lane) {
  using Shared = StreamShared<TX, TA, V, kGate, true>;
  constexpr int kG = kGate == kOne ? 1 : V, R = kRows;
  const gearb_recurrence_args &A = P.A;
  Turn<Shared::kStages> now, old;
  Turn<kRing> pair, opair;
  unsigned tiles = 0xffffffffu;
  for (m = 0; m < kLag || m - kLag < tiles; ++m) {
    if (tiles == 0xffffffffu) {
      if (!warp_wait(&sm.full[now.i], now.parity)) return true;
      if (!sm.plan[now.i].valid) tiles = m;
    }
    if (m < tiles) {
      const Plan &pl = sm.plan[now.i];
      const WarpRows<TX, TA, V, kGate, true> rows(P, pl, sm, now.i, warp, lane);
      float as[R][kG], x[V], ca[V], ch[V], cc[V];
#pragma unroll
      for (int v = 0; v < V; ++v) { ca[v] = 1.0f; ch[v] = cc[v] = 0.0f; }
#pragma unroll
      for (int k = 0; k < R; ++k) rows.get_a(k, A.gate_log, true, as[k]);
      if (pl.rec.plain) {
#pragma unroll
        for (int k = 0; k < R; ++k) {
          rows.get_x(k, x);
          fma_v(ch, as[k], ch, x);
          mul_v(ca, as[k], ca);
        }
#pragma unroll
        for (int k = R - 1; k >= 0; --k) {
          rows.get_dout(k, x);
#pragma unroll
          for (int v = 0; v < V; ++v) x[v] += cc[v];
          mul_v(cc, as[k], x);
        }
      } else {
        const unsigned live = pl.rec.live[warp], start = pl.rec.start[warp], end = pl.rec.end[warp];
        const int d = pl.d0 + lane * V;
        const bool on = lane * V < pl.cols;
#pragma unroll
        for (int k = R - 1; k >= 0; --k) {
          if (end >> k & 1u) state_load<V>(A.dstate, pl.rec.seq[warp * R + k], A.width, d, on, cc);
          rows.get_dout(k, x);
          if (live >> k & 1u) {
#pragma unroll
            for (int v = 0; v < V; ++v) x[v] += cc[v];
            mul_v(cc, as[k], x);
          }
        }
#pragma unroll
        for (int k = 0; k < R; ++k) {
          rows.get_x(k, x);
          if (live >> k & 1u) {
            mul_v(ca, as[k], ca);
            step_row(A, pl, start, k, warp * R + k, d, on, as[k], x, ch);
          }
        }
      }
      if (m >= kRing && !warp_wait(&sm.read[pair.i], pair.parity ^ 1u)) return true;
      auto &pr = sm.pairs[pair.i];
      store_pack<float, V>(&pr.a[warp][lane * V], ca);
      store_pack<float, V>(&pr.h[warp][lane * V], ch);
      store_pack<float, V>(&pr.c[warp][lane * V], cc);
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.paired[pair.i]);
      now.next();
      pair.next();
    }
    if (m >= kLag && m - kLag < tiles) {
      const Plan &pl = sm.plan[old.i];
      const int n = pl.rows - warp * R, d = pl.d0 + lane * V;
      const bool on = lane * V < pl.cols;
      if (!warp_wait(&sm.ready[opair.i], opair.parity) || !warp_wait(&sm.entered[old.i], old.parity)) return true;
      float h[V], c[V], f[V], e[V];
      auto &pr = sm.pairs[opair.i];
      auto &ed = sm.edge[old.i];
      unpack(*reinterpret_cast<const Pack<float, V> *>(&pr.h[warp][lane * V]), h);
      unpack(*reinterpret_cast<const Pack<float, V> *>(&pr.c[warp][lane * V]), c);
      if (!(pl.rec.cut >> warp & 1u)) {
        unpack(*reinterpret_cast<const Pack<float, V> *>(&pr.a[warp][lane * V]), f);
        unpack(*reinterpret_cast<const Pack<float, V> *>(&ed.front[lane * V]), e);
        fma_v(h, f, e, h);
      }
      if (!(pl.rec.bcut >> warp & 1u)) {
        unpack(*reinterpret_cast<const Pack<float, V> *>(&pr.b[warp][lane * V]), f);
        unpack(*reinterpret_cast<const Pack<float, V> *>(&ed.in[lane * V]), e);
        fma_v(c, f, e, c);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.read[opair.i]);
      if (n > 0) {
        const WarpRows<TX, TA, V, kGate, true> rows(P, pl, sm, old.i, warp, lane);
        const int sign = A.reverse ? -1 : 1, row0 = pl.row0 + sign * warp * R;
        const int64_t xs = sign * A.width, gs = sign * A.gates;
        TX *dx = static_cast<TX *>(A.dx) + (row0 * A.width + d);
        TA *dgate = static_cast<TA *>(A.dgate) + (row0 * A.gates + (kGate == kOne ? pl.gate : d));
        float as[R][kG], hp[R][V], part[R], x[V];
#pragma unroll
        for (int k = 0; k < R; ++k) rows.get_a(k, A.gate_log, false, as[k]);
        if (pl.rec.plain) {
#pragma unroll
          for (int k = 0; k < R; ++k) {
            rows.get_x(k, x);
#pragma unroll
            for (int v = 0; v < V; ++v) hp[k][v] = h[v];
            fma_v(h, as[k], h, x);
          }
#pragma unroll
          for (int k = R - 1; k >= 0; --k) {
            float g[V], da[V];
            rows.get_dout(k, g);
            part[k] = 0.0f;
#pragma unroll
            for (int v = 0; v < V; ++v) g[v] += c[v];
            mul_v(c, as[k], g);
#pragma unroll
            for (int v = 0; v < V; ++v) {
              da[v] = __fmul_rn(A.gate_log ? c[v] : g[v], hp[k][v]);
              part[k] += on ? da[v] : 0.0f;
            }
            if (on) {
              store_pack<TX, V>(dx + k * xs, g);
              if constexpr (kGate == kOwn) store_pack<TA, V>(dgate + k * gs, da);
            }
          }
        } else {
          const unsigned live = pl.rec.live[warp], start = pl.rec.start[warp], end = pl.rec.end[warp];
#pragma unroll
          for (int k = 0; k < R; ++k) {
            const bool st = start >> k & 1u;
            if (st) state_load<V>(A.h0, pl.rec.seq[warp * R + k], A.width, d, on, h);  // zeros without h0
            rows.get_x(k, x);
#pragma unroll
            for (int v = 0; v < V; ++v) hp[k][v] = h[v];
            if (live >> k & 1u) {
              if (st && !A.h0) {
#pragma unroll
                for (int v = 0; v < V; ++v) h[v] = x[v];
              } else {
                fma_v(h, as[k], h, x);
              }
            }
          }
#pragma unroll
          for (int k = R - 1; k >= 0; --k) {
            const bool lv = live >> k & 1u, st = start >> k & 1u;
            if (end >> k & 1u) state_load<V>(A.dstate, pl.rec.seq[warp * R + k], A.width, d, on, c);
            float g[V], da[V];
            rows.get_dout(k, g);
            part[k] = 0.0f;
#pragma unroll
            for (int v = 0; v < V; ++v) {
              const float av = as[k][kGate == kOne ? 0 : v];
              g[v] = lv ? g[v] + c[v] : 0.0f;
              if (lv) c[v] = __fmul_rn(av, g[v]);
              // the first row of a sequence without h0 is h = x: its gate plays no part
              da[v] = (lv && !(st && !A.h0)) ? __fmul_rn(A.gate_log ? c[v] : g[v], hp[k][v]) : 0.0f;
              part[k] += on ? da[v] : 0.0f;
            }
            if (on && (lv || (A.zero_rest && k < n))) {
              store_pack<TX, V>(dx + k * xs, g);
              if constexpr (kGate == kOwn) store_pack<TA, V>(dgate + k * gs, da);
            }
            if (st) state_store<V>(A.dh0, pl.rec.seq[warp * R + k], A.width, d, on, c);
          }
        }
        if constexpr (kGate == kOne) {
          const float sum = sum_rows(part, lane);
          const int k = row_of_lane(lane);
          if (lane % kSpare == 0 && k < n && ((pl.rec.live[warp] >> k & 1u) || A.zero_rest)) {
            if (P.blocks_per_gate == 1) dgate[k * gs] = from_f<TA>(sum);
            else P.gate_part[(pl.part * P.rows + row0 + k * sign) * A.gates + pl.gate] = sum;
          }
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // a was written where the next copy will write
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.empty[old.i]);
      old.next();
      opair.next();
    }
  }
  return false;
}

// What an item's rows, states and published words hold when it was given up: NaN, but for rows of no sequence and words
// that were there already.  All threads.
template <typename TX, typename TA, int V, int kGate, bool kBackward>
__device__ void give_up_item(const Params &P, unsigned item) {
  const gearb_recurrence_args &A = P.A;
  const float nan = __uint_as_float(0x7fffffffu);
  const Place at = place_of_item<V, kGate, kBackward>(P, item);
  const TileRec &rec = P.recs[at.tile];
  const int n = static_cast<int>(at.i1 - at.i0), cols = static_cast<int>(at.d1 - at.d0 < 32 * V ? at.d1 - at.d0 : 32 * V);
  TX *rows = static_cast<TX *>(kBackward ? A.dx : A.out);
  float *states = kBackward ? A.dh0 : A.state_out;
  for (int e = threadIdx.x; e < n * cols; e += kStreamThreads) {
    const int k = e / cols;
    const int64_t row = row_of(P, at.i0 + k), d = at.d0 + (e - k * cols);
    const bool live = rec.live[k / kRows] >> (k % kRows) & 1u;
    const float v = live ? nan : 0.0f;
    if (live || A.zero_rest) {
      rows[row * A.width + d] = from_f<TX>(v);
      if (kBackward && kGate == kOwn) static_cast<TA *>(A.dgate)[row * A.gates + d] = from_f<TA>(v);
      if (kBackward && kGate == kOne && e == k * cols) {
        if (P.blocks_per_gate == 1) static_cast<TA *>(A.dgate)[row * A.gates + at.gate] = from_f<TA>(v);
        else P.gate_part[(at.part * P.rows + row) * A.gates + at.gate] = v;
      }
    }
    if (states && ((kBackward ? rec.start : rec.end)[k / kRows] >> (k % kRows) & 1u))
      states[static_cast<int64_t>(rec.seq[k]) * A.width + d] = nan;
  }
  if (!P.chain) return;
  const int64_t t = kBackward ? P.tiles - 1 - at.tile : at.tile, sb = t / kSuper, sec = t >> P.section_shift;
  for (int c = threadIdx.x; c < cols; c += kStreamThreads) {
    const int64_t d = at.d0 + c;
    if (!kBackward && A.carry && rec.open) A.carry[at.tile * A.width + d] = nan;
    auto unset = [](const float2 &q) { return __float_as_uint(q.x) == kUnset || __float_as_uint(q.y) == kUnset; };
    float2 *own = P.agg + t * A.width + d;
    if (unset(peek_pair(own))) publish_pair(own, nan, nan);
    if (t % kSuper != kSuper - 1 || t + 1 >= P.tiles) continue;
    if (t + 1 == (sec + 1) << P.section_shift) {
      float *state = P.section + (sec + 1) * A.width + d;
      bool seen = true;
      if (poll_word(reinterpret_cast<const unsigned *>(state), 0, seen) == 0x7fffffffu) publish_word(state, nan);
    } else if (unset(peek_pair(P.super + sb * A.width + d))) {
      publish_pair(P.super + sb * A.width + d, nan, nan);
    }
  }
}

// A wait ran into its limit: the roles have ended somewhere.  Copies under way have to land before the CTA leaves its shared
// memory; tiles that are not done, and those that nobody has taken, are given up, so that no row is left unwritten and no
// CTA waits for what will not come.  All threads.
template <typename TX, typename TA, int V, int kGate, bool kBackward>
__device__ __noinline__ void abandon(const Params &P, StreamShared<TX, TA, V, kGate, kBackward> &sm) {
  constexpr unsigned kStages = StreamShared<TX, TA, V, kGate, kBackward>::kStages;
  unsigned from = sm.done[0];
  for (int w = 1; w < kWarps; ++w) from = sm.done[w] < from ? sm.done[w] : from;
  const unsigned to = sm.issued_tiles;  // at most kStages more: a stage is used again when all warps are done with it
  if (threadIdx.x == 0) {
    if (P.A.status) atomicOr(reinterpret_cast<unsigned *>(P.A.status), GEARB_ST_SCAN_ABORTED);
    bool recorded[kRecorders];  // whether the recorder has been at the tiles so far
    for (int r = 0; r < kRecorders; ++r) recorded[r] = true;
    for (unsigned m = from; m < to; ++m) {
      const unsigned stage = m % kStages, r = m % kRecorders;
      if (is_turn(sm.recorded[r], m)) recorded[r] = false;
      if (!recorded[r]) mbar_arrive(&sm.full[stage]);  // in its recorder's place
      mbar_wait(&sm.full[stage], m / kStages & 1u);
    }
  }
  __syncthreads();
  for (unsigned m = from; m < to; ++m) give_up_item<TX, TA, V, kGate, kBackward>(P, sm.item[m % kStages]);
  const Items items = items_of<kBackward>(P);
  for (;;) {
    const unsigned item = sm.next;
    if (item >= items.end) return;
    give_up_item<TX, TA, V, kGate, kBackward>(P, item);
    __syncthreads();
    if (threadIdx.x == 0) sm.next = item_behind(P, items, item);
    __syncthreads();
  }
}

template <typename TX, typename TA, int V, int kGate, bool kBackward>
__device__ __forceinline__ void init_barriers(StreamShared<TX, TA, V, kGate, kBackward> &sm) {
  if (threadIdx.x == 0) {
    for (unsigned s = 0; s < StreamShared<TX, TA, V, kGate, kBackward>::kStages; ++s) {
      mbar_init_count(&sm.full[s], 2);  // the issuer (and its copies' bytes), the recorder
      mbar_init_count(&sm.empty[s], kWarps);
      mbar_init_count(&sm.entered[s], 4);
      mbar_init_count(&sm.issued[s], 1);
    }
    for (unsigned s = 0; s < kRing; ++s) {
      mbar_init_count(&sm.paired[s], kWarps);
      mbar_init_count(&sm.ready[s], 4);
      mbar_init_count(&sm.read[s], kWarps);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
}

template <typename TX, typename TA, int V, int kGate, bool kLong>
__global__ void __launch_bounds__(kStreamThreads, 1) forward_stream_kernel(const __grid_constant__ Params P,
                                                                           const __grid_constant__ Maps maps) {
  using Shared = StreamShared<TX, TA, V, kGate, false>;
  extern __shared__ __align__(1024) unsigned char raw_smem[];
  auto &sm = *reinterpret_cast<Shared *>(raw_smem);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  init_barriers(sm);
  bool lost = false;
  if (warp == kWarps + 8 + kRecorders) {
    if (lane == 0) lost = issue_tiles<TX, TA, V, kGate, false>(P, maps, sm);
  } else if (P.no_waits) {
    lost = true;
    if (threadIdx.x < kWarps) sm.done[threadIdx.x] = 0;
    if (threadIdx.x < kRecorders) {
      sm.recorded[threadIdx.x].i = threadIdx.x;
      sm.recorded[threadIdx.x].parity = 0;
    }
  } else if (warp < kWarps) {
    unsigned m;
    lost = compute_forward<TX, TA, V, kGate>(P, sm, m, warp, lane);
    if (lane == 0) sm.done[warp] = m < kLag ? 0 : m - kLag;
  } else if (warp < kWarps + 4) {
    lost = publish_tiles<TX, TA, V, kGate, false>(P, sm, threadIdx.x - kThreads, lane);
  } else if (warp < kWarps + 8) {
    lost = finish_tiles<TX, TA, V, kGate, false, kLong>(P, sm, threadIdx.x - kThreads - 128, lane);
  } else {
    lost = record_tiles<TX, TA, V, kGate, false>(P, sm, warp - kWarps - 8, lane);
  }
  __syncwarp();
  if (__syncthreads_or(lost)) abandon(P, sm);
}

template <typename TX, typename TA, int V, int kGate, bool kLong>
__global__ void __launch_bounds__(kStreamThreads, 1) backward_stream_kernel(const __grid_constant__ Params P,
                                                                            const __grid_constant__ Maps maps) {
  using Shared = StreamShared<TX, TA, V, kGate, true>;
  extern __shared__ __align__(1024) unsigned char raw_smem[];
  auto &sm = *reinterpret_cast<Shared *>(raw_smem);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  init_barriers(sm);
  bool lost = false;
  if (warp == kWarps + 8 + kRecorders) {
    if (lane == 0) lost = issue_tiles<TX, TA, V, kGate, true>(P, maps, sm);
  } else if (P.no_waits) {
    lost = true;
    if (threadIdx.x < kWarps) sm.done[threadIdx.x] = 0;
    if (threadIdx.x < kRecorders) {
      sm.recorded[threadIdx.x].i = threadIdx.x;
      sm.recorded[threadIdx.x].parity = 0;
    }
  } else if (warp < kWarps) {
    unsigned m;
    lost = compute_backward<TX, TA, V, kGate>(P, sm, m, warp, lane);
    if (lane == 0) sm.done[warp] = m < kLag ? 0 : m - kLag;
  } else if (warp < kWarps + 4) {
    lost = publish_tiles<TX, TA, V, kGate, true>(P, sm, threadIdx.x - kThreads, lane);
  } else if (warp < kWarps + 8) {
    lost = finish_tiles<TX, TA, V, kGate, true, kLong>(P, sm, threadIdx.x - kThreads - 128, lane);
  } else {
    lost = record_tiles<TX, TA, V, kGate, true>(P, sm, warp - kWarps - 8, lane);
  }
  __syncwarp();
  if (__syncthreads_or(lost)) abandon(P, sm);
}

// A matrix of [rows][width] for boxes of kTile rows and 32 * V channels.
template <typename T>
int make_map(CUtensorMap *map, const void *base, int64_t width, int64_t rows, int64_t row_stride, int box) {
  const CUtensorMapDataType type = sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16;
  return encode_map(map, type, const_cast<void *>(base), width, rows, row_stride * static_cast<int64_t>(sizeof(T)), box, kTile);
}

template <typename TX, typename TA, int V, int kGate, bool kBackward>
int launch_stream(Params &p, cudaStream_t stream) {
  const gearb_recurrence_args &a = p.A;
  p.blocks_per_gate = kGate == kOne ? (p.per + 32 * V - 1) / (32 * V) : 1;
  const int64_t ncol = kGate == kOne ? a.gates * p.blocks_per_gate : (a.width + 32 * V - 1) / (32 * V);
  // Items are counted in 32 bits, and every CTA takes numbers beyond the last.
  GEARB_REQUIRE(p.tiles <= (int64_t(1) << 31) / ncol - 1, "recurrence: too many tiles for one launch");
  p.ncol = static_cast<int>(ncol);
  int rc = launch_prepare(p, stream);
  if (rc != GEARB_OK) return rc;
  Maps maps;
  rc = make_map<TX>(&maps.x, a.x, a.width, p.rows, a.x_row_stride, 32 * V);
  if (rc == GEARB_OK && kGate == kOwn) rc = make_map<TA>(&maps.gate, a.gate, a.width, p.rows, a.gate_row_stride, 32 * V);
  if (rc == GEARB_OK && kBackward) rc = make_map<TX>(&maps.dout, a.dout, a.width, p.rows, a.dout_row_stride, 32 * V);
  if (rc != GEARB_OK) return rc;
  constexpr int kSmem = sizeof(StreamShared<TX, TA, V, kGate, kBackward>);
  static_assert(kSmem <= kSmemMost, "fits one SM");
  void (*kernel)(Params, Maps);
  // a kernel each: with both ways in one, packed heads take 10 % longer
  p.section_shift = section_shift_of(p);
  const bool far = p.chain && p.section_shift == kLongSection;
  if constexpr (kBackward) kernel = far ? backward_stream_kernel<TX, TA, V, kGate, true> : backward_stream_kernel<TX, TA, V, kGate, false>;
  else kernel = far ? forward_stream_kernel<TX, TA, V, kGate, true> : forward_stream_kernel<TX, TA, V, kGate, false>;
  GEARB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
  const int64_t most = sm_count(), items = p.tiles * ncol;
  kernel<<<static_cast<unsigned>(items < most ? items : most), kStreamThreads, kSmem, stream>>>(p, maps);
  GEARB_CUDA(cudaGetLastError());
  return GEARB_OK;
}

// TMA takes a matrix whose base and rows start on 16 bytes, and copies that start on 16 bytes; rows that overlap (sr below
// the width) are not among the layouts that its documentation describes.
inline bool matrix_ok(const void *p, int64_t width, int64_t sr, int size) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && sr >= width && sr < (int64_t(1) << 37) && sr * size % 16 == 0;
}

// Channels a lane in the streaming kernel, 0: not for it.
template <typename TX, typename TA>
int stream_width(const Params &p, bool backward) {
  const gearb_recurrence_args &a = p.A;
  const bool shared = a.gates < a.width;
  if (!p.flat || p.rows >= (int64_t(1) << 31) || !matrix_ok(a.x, a.width, a.x_row_stride, sizeof(TX))) return 0;
  if (!shared && !matrix_ok(a.gate, a.width, a.gate_row_stride, sizeof(TA))) return 0;
  if (backward) {
    if (!matrix_ok(a.dout, a.width, a.dout_row_stride, sizeof(TX)) || a.width % 2 != 0) return 0;
    if (!vector_ok(a.dx, 0, 0, sizeof(TX), 2) || (!shared && !vector_ok(a.dgate, 0, 0, sizeof(TA), 2))) return 0;
    if (shared ? (p.per <= 32 || p.per * sizeof(TX) % 16 != 0) : a.width <= 32) return 0;
    return 2;
  }
  if (a.width <= 32 || a.width % 2 != 0) return 0;
  // a block's channels may span as many gates as the table holds
  auto spans = [&](int v) { return !shared || (32 * v - 2) / p.per + 2 <= kTableGates; };
  const bool four = a.width > 64 && a.width % 4 == 0 && vector_ok(a.out, 0, 0, sizeof(TX), 4) && spans(4);
  if (four && (shared || sizeof(TX) + sizeof(TA) <= 6)) return 4;
  return vector_ok(a.out, 0, 0, sizeof(TX), 2) && spans(2) ? 2 : 0;
}

template <typename TX, typename TA>
int launch_any(Params &p, bool backward, cudaStream_t stream) {
  if (p.narrow_rows == 16) return launch_narrow<TX, TA, 16>(p, backward, stream);
  if (p.narrow_rows == 4) return launch_narrow<TX, TA, 4>(p, backward, stream);
  const int v = stream_width<TX, TA>(p, backward);
  const bool shared = p.A.gates < p.A.width;
  if (v == 0) return launch_wide_any<TX, TA>(p, backward, stream);
  if (backward)
    return shared ? launch_stream<TX, TA, 2, kOne, true>(p, stream) : launch_stream<TX, TA, 2, kOwn, true>(p, stream);
  if (shared)
    return v == 4 ? launch_stream<TX, TA, 4, kTable, false>(p, stream) : launch_stream<TX, TA, 2, kTable, false>(p, stream);
  // four channels of eight bytes would leave room for two tiles
  if constexpr (sizeof(TX) + sizeof(TA) <= 6)
    if (v == 4) return launch_stream<TX, TA, 4, kOwn, false>(p, stream);
  return launch_stream<TX, TA, 2, kOwn, false>(p, stream);
}

}  // namespace rec
}  // namespace gearb
