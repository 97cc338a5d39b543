// Kernels of the recurrences for long calls whose rows lie in one TMA-addressable matrix.
//
// The tiles are those of recurrence_wide.cuh, but the CTAs stay, one per SM, and their warps have roles, so that
// nothing waits in line:
//   planner     takes the next tile's number from the counter, works out once for everybody where the tile lies and
//               which rows start or end a sequence, and starts its copies (one tensor copy per input)
//   compute     first look at tile m: (A, H) of each warp's rows; then, tile m - 1 again: its rows from the state
//               before them, and out
//   publishers  one thread per channel: turn the warps' pairs into those of all rows before each warp, publish the
//               tile's
//   finishers   one thread per channel: the state in front of the tile from what the tiles before published
// They meet at mbarriers only.  Measured on the way, 2 x 16384 x 2048 bf16 with float32 gates (82 us at the copy rate):
// a CTA per tile 170 us whatever the types; CTAs that stay but finish a tile before they begin the next: every tile
// spent 6700 of 11000 cycles looking back; one bulk copy per row: an SM starts one about every 35 cycles, 180 us;
// every warp finding its rows' place itself: 600 of 1000 instructions; both phases' rows in registers: spills, 234 us;
// several tiles' numbers taken at once: tiles wait for others far back in another CTA's queue, 250 to 600 us; two CTA
// barriers a tile in place of the roles: 136 us.
#pragma once

#include <cuda.h>

#include "recurrence_wide.cuh"

namespace gearb {
namespace rec {

constexpr int kStreamThreads = kThreads + 9 * 32;  // compute, 4 publishers, 4 finishers, planner
constexpr int kSmemMost = 227 * 1024;
#ifndef GEARB_REC_STAGES
#define GEARB_REC_STAGES 6
#endif

constexpr unsigned kWaitLimit = 1u << 20;  // mbarrier polls before a copy is declared lost

__device__ __forceinline__ uint32_t smem_addr(const void *p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void mbar_init(uint64_t *bar) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_addr(bar)));
}
__device__ __forceinline__ void mbar_expect(uint64_t *bar, unsigned bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_addr(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_wait(uint64_t *bar, unsigned parity) {
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
template <typename TX, typename TA, int V, bool kShared, bool kBackward>
struct Stage {
  alignas(128) TX x[kTile][32 * V];
  alignas(128) TX dout[kBackward ? kTile : 1][kBackward ? 32 * V : 8];
  alignas(128) TA gate[kShared ? 1 : kTile][kShared ? 8 : 32 * V];
  static constexpr unsigned kBytes = sizeof(TX) * 32 * V * kTile * (kBackward ? 2 : 1) +
                                     (kShared ? 0 : sizeof(TA) * 32 * V * kTile);
};

// What the planning warp works out about a tile.  Rows are counted in 32 bits here (the entry point sends longer calls
// elsewhere).
struct Plan {
  int valid;
  int tile, rows;  // rows of the scan in it
  int row0;        // matrix row of the first of them; the others follow it, or precede it in a reverse call
  int d0, cols;    // first channel, channels
  int gate, part;  // shared gates: the gate, and which block of its channels
  int plain;       // one sequence goes through the whole tile: no row of it is its first or last
  int lo;          // look back as far as this tile, counted in the order of the tickets; -1: nothing is needed from before
  int open;        // backward: the first row continues a sequence of an earlier tile
  unsigned starts, ends;  // bit w: a sequence starts (ends) in warp w's rows
  unsigned cut;    // bit w: a sequence starts in rows of the tile before warp w's (bit kWarps: anywhere in it)
  unsigned bcut;   // bit w: a sequence ends in rows of the tile behind warp w's (bit kWarps: anywhere in it)
  alignas(16) unsigned char live[kWarps], start[kWarps], end[kWarps];  // bits: rows of each warp
  int seq[kTile];                                                     // sequence of each row (unless plain)
  float a[kTile];                                                     // shared gates: a of each row
};

template <int V, bool kBackward>
struct Pairs {  // of the warps of one tile; then of all rows before (backward: behind) each warp's
  alignas(16) float a[kWarps][32 * V];
  alignas(16) float h[kWarps][32 * V];
  alignas(16) float b[kBackward ? kWarps : 1][kBackward ? 32 * V : 4];
  alignas(16) float c[kBackward ? kWarps : 1][kBackward ? 32 * V : 4];
};
template <int V>
struct Edge {  // of one tile: its own pair, and the state in front of it
  float a[32 * V], h[32 * V], in[32 * V];
};

template <typename TX, typename TA, int V, bool kShared, bool kBackward>
struct StreamShared {
  using StageT = Stage<TX, TA, V, kShared, kBackward>;
  static constexpr int kEach = static_cast<int>(sizeof(StageT) + sizeof(Edge<V>) + sizeof(Plan)) + 64;
  static constexpr int kFit = (kSmemMost - 2 * static_cast<int>(sizeof(Pairs<V, kBackward>)) - 256) / kEach;
  static constexpr unsigned kStages = kFit > GEARB_REC_STAGES ? GEARB_REC_STAGES : kFit;
  static_assert(kStages >= 3, "two tiles in work and one on its way");
  StageT stage[kStages];
  Pairs<V, kBackward> pairs[2];
  Edge<V> edge[kStages];
  Plan plan[kStages];
  uint64_t full[kStages], empty[kStages];  // the tile's rows and plan are there; the tile is done with
  uint64_t entered[kStages];               // edge.in is there
  uint64_t paired[2], ready[2], read[2];   // the warps' pairs; turned and edge.a, edge.h there; read again
};

// The tile before (in the order of the tickets): what its predecessors published, asked for early.
struct Peek {
  float2 q[kSuper - 1];
  float s;
};
__device__ __forceinline__ void peek_back(const Params &P, int at, int lo, int d, Peek &k) {
  const int sb = at / kSuper, sb0 = sb * kSuper;
  const bool need_super = lo < sb0;
  const int j0 = need_super ? sb0 : lo, count = at - j0;
  const float2 *p = P.agg + j0 * P.A.width + d;
#pragma unroll
  for (int u = 0; u < kSuper - 1; ++u)
    if (u < count) k.q[u] = peek_pair(p + u * P.A.width);
  if (need_super) {
    unsigned w;
    asm volatile("ld.relaxed.gpu.global.u32 %0, [%1];" : "=r"(w) : "l"(P.super + sb * P.A.width + d) : "memory");
    k.s = __uint_as_float(w);
  }
}
// The state in front of tile `at`: as look_back, from what was peeked at, waiting for what was not there yet.
__device__ __forceinline__ float settle_back(const Params &P, int at, int lo, int d, Peek &k, bool &lost) {
  const int sb = at / kSuper, sb0 = sb * kSuper;
  const bool need_super = lo < sb0;
  const int j0 = need_super ? sb0 : lo, count = at - j0;
  const float2 *p = P.agg + j0 * P.A.width + d;
  float pa = 1.0f, ph = 0.0f;
#pragma unroll
  for (int u = 0; u < kSuper - 1; ++u)
    if (u < count) {
      if (__float_as_uint(k.q[u].x) == kUnset || __float_as_uint(k.q[u].y) == kUnset)
        k.q[u] = poll_pair(p + u * P.A.width, lost);
      ph = (u == 0 && !need_super) ? k.q[u].y : fmaf(k.q[u].x, ph, k.q[u].y);
      pa *= k.q[u].x;
    }
  if (!need_super) return ph;
  if (__float_as_uint(k.s) == kUnset)
    k.s = __uint_as_float(poll_word(reinterpret_cast<const unsigned *>(P.super + sb * P.A.width + d), lost));
  return fmaf(pa, k.s, ph);
}

// The planning warp.
template <typename TX, typename TA, int V, bool kShared, bool kBackward>
__device__ __forceinline__ void plan_tiles(const Params &P, const Maps &maps, StreamShared<TX, TA, V, kShared, kBackward> &sm,
                                           int lane) {
  using Shared = StreamShared<TX, TA, V, kShared, kBackward>;
  constexpr unsigned kStages = Shared::kStages;
  const gearb_recurrence_args &A = P.A;
  const unsigned items = static_cast<unsigned>(P.tiles * P.ncol);
  // lane 0: the next number.  One at a time from the start: CTAs that took several at once would come to tiles much
  // later than others come to the tiles behind them, and those would wait.
  unsigned next = 0;
  if (lane == 0) next = P.chain ? atomicAdd(P.ticket, 1u) + 1u : blockIdx.x;  // the counter starts at 0xffffffff
  unsigned stage = 0, parity = 0;
  for (unsigned m = 0;; ++m) {
    if (m >= kStages) {
      const bool free = mbar_wait(&sm.empty[stage], parity ^ 1u);
      if (!__all_sync(kAll, free)) {  // a warp of this CTA is stuck: nothing more is started
        if (lane == 0 && A.status) atomicOr(reinterpret_cast<unsigned *>(A.status), GEARB_ST_SCAN_ABORTED);
        return;
      }
    }
    const unsigned item = __shfl_sync(kAll, next, 0);
    Plan &pl = sm.plan[stage];
    if (item >= items) {
      if (lane == 0) {
        pl.valid = 0;
        mbar_arrive(&sm.full[stage]);
        mbar_arrive(&sm.full[stage]);
      }
      return;
    }
    if (lane == 0) {  // asked for now, needed a tile later
      next = P.chain ? atomicAdd(P.ticket, 1u) + 1u : item + gridDim.x;
    }
    Place at;
    const unsigned t = item / static_cast<unsigned>(P.ncol);
    const int c = static_cast<int>(item - t * static_cast<unsigned>(P.ncol));
    at.tile = kBackward ? P.tiles - 1 - t : t;
    at.i0 = at.tile * P.tile_rows;
    at.i1 = at.i0 + P.tile_rows < P.rows ? at.i0 + P.tile_rows : P.rows;
    at.gate = kShared ? c / P.blocks_per_gate : 0;
    at.part = kShared ? c - static_cast<int>(at.gate) * P.blocks_per_gate : 0;
    at.d0 = kShared ? at.gate * P.per + at.part * 32 * V : c * 32 * V;
    at.d1 = kShared ? (at.gate + 1) * P.per : A.width;
    const int n = static_cast<int>(at.i1 - at.i0);
    const int row0 = static_cast<int>(row_of(P, at.i0));
    if (lane == 0) {
      // a reverse call's tile ends at row0: its box begins kTile - 1 rows before, if need be in front of the matrix
      const int bc = static_cast<int>(at.d0), br = A.reverse ? row0 - (kTile - 1) : row0;
      mbar_expect(&sm.full[stage], Shared::StageT::kBytes);  // arrives below
      tensor_load(sm.stage[stage].x, &maps.x, bc, br, &sm.full[stage]);
      if constexpr (!kShared) tensor_load(sm.stage[stage].gate, &maps.gate, bc, br, &sm.full[stage]);
      if constexpr (kBackward) tensor_load(sm.stage[stage].dout, &maps.dout, bc, br, &sm.full[stage]);
    }
    if constexpr (kShared) {
#pragma unroll
      for (int k = lane; k < kTile; k += 32) {
        float own = 0.0f;
        if (k < n)
          own = to_f(static_cast<const TA *>(A.gate)[(A.reverse ? row0 - k : row0 + k) * A.gate_row_stride + at.gate]);
        pl.a[k] = A.gate_log ? exp_of(own) : own;
      }
    }
    const TileRows tr = A.offsets ? tile_rows_packed(P, at, lane) : tile_rows_dense(P, at);
    int64_t first_start = tr.first_start, last_end = tr.last_end;
    bool first_open = true, last_open = true;  // the first (last) row's sequence began (goes on) elsewhere
    if (!tr.interior) {
#pragma unroll
      for (int half = 0; half < kTile / 32; ++half) {
        const int n0 = n - half * 32, nn = n0 < 0 ? 0 : (n0 > 32 ? 32 : n0);
        const RowMap rm = map_rows(A, P.rows, at.i0 + half * 32, nn, lane);
        pl.seq[half * 32 + lane] = rm.seq;
        if (lane < 32 / kRows) {
          const int w = half * (32 / kRows) + lane;
          pl.live[w] = static_cast<unsigned char>(rm.live >> (kRows * lane) & kAllRows);
          pl.start[w] = static_cast<unsigned char>(rm.start >> (kRows * lane) & kAllRows);
          pl.end[w] = static_cast<unsigned char>(rm.end >> (kRows * lane) & kAllRows);
        }
        if (half == 0) {
          first_start = rm.first_start;
          first_open = rm.live & ~rm.start & 1u;
        }
        if (nn > 0) {
          last_end = rm.last_end;
          last_open = (rm.live & ~rm.end) >> (nn - 1) & 1u;
        }
      }
    } else if (lane < kWarps) {
      pl.live[lane] = static_cast<unsigned char>(kAllRows);
      pl.start[lane] = pl.end[lane] = 0;
    }
    __syncwarp();
    if (lane == 0) {
      pl.valid = 1;
      pl.tile = static_cast<int>(at.tile);
      pl.rows = n;
      pl.row0 = row0;
      pl.d0 = static_cast<int>(at.d0);
      pl.cols = static_cast<int>(at.d1 - at.d0 < 32 * V ? at.d1 - at.d0 : 32 * V);
      pl.gate = static_cast<int>(at.gate);
      pl.part = at.part;
      pl.plain = tr.interior;
      unsigned cut = 0, bcut = 0, starts = 0, ends = 0;
      if (!tr.interior) {
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          if (pl.start[w]) {
            starts |= 1u << w;
            cut |= ~0u << (w + 1);
          }
          if (pl.end[w]) {
            ends |= 1u << w;
            bcut |= ((1u << w) - 1u) | 1u << kWarps;
          }
        }
      }
      pl.starts = starts;
      pl.ends = ends;
      pl.cut = cut;
      pl.bcut = bcut;
      const int64_t from = quotient(first_start, P.tile_rows);
      pl.open = P.chain && first_open && from < at.tile;
      pl.lo = -1;
      if (!kBackward) {
        if (pl.open) pl.lo = static_cast<int>(from);
      } else if (P.chain && last_open) {
        const int64_t lo = P.tiles - 1 - quotient(last_end, P.tile_rows);
        if (lo < static_cast<int64_t>(t)) pl.lo = static_cast<int>(lo);
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&sm.full[stage]);  // the plan is there; the copies count themselves
    empty_sequences(P, at, 32 * V, kBackward ? A.dstate : A.h0, kBackward ? A.dh0 : A.state_out, lane);
    if (++stage == kStages) {
      stage = 0;
      parity ^= 1u;
    }
  }
}

// A warp's rows of a tile in its stage: row k of the warp (in scan order) at k * step.
template <typename TX, typename TA, int V, bool kShared, bool kBackward>
struct WarpRows {
  static constexpr int kW = 32 * V, kG = kShared ? 1 : V;
  TX *x, *dout;
  TA *gate;
  const float *shared_a;
  int step;
  __device__ __forceinline__ WarpRows(const Params &P, const Plan &pl, Stage<TX, TA, V, kShared, kBackward> &st, int warp,
                                      int lane) {
    const int k0 = P.A.reverse ? kTile - 1 - warp * kRows : warp * kRows, at = k0 * kW + lane * V;
    step = P.A.reverse ? -kW : kW;
    x = st.x[0] + at;
    dout = st.dout[0] + (kBackward ? at : 0);
    gate = st.gate[0] + (kShared ? 0 : at);
    shared_a = pl.a + warp * kRows;
  }
  __device__ __forceinline__ void get_x(int k, float (&f)[V]) const {
    unpack(*reinterpret_cast<const Pack<TX, V> *>(x + k * step), f);
  }
  __device__ __forceinline__ void get_dout(int k, float (&f)[V]) const {
    unpack(*reinterpret_cast<const Pack<TX, V> *>(dout + k * step), f);
  }
  // a of row k.  The first look turns a float32 log gate into a where it lies; a 16-bit one is turned at every look.
  __device__ __forceinline__ void get_a(int k, int log, bool first, float (&a)[kG]) const {
    if constexpr (kShared) {
      a[0] = shared_a[k];
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

// Finishers: the state in front of every tile (backward: behind it), and that in front of the next superblock.
template <typename TX, typename TA, int V, bool kShared, bool kBackward>
__device__ __forceinline__ bool finish_tiles(const Params &P, StreamShared<TX, TA, V, kShared, kBackward> &sm, int c, int lane) {
  using Shared = StreamShared<TX, TA, V, kShared, kBackward>;
  const gearb_recurrence_args &A = P.A;
  bool lost = false;
  unsigned stage = 0, parity = 0;
  for (unsigned m = 0;; ++m) {
    if (!warp_wait(&sm.full[stage], parity)) return true;
    const Plan &pl = sm.plan[stage];
    if (!pl.valid) return lost;
    const int tile = kBackward ? static_cast<int>(P.tiles) - 1 - pl.tile : pl.tile, lo = pl.lo, d = pl.d0 + c;
    const bool on = c < pl.cols;
    float in = 0.0f;
    if (on && lo >= 0) {
      Peek peek;
      peek_back(P, tile, lo, d, peek);
      in = settle_back(P, tile, lo, d, peek, lost);
      if (!kBackward && A.carry) A.carry[pl.tile * A.width + d] = in;
    }
    if (P.chain && tile % kSuper == kSuper - 1 && tile + 1 < P.tiles) {
      const bool cut = (kBackward ? pl.bcut : pl.cut) >> kWarps & 1u;
      if (!warp_wait(&sm.ready[m & 1], m >> 1 & 1u)) return true;
      if (on) {
        const float h = sm.edge[stage].h[c];
        publish_word(P.super + ((tile / kSuper + 1) * A.width + d), cut ? h : fmaf(sm.edge[stage].a[c], in, h));
      }
    }
    if (c < 32 * V) sm.edge[stage].in[c] = in;
    __syncwarp();
    if (lane == 0) mbar_arrive(&sm.entered[stage]);
    if (++stage == Shared::kStages) {
      stage = 0;
      parity ^= 1u;
    }
  }
}

template <typename TX, typename TA, int V, bool kShared>
__device__ __forceinline__ bool publish_tiles(const Params &P, StreamShared<TX, TA, V, kShared, false> &sm, int c, int lane) {
  using Shared = StreamShared<TX, TA, V, kShared, false>;
  unsigned stage = 0, parity = 0;
  for (unsigned m = 0;; ++m) {
    if (!warp_wait(&sm.full[stage], parity)) return true;
    const Plan &pl = sm.plan[stage];
    if (!pl.valid) return false;
    if (!warp_wait(&sm.paired[m & 1], m >> 1 & 1u)) return true;
    if (c < pl.cols) {
      auto &pr = sm.pairs[m & 1];
      const unsigned starts = pl.starts;
      float b[kWarps], h[kWarps], ta = 1.0f, th = 0.0f;
#pragma unroll
      for (int q = 0; q < kWarps; ++q) { b[q] = pr.a[q][c]; h[q] = pr.h[q][c]; }
#pragma unroll
      for (int q = 0; q < kWarps; ++q) {
        pr.a[q][c] = ta;
        pr.h[q][c] = th;
        th = (starts >> q & 1u) ? h[q] : fmaf(b[q], th, h[q]);
        ta *= b[q];
      }
      if (P.chain) publish_pair(P.agg + (pl.tile * P.A.width + pl.d0 + c), ta, th);
      sm.edge[stage].a[c] = ta;
      sm.edge[stage].h[c] = th;
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&sm.ready[m & 1]);
    if (++stage == Shared::kStages) {
      stage = 0;
      parity ^= 1u;
    }
  }
}

template <typename TX, typename TA, int V, bool kShared>
__device__ __forceinline__ bool compute_forward(const Params &P, StreamShared<TX, TA, V, kShared, false> &sm, int warp,
                                                int lane) {
  using Shared = StreamShared<TX, TA, V, kShared, false>;
  constexpr int kG = kShared ? 1 : V, R = kRows;
  const gearb_recurrence_args &A = P.A;
  unsigned stage = 0, parity = 0, ostage = 0, oparity = 0;
  for (unsigned m = 0;; ++m) {
    if (!warp_wait(&sm.full[stage], parity)) return true;
    const Plan &pl = sm.plan[stage];
    const bool valid = pl.valid;
    if (valid) {
      const WarpRows<TX, TA, V, kShared, false> rows(P, pl, sm.stage[stage], warp, lane);
      float a[kG], ca[V], ch[V], x[V];
#pragma unroll
      for (int v = 0; v < V; ++v) { ca[v] = 1.0f; ch[v] = 0.0f; }
      if (pl.plain) {
#pragma unroll
        for (int k = 0; k < R; ++k) {
          rows.get_a(k, A.gate_log, true, a);
          rows.get_x(k, x);
          fma_v(ch, a, ch, x);
          mul_v(ca, a, ca);
        }
      } else {
        const unsigned live = pl.live[warp], start = pl.start[warp];
        const int d = pl.d0 + lane * V;
#pragma unroll
        for (int k = 0; k < R; ++k) {
          rows.get_a(k, A.gate_log, true, a);
          if (!(live >> k & 1u)) continue;
          rows.get_x(k, x);
          if (start >> k & 1u) {
            if (A.h0) {
              float h0[V];
              state_load<V>(A.h0, pl.seq[warp * R + k], A.width, d, lane * V < pl.cols, h0);
              fma_v(ch, a, h0, x);
            } else {
#pragma unroll
              for (int v = 0; v < V; ++v) ch[v] = x[v];
            }
          } else {
            fma_v(ch, a, ch, x);
          }
          mul_v(ca, a, ca);
        }
      }
      if (m >= 2 && !warp_wait(&sm.read[m & 1], (m >> 1) - 1u & 1u)) return true;
      store_pack<float, V>(&sm.pairs[m & 1].a[warp][lane * V], ca);
      store_pack<float, V>(&sm.pairs[m & 1].h[warp][lane * V], ch);
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.paired[m & 1]);
    }
    if (m > 0) {
      const unsigned o = m - 1;
      const Plan &opl = sm.plan[ostage];
      const int n = opl.rows - warp * R, d = opl.d0 + lane * V;
      const bool on = lane * V < opl.cols;
      if (!warp_wait(&sm.ready[o & 1], o >> 1 & 1u) || !warp_wait(&sm.entered[ostage], oparity)) return true;
      float a[kG], h[V], x[V], in[V];
      unpack(*reinterpret_cast<const Pack<float, V> *>(&sm.pairs[o & 1].h[warp][lane * V]), h);
      if (!(opl.cut >> warp & 1u)) {
        float pa[V];
        unpack(*reinterpret_cast<const Pack<float, V> *>(&sm.pairs[o & 1].a[warp][lane * V]), pa);
        unpack(*reinterpret_cast<const Pack<float, V> *>(&sm.edge[ostage].in[lane * V]), in);
        fma_v(h, pa, in, h);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.read[o & 1]);
      if (n > 0) {
        const WarpRows<TX, TA, V, kShared, false> rows(P, opl, sm.stage[ostage], warp, lane);
        const int64_t step = A.reverse ? -A.width : A.width;
        TX *out = static_cast<TX *>(A.out) + ((A.reverse ? opl.row0 - warp * R : opl.row0 + warp * R) * A.width + d);
        if (opl.plain) {
#pragma unroll
          for (int k = 0; k < R; ++k) {
            rows.get_a(k, A.gate_log, false, a);
            rows.get_x(k, x);
            fma_v(h, a, h, x);
            if (on) store_pack<TX, V>(out, h);
            out += step;
          }
        } else {
          const unsigned live = opl.live[warp], start = opl.start[warp], end = opl.end[warp];
#pragma unroll
          for (int k = 0; k < R; ++k) {
            if (live >> k & 1u) {
              rows.get_a(k, A.gate_log, false, a);
              rows.get_x(k, x);
              if (start >> k & 1u) {
                if (A.h0) {
                  float h0[V];
                  state_load<V>(A.h0, opl.seq[warp * R + k], A.width, d, on, h0);
                  fma_v(h, a, h0, x);
                } else {
#pragma unroll
                  for (int v = 0; v < V; ++v) h[v] = x[v];
                }
              } else {
                fma_v(h, a, h, x);
              }
              if (on) store_pack<TX, V>(out, h);
              if (end >> k & 1u) state_store<V>(A.state_out, opl.seq[warp * R + k], A.width, d, on, h);
            } else if (k < n && A.zero_rest && on) {
              const float z[V] = {};
              store_pack<TX, V>(out, z);
            }
            out += step;
          }
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // a was written where the next copy will write
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.empty[ostage]);
      if (++ostage == Shared::kStages) {
        ostage = 0;
        oparity ^= 1u;
      }
    }
    if (!valid) return false;
    if (++stage == Shared::kStages) {
      stage = 0;
      parity ^= 1u;
    }
  }
}

template <typename TX, typename TA, int V, bool kShared, bool kBackward>
__device__ __forceinline__ void init_barriers(StreamShared<TX, TA, V, kShared, kBackward> &sm) {
  if (threadIdx.x == 0) {
    for (unsigned s = 0; s < StreamShared<TX, TA, V, kShared, kBackward>::kStages; ++s) {
      mbar_init_count(&sm.full[s], 2);  // the expected bytes, and the plan
      mbar_init_count(&sm.empty[s], kWarps);
      mbar_init_count(&sm.entered[s], 4);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init_count(&sm.paired[s], kWarps);
      mbar_init_count(&sm.ready[s], 4);
      mbar_init_count(&sm.read[s], kWarps);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
}

template <typename TX, typename TA, int V, bool kShared>
__global__ void __launch_bounds__(kStreamThreads, 1) forward_stream_kernel(const __grid_constant__ Params P,
                                                                           const __grid_constant__ Maps maps) {
  using Shared = StreamShared<TX, TA, V, kShared, false>;
  extern __shared__ __align__(1024) unsigned char raw_smem[];
  auto &sm = *reinterpret_cast<Shared *>(raw_smem);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  init_barriers(sm);
  bool lost = false;
  if (warp < kWarps) lost = compute_forward<TX, TA, V, kShared>(P, sm, warp, lane);
  else if (warp < kWarps + 4) lost = publish_tiles<TX, TA, V, kShared>(P, sm, threadIdx.x - kThreads, lane);
  else if (warp < kWarps + 8) lost = finish_tiles<TX, TA, V, kShared, false>(P, sm, threadIdx.x - kThreads - 128, lane);
  else plan_tiles<TX, TA, V, kShared, false>(P, maps, sm, lane);
  if (lost && lane == 0 && P.A.status) atomicOr(reinterpret_cast<unsigned *>(P.A.status), GEARB_ST_SCAN_ABORTED);
}

// A matrix of [rows][width] for boxes of kTile rows and 32 * V channels.
template <typename T>
int make_map(CUtensorMap *map, const void *base, int64_t width, int64_t rows, int64_t row_stride, int box) {
  const CUtensorMapDataType type = sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16;
  return encode_map(map, type, const_cast<void *>(base), width, rows, row_stride * static_cast<int64_t>(sizeof(T)), box, kTile);
}

template <typename TX, typename TA, int V, bool kShared>
int launch_stream(Params &p, cudaStream_t stream) {
  const gearb_recurrence_args &a = p.A;
  p.blocks_per_gate = kShared ? (p.per + 32 * V - 1) / (32 * V) : 1;
  const int64_t ncol = kShared ? a.gates * p.blocks_per_gate : (a.width + 32 * V - 1) / (32 * V);
  // Items are counted in 32 bits, and every CTA takes two numbers beyond the last.
  GEARB_REQUIRE(p.tiles <= (int64_t(1) << 31) / ncol - 1, "recurrence: too many tiles for one launch");
  p.ncol = static_cast<int>(ncol);
  Maps maps;
  int rc = make_map<TX>(&maps.x, a.x, a.width, p.rows, a.x_row_stride, 32 * V);
  if (rc == GEARB_OK && !kShared) rc = make_map<TA>(&maps.gate, a.gate, a.width, p.rows, a.gate_row_stride, 32 * V);
  if (rc != GEARB_OK) return rc;
  constexpr int kSmem = sizeof(StreamShared<TX, TA, V, kShared, false>);
  static_assert(kSmem <= kSmemMost, "fits one SM");
  auto kernel = forward_stream_kernel<TX, TA, V, kShared>;
  GEARB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
  const int64_t most = sm_count(), items = p.tiles * ncol;
  kernel<<<static_cast<unsigned>(items < most ? items : most), kStreamThreads, kSmem, stream>>>(p, maps);
  GEARB_CUDA(cudaGetLastError());
  return GEARB_OK;
}

// TMA takes a matrix whose base and rows start on 16 bytes, and copies that start on 16 bytes.
inline bool matrix_ok(const void *p, int64_t sr, int size) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && sr > 0 && sr * size % 16 == 0 && sr * size < (int64_t(1) << 40);
}
template <typename TX, typename TA>
bool stream_fits(const Params &p, bool backward) {
  const gearb_recurrence_args &a = p.A;
  if (backward) return false;
  const bool shared = a.gates < a.width;
  if (!p.flat || p.V < 2 || p.rows >= (int64_t(1) << 31) || !matrix_ok(a.x, a.x_row_stride, sizeof(TX))) return false;
  if (shared) return p.per * sizeof(TX) % 16 == 0;
  return matrix_ok(a.gate, a.gate_row_stride, sizeof(TA));
}

template <typename TX, typename TA>
int launch_any(Params &p, bool backward, cudaStream_t stream) {
  if (!stream_fits<TX, TA>(p, backward)) return launch_wide_any<TX, TA>(p, backward, stream);
  const bool shared = p.A.gates < p.A.width;
  if (shared) return p.V == 4 ? launch_stream<TX, TA, 4, true>(p, stream) : launch_stream<TX, TA, 2, true>(p, stream);
  if constexpr (sizeof(TX) + sizeof(TA) <= 6)
    if (p.V == 4) return launch_stream<TX, TA, 4, false>(p, stream);
  return launch_stream<TX, TA, 2, false>(p, stream);
}

}  // namespace rec
}  // namespace gearb
