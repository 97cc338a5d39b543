// Host side of the recurrences: checks, sizes, choice of the kernel, and the entry points.
#include <cuda.h>

#include <atomic>

#include "recurrence_narrow.cuh"

namespace gearb {

using namespace rec;

namespace rec {

// cuTensorMapEncodeTiled, looked up in the driver once (the library links the runtime only).
int encode_map(CUtensorMap *map, CUtensorMapDataType type, void *base, int64_t width, int64_t rows, int64_t row_bytes, int box_w,
               int box_h) {
  using Encode = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                              const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static std::atomic<Encode> known{nullptr};
  Encode encode = known.load(std::memory_order_acquire);
  if (!encode) {
    void *fn = nullptr;
    cudaDriverEntryPointQueryResult found;
    GEARB_CUDA(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &found));
    if (found != cudaDriverEntryPointSuccess || !fn)
      return fail(GEARB_ERR_UNSUPPORTED, "the driver has no cuTensorMapEncodeTiled");
    encode = reinterpret_cast<Encode>(fn);
    known.store(encode, std::memory_order_release);
  }
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(width), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(row_bytes)};
  const cuuint32_t box[2] = {static_cast<cuuint32_t>(box_w), static_cast<cuuint32_t>(box_h)}, step[2] = {1, 1};
  const CUresult r = encode(map, type, 2, base, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(GEARB_ERR_CUDA, "cuTensorMapEncodeTiled failed with %d", static_cast<int>(r));
  return GEARB_OK;
}

}  // namespace rec

namespace {

std::atomic<int> g_wait_limit{-1};  // as gearb_recurrence_wait_limit has set it

// Joins the column blocks' sums of a gate whose channels span several of them, in order.  Rows of no
// sequence hold zeros when zero_rest is set; otherwise they are left as they are.
template <typename TA>
__global__ void __launch_bounds__(kThreads) gate_sum_kernel(const __grid_constant__ Params P) {
  const gearb_recurrence_args &A = P.A;
  const int64_t n = P.rows * A.gates;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < n;
       i += static_cast<int64_t>(gridDim.x) * kThreads) {
    if (A.offsets || A.lengths) {
      const int64_t row = i / A.gates;
      bool live;
      if (A.offsets) live = row >= __ldg(A.offsets) && row < __ldg(A.offsets + A.sequences);
      else live = row % A.time < __ldg(A.lengths + row / A.time);
      if (!live) {
        if (A.zero_rest) static_cast<TA *>(A.dgate)[i] = from_f<TA>(0.0f);
        continue;
      }
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

__device__ __forceinline__ void zero_span(char *p, int64_t n, int64_t me, int64_t threads) {
  int64_t head = (16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15;
  if (head > n) head = n;
  const int64_t vecs = (n - head) / 16, done = head + vecs * 16;
  if (me < head) p[me] = 0;
  if (me < n - done) p[done + me] = 0;
  for (int64_t i = me; i < vecs; i += threads) reinterpret_cast<uint4 *>(p + head)[i] = make_uint4(0, 0, 0, 0);
}

// One warp per tile: its rows among the sequences.  All warps: 0xff where tiles will publish, and zeros where packed
// sequences leave whole tiles.
__global__ void __launch_bounds__(kThreads) prepare_kernel(const __grid_constant__ Params P) {
  const gearb_recurrence_args &A = P.A;
  const int lane = threadIdx.x & 31;
  const int64_t threads = static_cast<int64_t>(gridDim.x) * kThreads, me = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  uint4 *fill = reinterpret_cast<uint4 *>(P.ticket);  // whole multiples of 256 bytes
  for (int64_t i = me; i < P.chain_bytes / 16; i += threads) fill[i] = make_uint4(kUnset, kUnset, kUnset, kUnset);
  const LiveTiles live_range = live_tiles(P);
  if (A.offsets && A.zero_rest) {
    const int64_t end = live_range.end * P.tile_rows, d0 = live_range.first * P.tile_rows, d1 = end < P.rows ? end : P.rows;
    auto zero = [&](void *base, int64_t row_bytes) {
      char *b = static_cast<char *>(base);
      zero_span(A.reverse ? b + (P.rows - d0) * row_bytes : b, d0 * row_bytes, me, threads);
      zero_span(A.reverse ? b : b + d1 * row_bytes, (P.rows - d1) * row_bytes, me, threads);
    };
    zero(P.backward ? A.dx : A.out, A.width * (A.x_dtype == GEARB_DT_F32 ? 4 : 2));
    if (P.backward && P.blocks_per_gate == 1) zero(A.dgate, A.gates * (A.gate_dtype == GEARB_DT_F32 ? 4 : 2));
  }
  // sequences without rows keep their state (backward: their gradient)
  float *to = P.backward ? A.dh0 : A.state_out;
  const float *old = P.backward ? A.dstate : A.h0;
  if (to && to != old && (A.offsets || A.lengths))
    for (int64_t s = me >> 5; s < A.sequences; s += threads >> 5) {
      const ScanOffsets so{A.offsets, P.rows, A.sequences, 0};
      if ((A.offsets ? so.at(s + 1) - so.at(s) : __ldg(A.lengths + s)) > 0) continue;
      for (int64_t d = lane; d < A.width; d += 32) to[s * A.width + d] = old ? old[s * A.width + d] : 0.0f;
    }
  for (int64_t tile = live_range.first + (me >> 5); tile < live_range.end; tile += threads >> 5) {
    Place at = {};
    at.tile = tile;
    at.i0 = tile * P.tile_rows;
    at.i1 = at.i0 + P.tile_rows < P.rows ? at.i0 + P.tile_rows : P.rows;
    const int n = static_cast<int>(at.i1 - at.i0);
    const TileRows tr = A.offsets ? tile_rows_packed(P, at, lane) : tile_rows_dense(P, at);
    TileRec &rec = P.recs[tile];
    int64_t first_start = tr.first_start, last_end = tr.last_end;
    bool first_open = true, last_open = true;  // the first (last) row's sequence began (goes on) elsewhere
    uint64_t live = ~uint64_t(0), start = 0, end = 0;
    if (!tr.interior) {
      live = 0;
#pragma unroll
      for (int half = 0; half < kTile / 32; ++half) {
        const int n0 = n - half * 32, nn = n0 < 0 ? 0 : (n0 > 32 ? 32 : n0);
        const RowMap rm = map_rows(A, P.rows, at.i0 + half * 32, nn, lane);
        rec.seq[half * 32 + lane] = rm.seq;
        live |= static_cast<uint64_t>(rm.live) << (half * 32);
        start |= static_cast<uint64_t>(rm.start) << (half * 32);
        end |= static_cast<uint64_t>(rm.end) << (half * 32);
        if (half == 0) {
          first_start = rm.first_start;
          first_open = rm.live & ~rm.start & 1u;
        }
        if (nn > 0) {
          last_end = rm.last_end;
          last_open = (rm.live & ~rm.end) >> (nn - 1) & 1u;
        }
      }
    }
    const bool s = lane < kWarps && (start >> (kRows * (lane & (kWarps - 1))) & kAllRows) != 0;
    const bool e = lane < kWarps && (end >> (kRows * (lane & (kWarps - 1))) & kAllRows) != 0;
    const unsigned starts = __ballot_sync(kAll, s), ends = __ballot_sync(kAll, e);
    if (lane < kWarps) {
      rec.live[lane] = static_cast<unsigned char>(live >> (kRows * lane) & kAllRows);
      rec.start[lane] = static_cast<unsigned char>(start >> (kRows * lane) & kAllRows);
      rec.end[lane] = static_cast<unsigned char>(end >> (kRows * lane) & kAllRows);
    }
    if (lane == 0) {
      rec.starts = starts;
      rec.ends = ends;
      // all bits above the lowest start; all below the highest end, and bit kWarps
      rec.cut = starts ? ~0u << __ffs(starts) : 0u;
      rec.bcut = ends ? ((1u << (31 - __clz(ends))) - 1u) | 1u << kWarps : 0u;
      rec.plain = tr.interior;
      rec.dead = live == 0;
      const int64_t from = quotient(first_start, P.tile_rows), back = P.tiles - 1 - tile;
      rec.open = P.chain && first_open && from < tile;
      rec.lo = rec.open ? static_cast<int>(from) : -1;
      const int64_t lo = P.tiles - 1 - quotient(last_end, P.tile_rows);
      rec.lo_back = P.chain && last_open && lo < back ? static_cast<int>(lo) : -1;
    }
  }
}

// One row a sequence, as in decoding: nothing to hand on, so every thread takes V channels of one row.  Bound by the
// launch for the usual sizes, by memory for large ones.
template <typename TX, typename TA, int V>
__global__ void __launch_bounds__(kThreads) step_kernel(const __grid_constant__ Params P) {
  const gearb_recurrence_args &A = P.A;
  const int64_t per_row = (A.width + V - 1) / V, n = A.batch * per_row;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < n;
       i += static_cast<int64_t>(gridDim.x) * kThreads) {
    const int64_t b = quotient(i, per_row), d = (i - b * per_row) * V;
    const TA *gate = static_cast<const TA *>(A.gate) + b * A.gate_batch_stride;
    float x[V], a[V], h[V];
    const Pack<TX, V> px = load_pack<TX, V>(static_cast<const TX *>(A.x) + b * A.x_batch_stride + d);
#pragma unroll
    for (int v = 0; v < V; ++v) x[v] = to_f(px.v[v]);
    if (P.per == 1) {
      const Pack<TA, V> pg = load_pack<TA, V>(gate + d);
#pragma unroll
      for (int v = 0; v < V; ++v) a[v] = to_f(pg.v[v]);
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) a[v] = to_f(gate[(d + v) / P.per]);
    }
    if (A.h0) {
      const Pack<float, V> p0 = load_pack<float, V>(A.h0 + b * A.width + d);
#pragma unroll
      for (int v = 0; v < V; ++v) h[v] = fmaf(A.gate_log ? exp_of(a[v]) : a[v], p0.v[v], x[v]);
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) h[v] = x[v];
    }
    store_pack<TX, V>(static_cast<TX *>(A.out) + b * A.width + d, h);
    if (A.state_out) store_pack<float, V>(A.state_out + b * A.width + d, h);
  }
}
template <typename TX, typename TA>
int launch_step(const Params &p, cudaStream_t stream) {
  const gearb_recurrence_args &a = p.A;
  const bool four = a.width % 4 == 0 && vector_ok(a.x, a.x_batch_stride, 0, sizeof(TX), 4) &&
                    vector_ok(a.out, 0, 0, sizeof(TX), 4) && vector_ok(a.h0, 0, 0, 4, 4) && vector_ok(a.state_out, 0, 0, 4, 4) &&
                    (p.per > 1 || vector_ok(a.gate, a.gate_batch_stride, 0, sizeof(TA), 4));
  const int64_t n = a.batch * (four ? a.width / 4 : a.width), blocks = (n + kThreads - 1) / kThreads;
  const int64_t most = static_cast<int64_t>(sm_count()) * 64;
  const unsigned grid = static_cast<unsigned>(blocks < most ? blocks : most);
  if (four) step_kernel<TX, TA, 4><<<grid, kThreads, 0, stream>>>(p);
  else step_kernel<TX, TA, 1><<<grid, kThreads, 0, stream>>>(p);
  GEARB_CUDA(cudaGetLastError());
  return GEARB_OK;
}

// ---- host -------------------------------------------------------------------
int64_t up256(int64_t v) { return (v + 255) / 256 * 256; }

// Tiling of a call, the same for its forward and backward pass: which kind of kernel, rows per tile, and whether tiles
// need anything from each other.
struct Tiling {
  int64_t rows, tiles;
  int tile_rows, chain, narrow_rows;
};
// SMs of a full B200.  A constant in place of sm_count(): tiles decide how states are rounded and how long the carry is, and
// these go by the sizes of a call alone, whatever part of a GPU it runs on.
constexpr int kFullSms = 148;
Tiling tiling_of(const gearb_recurrence_args &a) {
  Tiling t = {};
  t.rows = a.batch * a.time;
  int most = kTile;
  if (a.width <= kNarrowWidth) {
    // 16 rows a thread keep the memory busy; with 4 a small call is spread over four times as many SMs
    const int groups = kWarps * narrow_groups(static_cast<int>(a.width));
    t.narrow_rows = t.rows > int64_t(16) * groups * kFullSms ? 16 : 4;
    most = t.narrow_rows * groups;
  }
  t.tile_rows = most;
  t.chain = t.rows > most;
  if (!a.offsets && a.time > 0 && a.time <= most) {  // whole sequences per tile
    t.tile_rows = static_cast<int>(most / a.time * a.time);
    t.chain = 0;
  }
  t.tiles = (t.rows + t.tile_rows - 1) / t.tile_rows;
  return t;
}

struct Scratch {
  int64_t agg, super, section, recs, part, chain_bytes, total;
};
Scratch scratch_of(const gearb_recurrence_args &a, bool backward) {
  const Tiling t = tiling_of(a);
  const int64_t rows = t.rows, tiles = t.tiles;
  Scratch s = {};
  if (t.chain) {
    s.agg = 256;
    s.super = s.agg + up256(tiles * a.width * 8);
    s.section = s.super + up256((tiles / kSuper + 1) * a.width * 8);
    s.chain_bytes = s.section + up256((tiles / kSuper + 1) * a.width * 4);
  }
  s.recs = s.chain_bytes;
  s.part = s.recs + up256(tiles * static_cast<int64_t>(sizeof(TileRec)));
  s.total = s.part;
  const int64_t per = a.width / a.gates;
  if (backward && a.gates < a.width && per > 32) s.total += up256((per + 31) / 32 * rows * a.gates * 4);
  return s;
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

int launch(const gearb_recurrence_args &a, bool backward, cudaStream_t stream) {
  Params p = {};
  p.A = a;
  p.backward = backward;
  const Tiling t = tiling_of(a);
  p.rows = t.rows;
  p.tiles = t.tiles;
  p.tile_rows = t.tile_rows;
  p.chain = t.chain;
  p.narrow_rows = t.narrow_rows;
  const int limit = g_wait_limit.load(std::memory_order_relaxed);
  p.poll_limit = limit < 0 ? kPollLimit : limit;
  p.no_waits = limit == 0;
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
  if (!backward && a.time == 1 && !a.offsets && !a.lengths) {
    const bool own = a.gate_dtype == a.x_dtype;
    if (a.x_dtype == GEARB_DT_F32) return launch_step<float, float>(p, stream);
    if (a.x_dtype == GEARB_DT_F16) return own ? launch_step<__half, __half>(p, stream) : launch_step<__half, float>(p, stream);
    return own ? launch_step<__nv_bfloat16, __nv_bfloat16>(p, stream) : launch_step<__nv_bfloat16, float>(p, stream);
  }
  const Scratch s = scratch_of(a, backward);
  if (p.chain) {
    char *base = static_cast<char *>(a.scratch);
    p.ticket = reinterpret_cast<unsigned *>(base);
    p.agg = reinterpret_cast<float2 *>(base + s.agg);
    p.super = reinterpret_cast<float2 *>(base + s.super);
    p.section = reinterpret_cast<float *>(base + s.section);
    p.chain_bytes = s.chain_bytes;
  }
  p.recs = reinterpret_cast<TileRec *>(static_cast<char *>(a.scratch) + s.recs);
  p.gate_part = reinterpret_cast<float *>(static_cast<char *>(a.scratch) + s.part);
  auto period = [&](int64_t sb, int64_t sr) { return sb == a.time * sr || a.batch == 1 ? p.rows : a.time; };
  p.x_period = period(a.x_batch_stride, a.x_row_stride);
  p.gate_period = period(a.gate_batch_stride, a.gate_row_stride);
  p.dout_period = period(a.dout_batch_stride, a.dout_row_stride);
  p.flat = p.x_period == p.rows && p.gate_period == p.rows && (!backward || p.dout_period == p.rows);
  // Channels a lane: as many as alignment allows and the width (of a gate's channels) fills.
  const bool shared = a.gates < a.width;
  // A gate's gradient is summed over the warp where a block lies inside one gate; gates of up to 16 channels would leave
  // half of its lanes idle.
  p.by_gate = shared && backward && p.per > 16;
  const int64_t unit = p.by_gate ? p.per : a.width;
  const int xs = a.x_dtype == GEARB_DT_F32 ? 4 : 2, gs = a.gate_dtype == GEARB_DT_F32 ? 4 : 2;
  for (p.V = 4; p.V > 1; p.V /= 2) {
    const int v = p.V;
    if (unit % v != 0 || unit <= 32 * (v / 2)) continue;
    if (!vector_ok(a.x, a.x_batch_stride, a.x_row_stride, xs, v)) continue;
    if (!shared && !vector_ok(a.gate, a.gate_batch_stride, a.gate_row_stride, gs, v)) continue;
    if (!vector_ok(backward ? a.dx : a.out, 0, 0, xs, v)) continue;
    if (!backward) break;
    if (!vector_ok(a.dout, a.dout_batch_stride, a.dout_row_stride, xs, v)) continue;
    if (shared || vector_ok(a.dgate, 0, 0, gs, v)) break;
  }
  if (p.V == 1 && unit > 32) {
    p.V = 2;
    p.apart = 1;
  }
  const int rc = a.x_dtype == GEARB_DT_F32 ? launch_f32(p, backward, stream)
                 : a.x_dtype == GEARB_DT_F16 ? launch_f16(p, backward, stream) : launch_bf16(p, backward, stream);
  if (rc != GEARB_OK || !backward || p.blocks_per_gate <= 1) return rc;
  const int64_t blocks = (p.rows * a.gates + kThreads - 1) / kThreads, most = static_cast<int64_t>(sm_count()) * 8;
  const unsigned grid = static_cast<unsigned>(blocks < most ? blocks : most);
  if (a.gate_dtype == GEARB_DT_F32) gate_sum_kernel<float><<<grid, kThreads, 0, stream>>>(p);
  else if (a.gate_dtype == GEARB_DT_F16) gate_sum_kernel<__half><<<grid, kThreads, 0, stream>>>(p);
  else gate_sum_kernel<__nv_bfloat16><<<grid, kThreads, 0, stream>>>(p);
  GEARB_CUDA(cudaGetLastError());
  return GEARB_OK;
}

int run(const gearb_recurrence_args *args, bool backward, void *stream) {
  int64_t scratch = 0, carry = 0;
  int rc = gearb_recurrence_bytes(args, backward, &scratch, &carry);
  if (rc == GEARB_OK) rc = check_pointers(args, backward);
  if (rc != GEARB_OK) return rc;
  GEARB_REQUIRE(args->scratch_bytes >= scratch && (scratch == 0 || args->scratch),
                "recurrence: scratch of %lld bytes needed", (long long)scratch);
  GEARB_REQUIRE(reinterpret_cast<uintptr_t>(args->scratch) % 16 == 0, "recurrence: scratch must start on 16 bytes");
  GEARB_REQUIRE(!backward || carry == 0 || args->carry, "recurrence: the backward pass needs the forward pass's carry");
  return launch(*args, backward, as_stream(stream));
}

}  // namespace

int rec::launch_prepare(const Params &p, cudaStream_t stream) {
  int64_t warps = p.tiles > p.chain_bytes / 2048 ? p.tiles : p.chain_bytes / 2048;  // up to 64 bytes a thread
  if ((p.A.offsets || p.A.lengths) && warps < p.A.sequences) warps = p.A.sequences;
  if (p.A.offsets && p.A.zero_rest) {  // up to 256 bytes a thread, were there no sequences at all
    const int64_t bytes = p.rows * p.A.width * (p.A.x_dtype == GEARB_DT_F32 ? 4 : 2);
    if (warps < bytes / 8192) warps = bytes / 8192;
  }
  const int64_t blocks = (warps + kWarps - 1) / kWarps, most = static_cast<int64_t>(sm_count()) * 8;
  prepare_kernel<<<static_cast<unsigned>(blocks < most ? (blocks > 0 ? blocks : 1) : most), kThreads, 0, stream>>>(p);
  GEARB_CUDA(cudaGetLastError());
  return GEARB_OK;
}
}  // namespace gearb

using namespace gearb;

extern "C" {

int gearb_recurrence_bytes(const gearb_recurrence_args *args, int backward, int64_t *scratch_bytes,
                           int64_t *carry_bytes) {
  GEARB_REQUIRE(scratch_bytes && carry_bytes, "recurrence_bytes: null argument");
  const int rc = check_sizes(args);
  if (rc != GEARB_OK) return rc;
  const Tiling t = tiling_of(*args);
  *scratch_bytes = scratch_of(*args, backward != 0).total;
  *carry_bytes = t.chain ? t.tiles * args->width * 4 : 0;
  return GEARB_OK;
}

int gearb_recurrence_wait_limit(int polls) { return g_wait_limit.exchange(polls < 0 ? -1 : polls); }

int gearb_recurrence_forward(const gearb_recurrence_args *args, void *stream) {
  TraceRange trace("gearb:recurrence");
  return run(args, false, stream);
}

int gearb_recurrence_backward(const gearb_recurrence_args *args, void *stream) {
  TraceRange trace("gearb:recurrence_backward");
  return run(args, true, stream);
}

}  // extern "C"
