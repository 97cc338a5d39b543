// Trajectory-segment gather.
//
// gather_kernel is the fused multi-column form of the reference's
// fused_subcopy_collect (src/cuda/copy.cu:91-134): per request g and subscribed
// column it clips [ts+offset, ts+offset+length) to [0, len), and moves the
// clipped rows from  table + idx*trajectory_stride + column_offset + start*row
// to  dst + g*slot (+ slot - bytes when padding at the head), the addressing of
// CpuTrajectoryStorageHandler::sub (src/storage/handler.cc:78-131).
// vcopy_kernel is the generic offset-list form (vary_/fix_stride_copy_collect,
// src/cuda/copy.cu:12-89).
//
// Differences in HOW, not in WHAT:
//  * all subscribed columns of a batch go in one launch;
//  * one warp moves one 2 KiB piece of a slot with 16-byte accesses that are
//    consecutive across the lanes (the reference gives each thread its own 64
//    bytes, so a warp's 16-byte loads sit 64 bytes apart);
//  * source and destination may have any byte alignment: stores are aligned to
//    the destination, and a misaligned source is read as two aligned 16-byte
//    blocks that are funnel-shifted together (the reference casts both sides to
//    float4 and is only defined for 16-byte aligned addresses);
//  * all offsets are 64-bit (the reference's kernel parameters are int);
//  * a trajectory index outside the table is skipped and reported through the
//    status word instead of being dereferenced.
// The source pointer may be HBM or pinned mapped host memory; the code is the same.
#include "common.h"
#include "device_copy.cuh"

namespace gearb {
namespace {

constexpr int kThreads = 256;
constexpr int kWarpsPerBlock = kThreads / 32;
using dev::warp_copy;

__global__ void __launch_bounds__(kThreads) gather_kernel(const __grid_constant__ GatherParams P) {
  const int lane = threadIdx.x & 31;
  const int64_t warps_total = static_cast<int64_t>(gridDim.x) * kWarpsPerBlock;
  const int64_t items = P.n * P.chunks_per_request;
  unsigned flags = 0;
  for (int64_t item = static_cast<int64_t>(blockIdx.x) * kWarpsPerBlock + (threadIdx.x >> 5);
       item < items; item += warps_total) {
    const int64_t g = item / P.chunks_per_request;
    const int q = static_cast<int>(item - g * P.chunks_per_request);
    const int c = dev::column_of_piece(P, q);
    dev::gather_piece(P, P.cols[c], q - P.cols[c].chunk_first, g, __ldg(P.idx + g), __ldg(P.ts + g),
                      __ldg(P.len + g), lane, flags, P.table);
  }
  if (flags && P.status && lane == 0) atomicOr(reinterpret_cast<unsigned *>(P.status), flags);
}

struct VcopyArgs {
  const uint8_t *src;
  uint8_t *dst;
  const int64_t *src_off, *dst_off, *lengths;
  int64_t fixed_length;  // used when lengths == nullptr
  int64_t n;
  int32_t chunks_per_slice;
  int32_t chunk_bytes;
};

__global__ void __launch_bounds__(kThreads) vcopy_kernel(const VcopyArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t warps_total = static_cast<int64_t>(gridDim.x) * kWarpsPerBlock;
  const int64_t items = a.n * a.chunks_per_slice;
  for (int64_t item = static_cast<int64_t>(blockIdx.x) * kWarpsPerBlock + (threadIdx.x >> 5);
       item < items; item += warps_total) {
    const int64_t g = item / a.chunks_per_slice;
    const int64_t c0 = (item - g * a.chunks_per_slice) * a.chunk_bytes;
    const int64_t length = a.lengths ? __ldg(a.lengths + g) : a.fixed_length;
    int64_t c1 = c0 + a.chunk_bytes;
    if (c1 > length) c1 = length;
    if (c1 > c0)
      warp_copy(a.dst + __ldg(a.dst_off + g) + c0, a.src + __ldg(a.src_off + g) + c0,
                static_cast<int>(c1 - c0), lane);
  }
}

__global__ void segment_lengths_kernel(const __grid_constant__ GatherParams P, int64_t *out) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i >= P.n) return;
  int64_t start, rows;
  unsigned flags = 0;
  dev::clip_segment(P, P.cols[0], P.idx[i], P.ts[i], P.len[i], start, rows, flags);
  out[i] = rows;
}

// Packed / paged gather.
//
// A CTA takes a request (or a slice of one, where the requests are few): its indexes are looked up once, and its warps
// share its rows out.  Packed rows of a column are one run of bytes; so are the rows of a page.  Columns that are
// packed, or have 64 bytes a row or 512 a page, go in pieces of at most 4 KiB of a run.  The smaller columns of a paged
// request go together, 64 rows a warp, a row a lane, each row's slot looked up once for all of them: a page's run of
// them would occupy a few lanes only.  Bound by memory: 2 x bytes; what it takes is many warps with few registers.
// Measured on 8192 requests of config 3's rows in pages of 16 (118 us at the copy rate): a warp per 2 KiB of any
// column, a page's run at a time, 2180 us; a warp per piece of some request, with four 16-byte blocks a lane in
// flight, 340 to 750 us, faster with fewer registers than with fewer spills; as it is 200 us, 60 % of the warps resident,
// 16.6 of 23 stall cycles an issue on loads.
constexpr int kPackedPiece = 4096;

__device__ __forceinline__ void copy_run(uint8_t *d, const uint8_t *s, int nbytes, int lane) {
  int head = static_cast<int>((16u - (reinterpret_cast<uintptr_t>(d) & 15u)) & 15u);
  if (head > nbytes) head = nbytes;
  if (lane < head) d[lane] = s[lane];
  d += head;
  s += head;
  nbytes -= head;
  const int nvec = nbytes >> 4;
  const unsigned sh = static_cast<unsigned>(reinterpret_cast<uintptr_t>(s) & 15u);
  uint4 *dv = reinterpret_cast<uint4 *>(d);
  // two aligned blocks hold a block of the destination, where the source is not aligned like it
  const uint4 *sv = reinterpret_cast<const uint4 *>(s - sh);
  const unsigned ws = sh >> 2, bs = (sh & 3u) * 8u;
#pragma unroll 2
  for (int v = lane; v < nvec; v += 32) {
    const uint4 a = __ldg(sv + v);
    if (sh == 0) {
      dv[v] = a;
    } else {
      const uint4 b = __ldg(sv + v + 1);
      dv[v] = dev::shift_pair(a, b, ws, bs);
    }
  }
  const int done = nvec << 4;
  if (lane < nbytes - done) d[done + lane] = s[done + lane];
}

template <typename U>
__device__ __forceinline__ void copy_rows(uint8_t *dst, const uint8_t *src, int row, int64_t s0, int64_t s1, int lane) {
  src += lane * row;
  for (int c = 0; c < row; c += static_cast<int>(sizeof(U))) {
    U a, b;
    if (s0 >= 0) a = __ldg(reinterpret_cast<const U *>(src + c));
    if (s1 >= 0) b = __ldg(reinterpret_cast<const U *>(src + 32 * row + c));
    if (s0 >= 0) *reinterpret_cast<U *>(dst + s0 * row + c) = a;
    if (s1 >= 0) *reinterpret_cast<U *>(dst + s1 * row + c) = b;
  }
}

__global__ void __launch_bounds__(kThreads, 6) gather_packed_kernel(const __grid_constant__ GatherParams P,
                                                                    const __grid_constant__ PackedDst D) {
  const int lane = threadIdx.x & 31;
  const int64_t g = blockIdx.x;
  unsigned flags = 0;
  const int64_t idx = __ldg(P.idx + g), o0 = __ldg(D.offsets + g), o1 = __ldg(D.offsets + g + 1);
  const int64_t past = D.past ? __ldg(D.past + g) : 0;
  int64_t start, count64;
  {
    GatherColumn rows_of = {};  // the columns share one pattern: the clipped segment in rows
    rows_of.row = 1;
    rows_of.pat_offset = P.cols[0].pat_offset;
    rows_of.pat_length = P.cols[0].pat_length;
    dev::clip_segment(P, rows_of, idx, __ldg(P.ts + g), __ldg(P.len + g), start, count64, flags);
  }
  if (o0 < 0 || past < 0 || past > D.room) {
    flags |= GEARB_ST_BAD_REQUEST;
    count64 = 0;
  } else if (o1 <= o0) {  // before the difference, which may pass 64 bits
    count64 = 0;
  } else if (count64 > o1 - o0) {
    count64 = o1 - o0;
  }
  const int count = static_cast<int>(count64);  // at most the pattern's length
  const uint8_t *base = P.table + idx * P.traj_stride;
  // positions are at most 2^31 + the pattern's length
  auto block_of = [&](uint64_t pos) -> uint64_t {
    if (D.page_shift >= 0) return pos >> D.page_shift;
    if ((pos >> 32) == 0) return static_cast<unsigned>(pos) / static_cast<unsigned>(D.page);
    return pos / static_cast<uint64_t>(D.page);
  };
  auto page_at = [&](uint64_t blk) -> int64_t {
    return blk < static_cast<uint64_t>(D.max_blocks) ? __ldg(D.block_table + g * D.max_blocks + static_cast<int64_t>(blk)) : -1;
  };
  const uint64_t blk0 = D.block_table ? block_of(static_cast<uint64_t>(past)) : 0;
  const int in0 = D.block_table ? static_cast<int>(past - static_cast<int64_t>(blk0) * D.page) : 0;
  // runs a column's rows make, and 64-row groups of the small columns
  const int runs = count == 0 ? 0 : !D.block_table ? 1 : static_cast<int>(block_of(static_cast<uint64_t>(in0) + count - 1)) + 1;
  const int first = static_cast<int>(blockIdx.y) * kWarpsPerBlock + (threadIdx.x >> 5);
  const int step = static_cast<int>(gridDim.y) * kWarpsPerBlock;
  int at = first;  // this warp's next piece, counted from the current column's first
  for (int ci = 0; ci < D.big; ++ci) {
    const GatherColumn &col = P.cols[ci];
    const int row = col.row;
    const int64_t limit = D.dst_rows[ci];
    const uint8_t *src = base + col.col_offset + start * row;
    const int pieces = col.reserved ? col.reserved : static_cast<int>((static_cast<int64_t>(count) * row + kPackedPiece - 1) / kPackedPiece);
    const int64_t total = static_cast<int64_t>(runs) * pieces;
    int64_t k = at;
    for (; k < total; k += step) {
      const int run = static_cast<int>(k / pieces), piece = static_cast<int>(k - static_cast<int64_t>(run) * pieces);
      int64_t t = 0, rows = count, slot = o0;
      if (D.block_table) {
        const int64_t page = page_at(blk0 + run), in = run == 0 ? in0 : 0;
        t = run == 0 ? 0 : static_cast<int64_t>(run) * D.page - in0;
        rows = D.page - in < count - t ? D.page - in : count - t;
        slot = page < 0 ? limit : page * D.page + in;
      }
      int64_t n = slot < limit ? limit - slot : 0;  // rows inside the destination
      if (n < rows) flags |= GEARB_ST_BAD_REQUEST;
      else n = rows;
      const int64_t b0 = static_cast<int64_t>(piece) * kPackedPiece, b1 = n * row < b0 + kPackedPiece ? n * row : b0 + kPackedPiece;
      if (b1 > b0) copy_run(col.dst + slot * row + b0, src + t * row + b0, static_cast<int>(b1 - b0), lane);
    }
    at = static_cast<int>(k - total);
  }
  if (D.big == P.ncols) {
    if (flags && P.status) atomicOr(reinterpret_cast<unsigned *>(P.status), flags);
    return;
  }
  for (int64_t t = static_cast<int64_t>(at) * 64; t < count; t += static_cast<int64_t>(step) * 64) {
    int64_t slot[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int64_t r = t + 32 * k + lane;
      slot[k] = -1;
      if (r >= count) continue;
      const uint64_t pos = static_cast<uint64_t>(past + r), blk = block_of(pos);
      const int64_t page = page_at(blk);
      if (page >= 0) slot[k] = page * D.page + static_cast<int64_t>(pos - blk * D.page);
      else flags |= GEARB_ST_BAD_REQUEST;
    }
    for (int c = D.big; c < P.ncols; ++c) {
      const GatherColumn &col = P.cols[c];
      const int64_t limit = D.dst_rows[c];
      int64_t s0 = slot[0], s1 = slot[1];
      if (s0 >= limit || s1 >= limit) flags |= GEARB_ST_BAD_REQUEST;
      if (s0 >= limit) s0 = -1;
      if (s1 >= limit) s1 = -1;
      const uint8_t *from = base + col.col_offset + (start + t) * col.row;
      const uintptr_t bits = reinterpret_cast<uintptr_t>(from) | reinterpret_cast<uintptr_t>(col.dst) |
                             static_cast<uintptr_t>(col.row);
      if ((bits & 7) == 0) copy_rows<uint2>(col.dst, from, col.row, s0, s1, lane);
      else if ((bits & 3) == 0) copy_rows<unsigned>(col.dst, from, col.row, s0, s1, lane);
      else if ((bits & 1) == 0) copy_rows<unsigned short>(col.dst, from, col.row, s0, s1, lane);
      else copy_rows<unsigned char>(col.dst, from, col.row, s0, s1, lane);
    }
  }
  if (flags && P.status) atomicOr(reinterpret_cast<unsigned *>(P.status), flags);
}

int grid_for(int64_t items) {
  int64_t blocks = (items + kWarpsPerBlock - 1) / kWarpsPerBlock;
  const int64_t cap = static_cast<int64_t>(sm_count()) * 64;
  if (blocks > cap) blocks = cap;
  if (blocks < 1) blocks = 1;
  return static_cast<int>(blocks);
}

}  // namespace

int launch_gather(const GatherParams &p, cudaStream_t stream) {
  if (p.n == 0 || p.ncols == 0) return GEARB_OK;
  const int64_t items = p.n * p.chunks_per_request;
  gather_kernel<<<grid_for(items), kThreads, 0, stream>>>(p);
  GEARB_CUDA(cudaGetLastError());
  return GEARB_OK;
}

int launch_segment_lengths(const GatherParams &p, int64_t *out, cudaStream_t stream) {
  const int64_t blocks = (p.n + kThreads - 1) / kThreads;
  GEARB_REQUIRE(blocks < (int64_t(1) << 31), "segment_lengths: too many requests");
  segment_lengths_kernel<<<static_cast<unsigned>(blocks), kThreads, 0, stream>>>(p, out);
  GEARB_CUDA(cudaGetLastError());
  return GEARB_OK;
}

int launch_gather_packed(const GatherParams &params, const PackedDst &dst, cudaStream_t stream) {
  GatherParams p = params;
  PackedDst d = dst;
  d.page_shift = -1;
  for (int s = 0; s < 32; ++s)
    if (d.page == int64_t(1) << s) d.page_shift = s;
  d.room = d.block_table ? d.max_blocks * d.page : 0;
  auto small = [&](const GatherColumn &c) { return d.block_table && c.row < 64 && c.row * d.page < 512; };
  // the columns that are copied in runs first
  d.big = 0;
  int at = 0;
  for (int pass = 0; pass < 2; ++pass)
    for (int c = 0; c < params.ncols; ++c)
      if (small(params.cols[c]) == (pass == 1)) {
        p.cols[at] = params.cols[c];
        d.dst_rows[at++] = dst.dst_rows[c];
        if (pass == 0) ++d.big;
      }
  int64_t pieces = 1;  // of a request of the pattern's length
  for (int c = 0; c < p.ncols; ++c) {
    GatherColumn &col = p.cols[c];
    const int64_t of_run = (d.page * col.row + kPackedPiece - 1) / kPackedPiece;
    GEARB_REQUIRE(static_cast<int64_t>(col.pat_length) * col.row < (int64_t(1) << 40) && of_run < (int64_t(1) << 31),
                  "gather_packed: request too large");
    col.reserved = d.block_table ? static_cast<int32_t>(of_run) : 0;  // pieces of a page's run; packed: by the request's rows
    if (c >= d.big) pieces += (col.pat_length + 63) / 64 / (p.ncols - d.big);
    else if (d.block_table) pieces += ((col.pat_length - 1) / d.page + 2) * of_run;
    else pieces += (static_cast<int64_t>(col.pat_length) * col.row + kPackedPiece - 1) / kPackedPiece;
  }
  GEARB_REQUIRE(p.n < (int64_t(1) << 31) && pieces < (int64_t(1) << 31), "gather_packed: request too large");
  // Slices: enough CTAs for the GPU where the requests alone are too few, but no CTA without a piece for its warps.
  const int64_t want = (static_cast<int64_t>(sm_count()) * 12 + p.n - 1) / p.n;
  int64_t slices = (pieces + kWarpsPerBlock - 1) / kWarpsPerBlock;
  if (slices > want) slices = want;
  if (slices > 65535) slices = 65535;
  gather_packed_kernel<<<dim3(static_cast<unsigned>(p.n), static_cast<unsigned>(slices < 1 ? 1 : slices)), kThreads, 0, stream>>>(p, d);
  GEARB_CUDA(cudaGetLastError());
  return GEARB_OK;
}

int launch_vcopy(const uint8_t *src, uint8_t *dst, const int64_t *src_off,
                 const int64_t *dst_off, const int64_t *lengths, int64_t fixed_length, int64_t n,
                 int64_t max_length, cudaStream_t stream) {
  GEARB_REQUIRE(n >= 0 && max_length >= 0, "vcopy: negative count or length");
  if (n == 0 || max_length == 0) return GEARB_OK;
  GEARB_REQUIRE(src && dst && src_off && dst_off, "vcopy: null pointer argument");
  VcopyArgs a;
  a.src = src; a.dst = dst; a.src_off = src_off; a.dst_off = dst_off; a.lengths = lengths;
  a.fixed_length = fixed_length; a.n = n;
  a.chunk_bytes = 2048;
  const int64_t cps = (max_length + a.chunk_bytes - 1) / a.chunk_bytes;
  GEARB_REQUIRE(cps < (int64_t(1) << 31), "vcopy: max_length too large");
  a.chunks_per_slice = static_cast<int32_t>(cps);
  vcopy_kernel<<<grid_for(n * cps), kThreads, 0, stream>>>(a);
  GEARB_CUDA(cudaGetLastError());
  return GEARB_OK;
}

}  // namespace gearb
