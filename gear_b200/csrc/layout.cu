// Offsets, block table and slot map of a batch of requests, from their lengths.
//
// n_r tokens are added to request r behind the past_r it has.  Two prefix sums over the requests
// (tokens, new pages) place every request; then every token's slot and every new page's table
// entry follow from its request alone.  All of it is integer arithmetic in 64 bits.
#include "common.h"

namespace gearb {
namespace {

constexpr int kThreads = 1024;

struct LayoutParams {
  gearb_layout_args a;
  int64_t *first_page;  // [requests]: place of the request's first new page in the free list
};

// Tokens the request adds and pages it needs for them.
__device__ __forceinline__ void request_need(const gearb_layout_args &a, int64_t r, int64_t &past, int64_t &n,
                                             int64_t &have, int64_t &need, unsigned &flags) {
  const int64_t room = a.max_blocks * a.page;
  past = a.past ? __ldg(a.past + r) : 0;
  if (past < 0 || past > room) {
    past = past < 0 ? 0 : room;
    flags |= GEARB_ST_LEN_CLAMPED;
  }
  n = __ldg(a.lengths + r);
  if (n < 0 || n > room - past) {
    n = n < 0 ? 0 : room - past;
    flags |= GEARB_ST_LEN_CLAMPED;
  }
  have = (past + a.page - 1) / a.page;
  need = (past + n + a.page - 1) / a.page - have;
}

__device__ __forceinline__ int64_t warp_inclusive(int64_t v, int lane) {
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t u = __shfl_up_sync(0xffffffffu, v, d);
    if (lane >= d) v += u;
  }
  return v;
}

__global__ void __launch_bounds__(kThreads) layout_scan_kernel(const __grid_constant__ LayoutParams P) {
  __shared__ int64_t wt[kThreads / 32], wp[kThreads / 32];
  const gearb_layout_args &a = P.a;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t tokens = 0, used = *a.used_in;
  if (used < 0) used = 0;
  unsigned flags = 0;
  for (int64_t r0 = 0; r0 < a.requests; r0 += kThreads) {
    const int64_t r = r0 + threadIdx.x;
    int64_t past, n = 0, have, need = 0;
    if (r < a.requests) request_need(a, r, past, n, have, need, flags);
    const int64_t it = warp_inclusive(n, lane), ip = warp_inclusive(need, lane);
    if (lane == 31) { wt[warp] = it; wp[warp] = ip; }
    __syncthreads();
    int64_t bt = tokens, bp = used;
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) { bt += wt[w]; bp += wp[w]; }
      tokens += wt[w];
      used += wp[w];
    }
    if (r < a.requests) {
      a.offsets[r] = bt + it - n;
      P.first_page[r] = bp + ip - need;
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    a.offsets[a.requests] = tokens;
    if (used > a.num_pages) {
      used = a.num_pages;
      flags |= GEARB_ST_NO_PAGE;
    }
    *a.used_out = used;
  }
  if (flags && a.status) atomicOr(reinterpret_cast<unsigned *>(a.status), flags);
}

__device__ __forceinline__ int32_t page_at(const gearb_layout_args &a, int64_t k) {
  if (k >= a.num_pages) return -1;
  return a.free_pages ? __ldg(a.free_pages + k) : static_cast<int32_t>(k);
}

// One thread per token: its slot, and the table entry of the page it is the first new token of.
__global__ void layout_fill_kernel(const __grid_constant__ LayoutParams P) {
  const gearb_layout_args &a = P.a;
  const int64_t total = a.offsets[a.requests];
  const int64_t end = total > a.max_tokens ? total : a.max_tokens;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < end;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    if (i >= total) {
      a.slot_map[i] = -1;
      continue;
    }
    int64_t lo = 0, hi = a.requests - 1;  // last request whose offset is <= i: it has this token
    while (lo < hi) {
      const int64_t mid = (lo + hi + 1) >> 1;
      if (a.offsets[mid] <= i) lo = mid;
      else hi = mid - 1;
    }
    const int64_t r = lo;
    int64_t past, n, have, need;
    unsigned flags = 0;
    request_need(a, r, past, n, have, need, flags);
    const int64_t pos = past + (i - a.offsets[r]), blk = pos / a.page, in_page = pos - blk * a.page;
    int32_t *entry = a.block_table + r * a.max_blocks + blk;
    const int32_t page = blk < have ? *entry : page_at(a, P.first_page[r] + (blk - have));
    if (blk >= have && in_page == 0) *entry = page;
    if (i < a.max_tokens) a.slot_map[i] = page < 0 ? -1 : page * a.page + in_page;
  }
}

}  // namespace
}  // namespace gearb

using namespace gearb;

extern "C" {

int64_t gearb_layout_scratch_bytes(int64_t requests) { return requests > 0 ? requests * 8 : 0; }

int gearb_layout_paged(const gearb_layout_args *args, void *stream) {
  TraceRange trace("gearb:layout");
  GEARB_REQUIRE(args, "layout: null argument");
  LayoutParams p;
  p.a = *args;
  const gearb_layout_args &a = p.a;
  GEARB_REQUIRE(a.requests >= 0 && a.max_tokens >= 0 && a.num_pages >= 0, "layout: negative size");
  GEARB_REQUIRE(a.page > 0 && a.max_blocks > 0, "layout: page and max_blocks must be positive");
  // keeps every sum of lengths inside 64 bits
  GEARB_REQUIRE(a.page <= (int64_t(1) << 31) / a.max_blocks && a.requests < (int64_t(1) << 31) &&
                    a.num_pages <= (int64_t(1) << 31),
                "layout: page * max_blocks, requests and num_pages are limited to 2^31");
  GEARB_REQUIRE(a.used_in && a.used_out && a.offsets, "layout: null argument");
  GEARB_REQUIRE(a.requests == 0 || (a.lengths && a.block_table), "layout: null argument");
  GEARB_REQUIRE(a.max_tokens == 0 || a.slot_map, "layout: max_tokens without a slot map");
  GEARB_REQUIRE(a.scratch_bytes >= gearb_layout_scratch_bytes(a.requests) && (a.requests == 0 || a.scratch),
                "layout: scratch of %lld bytes needed", (long long)gearb_layout_scratch_bytes(a.requests));
  p.first_page = static_cast<int64_t *>(a.scratch);
  layout_scan_kernel<<<1, kThreads, 0, as_stream(stream)>>>(p);
  GEARB_CUDA(cudaGetLastError());
  layout_fill_kernel<<<sm_count() * 8, 256, 0, as_stream(stream)>>>(p);
  GEARB_CUDA(cudaGetLastError());
  return GEARB_OK;
}

}  // extern "C"
