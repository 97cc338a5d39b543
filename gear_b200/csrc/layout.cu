// Offsets, block table and slot map of a batch of requests, from their lengths.
//
// n_r tokens are added to request r behind the past_r it has.  Two prefix sums over the requests (tokens, new pages)
// place every request; then every token's slot and every new page's table entry follow from its request alone.  All of it
// is integer arithmetic, in 64 bits where a sum or a slot may need them.
//
// What bounds it: writing 8 bytes per token (the slot map); for a decoding step, the launches.
//   layout_scan_kernel    one CTA, eight requests a thread: up to 8192 requests in one round.
//   layout_sums_kernel, layout_offsets_kernel   more requests: 4096 a CTA; a CTA adds up the sums before its own.
//   layout_fill_kernel    every warp takes one stretch of the tokens, looks its first request up once and walks on from
//                         there: up to 128 tokens of one request a step, four a lane; where less than 32 are left of
//                         it, 32 a step, each lane finding its request among the next 32 offsets, which the warp holds.
//                         Of tokens without slots only the pages are looked at.  How many there are is known on the device
//                         alone: 1024 requests of 16 M tokens with 64 slots, token by token, took one CTA 3.8 s.
// Up to 1024 requests and 4096 slots the scan and the fill are one launch of one CTA.  Measured: 131072 requests,
// 65 M tokens: 189 us (82 at the copy rate; issue slots are taken in 75 % of the cycles, by 64-bit slots' arithmetic), 254
// with 64-bit arithmetic throughout, 1950 with a binary search per token and one CTA's prefix sums.  256 requests, one
// token each: 3.5 us, a launch.
#include "common.h"
#include "warp_search.cuh"

namespace gearb {
namespace {

constexpr int kScanThreads = 1024;
constexpr int kPer = 8;                                // requests a thread
constexpr int64_t kScanMost = kScanThreads * kPer;
constexpr int64_t kFusedSlots = 4096;                  // beyond them the fill gets the whole GPU
constexpr int kBlock = 4096;                           // requests a CTA of the longer way
constexpr int kFillThreads = 256;
constexpr int kFillCtas = 6;                           // an SM: what the registers allow
constexpr int kStep = 128;                             // tokens a warp step
constexpr unsigned kAll = 0xffffffffu;

struct LayoutParams {
  gearb_layout_args a;
  int64_t *first_page;   // [requests]: place of the request's first new page in the free list
  int64_t *sums;         // [2][blocks]: tokens, then pages; then the pages of all
  int64_t blocks;
  int page_shift;        // log2 of the page size, -1: not a power of two
  int vector;            // the slot map can be written 16 bytes at a time
};

__device__ __forceinline__ unsigned page_of(const LayoutParams &P, unsigned pos) {
  return P.page_shift >= 0 ? pos >> P.page_shift : pos / static_cast<unsigned>(P.a.page);
}

// Tokens the request adds and pages it needs for them.
__device__ __forceinline__ void request_need(const LayoutParams &P, int64_t r, int64_t &past, int64_t &n, int64_t &have,
                                             int64_t &need, unsigned &flags) {
  const gearb_layout_args &a = P.a;
  const int64_t room = a.max_blocks * a.page;  // at most 2^31
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
  // ceil(x / page) for x <= 2^31: (x - 1) / page + 1 stays inside 32 bits
  have = past > 0 ? static_cast<int64_t>(page_of(P, static_cast<unsigned>(past - 1))) + 1 : 0;
  const int64_t end = past + n;
  need = (end > 0 ? static_cast<int64_t>(page_of(P, static_cast<unsigned>(end - 1))) + 1 : 0) - have;
}

// Inclusive sums over the CTA's threads of two values; totals to all.  `sm`: 2 x 32 words.
__device__ __forceinline__ void block_sums(int64_t &x, int64_t &y, int64_t &tx, int64_t &ty, int64_t (*sm)[32]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t u = __shfl_up_sync(kAll, x, d), v = __shfl_up_sync(kAll, y, d);
    if (lane >= d) { x += u; y += v; }
  }
  if (lane == 31) { sm[0][warp] = x; sm[1][warp] = y; }
  __syncthreads();
  int64_t u = lane < warps ? sm[0][lane] : 0, v = lane < warps ? sm[1][lane] : 0;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t s = __shfl_up_sync(kAll, u, d), t = __shfl_up_sync(kAll, v, d);
    if (lane >= d) { u += s; v += t; }
  }
  const int64_t bx = __shfl_sync(kAll, u, warp > 0 ? warp - 1 : 0), by = __shfl_sync(kAll, v, warp > 0 ? warp - 1 : 0);
  if (warp > 0) { x += bx; y += by; }
  tx = __shfl_sync(kAll, u, 31);
  ty = __shfl_sync(kAll, v, 31);
  __syncthreads();
}

// What placing one request's tokens takes.
struct Request {
  int64_t r, first, end;   // its tokens are [first, end) of the batch
  int64_t past, have, page0;
};
// `per` requests a thread from r0 on, in front of them `tokens` tokens and `pages` pages; what follows is added to both.
// `own` gets what the thread's (last) request is told.
template <int kRequests>
__device__ __forceinline__ void place_requests(const LayoutParams &P, int64_t r0, int64_t end, int64_t &tokens, int64_t &pages,
                                               unsigned &flags, int64_t (*sm)[32], Request *own = nullptr) {
  const gearb_layout_args &a = P.a;
  int64_t n[kRequests], need[kRequests], x = 0, y = 0, tx, ty;
  const int64_t r = r0 + static_cast<int64_t>(threadIdx.x) * kRequests;
#pragma unroll
  for (int k = 0; k < kRequests; ++k) {
    n[k] = need[k] = 0;
    int64_t past = 0, have = 0;
    if (r + k < end) request_need(P, r + k, past, n[k], have, need[k], flags);
    if (own) {
      own->past = past;
      own->have = have;
    }
    x += n[k];
    y += need[k];
  }
  const int64_t ox = x, oy = y;
  block_sums(x, y, tx, ty, sm);
  int64_t t = tokens + x - ox, p = pages + y - oy;
#pragma unroll
  for (int k = 0; k < kRequests; ++k)
    if (r + k < end) {
      a.offsets[r + k] = t;
      P.first_page[r + k] = p;
      if (own) *own = Request{r + k, t, t + n[k], own->past, own->have, p};
      t += n[k];
      p += need[k];
    }
  tokens += tx;
  pages += ty;
}

// Inside the pool, whatever the counter holds: sums of pages behind it stay inside 64 bits.
__device__ __forceinline__ int64_t used_before(const gearb_layout_args &a) {
  const int64_t u = *a.used_in;
  return u < 0 ? 0 : (u > a.num_pages ? a.num_pages : u);
}
__device__ __forceinline__ void finish_sums(const gearb_layout_args &a, int64_t tokens, int64_t pages, unsigned &flags) {
  a.offsets[a.requests] = tokens;
  if (pages > a.num_pages) {
    pages = a.num_pages;
    flags |= GEARB_ST_NO_PAGE;
  }
  *a.used_out = pages;
}

__device__ __forceinline__ int32_t page_at(const gearb_layout_args &a, int64_t k) {
  if (k >= a.num_pages) return -1;
  return a.free_pages ? __ldg(a.free_pages + k) : static_cast<int32_t>(k);
}

__device__ __forceinline__ Request load_request(const LayoutParams &P, int64_t r) {
  Request q;
  int64_t n, need;
  unsigned flags = 0;
  request_need(P, r, q.past, n, q.have, need, flags);
  q.r = r;
  q.first = P.a.offsets[r];
  q.end = q.first + n;
  q.page0 = P.first_page[r];
  return q;
}
// Slot of token i; writes the table entry of a page whose first new token it is.
__device__ __forceinline__ int64_t place_token(const LayoutParams &P, const Request &q, int64_t i) {
  const gearb_layout_args &a = P.a;
  const unsigned pos = static_cast<unsigned>(q.past + (i - q.first)), blk = page_of(P, pos);
  const unsigned in_page = pos - blk * static_cast<unsigned>(a.page);
  int32_t *entry = a.block_table + q.r * a.max_blocks + blk;
  const bool fresh = blk >= q.have;
  const int32_t page = fresh ? page_at(a, q.page0 + (blk - q.have)) : *entry;
  if (fresh && in_page == 0) *entry = page;
  return page < 0 ? -1 : static_cast<int64_t>(page) * a.page + in_page;
}

// Tokens [lo, hi) of the batch, which have no slots: the table entries of the pages that begin with one of them.  32 requests
// at a time, a lane each; the pages of long ones by the whole warp.
__device__ __forceinline__ void fill_pages(const LayoutParams &P, int64_t lo, int64_t hi, int lane) {
  const gearb_layout_args &a = P.a;
  if (lo >= hi) return;
  auto pages_of = [&](int64_t rows) -> int64_t { return rows > 0 ? int64_t(page_of(P, static_cast<unsigned>(rows - 1))) + 1 : 0; };
  int64_t r = warp_upper_bound<int64_t>(a.offsets, 0, a.requests, lo, lane, LoadPlain()) - 1;
  for (; r < a.requests && a.offsets[r] < hi; r += 32) {
    int64_t b = 0, end = 0, shift = 0;  // pages, and where they are in the free list
    if (r + lane < a.requests) {
      const Request q = load_request(P, r + lane);
      const int64_t t0 = q.first > lo ? q.first : lo, t1 = q.end < hi ? q.end : hi;
      if (t0 < t1) {
        b = pages_of(q.past + (t0 - q.first));
        if (b < q.have) b = q.have;
        end = pages_of(q.past + (t1 - q.first));
        shift = q.page0 - q.have;
      }
    }
    if (__all_sync(kAll, end - b <= 4)) {
      for (; b < end; ++b) a.block_table[(r + lane) * a.max_blocks + b] = page_at(a, shift + b);
      continue;
    }
    for (int l = 0; l < 32; ++l) {
      const int64_t from = __shfl_sync(kAll, b, l), to = __shfl_sync(kAll, end, l), in_list = __shfl_sync(kAll, shift, l);
      for (int64_t k = from + lane; k < to; k += 32) a.block_table[(r + l) * a.max_blocks + k] = page_at(a, in_list + k);
    }
  }
}

// Tokens [lo, stretch) by one warp.
__device__ __forceinline__ void fill_stretch(const LayoutParams &P, int64_t total, int64_t lo, int64_t stretch, int lane) {
  const gearb_layout_args &a = P.a;
  const int64_t hi = stretch < a.max_tokens ? stretch : a.max_tokens;  // with slots
  int64_t i = lo;
  if (i < total && i < hi) {
    // last request whose offset is <= i: it has this token
    Request q = load_request(P, warp_upper_bound<int64_t>(a.offsets, 0, a.requests, i, lane, LoadPlain()) - 1);
    while (i < hi && i < total) {
      if (i >= q.end) {  // usually the next request's
        q = load_request(P, q.r + 1);
        if (i >= q.end)
          q = load_request(P, warp_upper_bound<int64_t>(a.offsets, q.r, a.requests, i, lane, LoadPlain()) - 1);
      }
      const int64_t rest = q.end < hi ? q.end - i : hi - i;  // tokens of this request
      if (rest >= 32) {
        // up to 128 tokens of one request, a group of four a lane, from a multiple of four on.  Counted from the lane's group: a
        // request may have 2^31 tokens, so counted from its first they pass 31 bits.
        const int64_t from = i & ~int64_t(3), stop = i + rest < from + kStep ? i + rest : from + kStep;
        const int before = static_cast<int>(i - from) - 4 * lane, skip = before > 0 ? before : 0;  // of the group, not its own
        const int end = static_cast<int>(stop - from) - 4 * lane;
        if (skip < end) {
          const unsigned size = static_cast<unsigned>(a.page), have = static_cast<unsigned>(q.have);
          const unsigned pos = static_cast<unsigned>(q.past) + static_cast<unsigned>(i - q.first) + static_cast<unsigned>(skip - before),
                         blk = page_of(P, pos);
          const unsigned in_page = pos - blk * size, left = size - in_page;  // tokens the page has room for
          int32_t *entries = a.block_table + q.r * a.max_blocks;
          auto look_up = [&](unsigned b, bool first) -> int64_t {
            if (b < have) return entries[b];
            const int32_t page = page_at(a, q.page0 + (b - have));
            if (first) entries[b] = page;
            return page;
          };
          int64_t page = look_up(blk, in_page == 0);
          int64_t base = page < 0 ? -1 : page * a.page + in_page;
          unsigned b = blk, used = 0, room = left;
          int64_t s[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            s[k] = -1;
            if (k < skip || k >= end) continue;
            if (used == room) {  // the next page; only pages of less than four rows come here twice
              page = look_up(++b, true);
              base = page < 0 ? -1 : page * a.page;
              used = 0;
              room = size;
            }
            s[k] = base < 0 ? -1 : base + used;
            ++used;
          }
          const int64_t t = from + 4 * lane;
          if (skip == 0 && end >= 4 && P.vector) {
            longlong2 *to = reinterpret_cast<longlong2 *>(a.slot_map + t);
            __stcs(to, make_longlong2(s[0], s[1]));
            __stcs(to + 1, make_longlong2(s[2], s[3]));
          } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (k >= skip && k < end) a.slot_map[t + k] = s[k];
          }
        }
        i = stop;
        continue;
      }
      // up to 32 tokens of any requests: each lane finds its own among 32 offsets at a time
      const int64_t t = i + lane;
      const bool mine = t < hi && t < total;
      bool settled = !mine;
      int64_t r = q.r;
      for (int64_t s = q.r + 1; !__all_sync(kAll, settled); s += 32) {
        const int64_t b = s + lane <= a.requests ? a.offsets[s + lane] : total + 1;
        int count = 0;  // offsets of the window at or before this lane's token
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) {
          const int64_t probe = __shfl_sync(kAll, b, count + d - 1);
          if (probe <= t) count += d;
        }
        const int64_t top = __shfl_sync(kAll, b, 31);
        if (count == 31 && top <= t) count = 32;
        if (!settled && count < 32) {
          settled = true;
          r = s + count - 1;
        }
      }
      if (mine) {
        const Request own = r == q.r ? q : load_request(P, r);
        a.slot_map[t] = place_token(P, own, t);
      }
      i += 32;
    }
  }
  for (int64_t t = (total > lo ? total : lo) + lane; t < hi; t += 32) a.slot_map[t] = -1;  // behind the last token
  fill_pages(P, lo > hi ? lo : hi, stretch < total ? stretch : total, lane);
}

// One CTA: the prefix sums, and with kFill (a request a thread at most) everything.
template <bool kFill>
__global__ void __launch_bounds__(kScanThreads) layout_scan_kernel(const __grid_constant__ LayoutParams P) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ int64_t sm[2][32];
  const gearb_layout_args &a = P.a;
  int64_t tokens = 0, pages = used_before(a);
  unsigned flags = 0;
  __syncthreads();  // everybody has read used_in: used_out may be the same word
  Request own{0, 0, 0, 0, 0, 0};
  if (kFill || a.requests <= kScanThreads) place_requests<1>(P, 0, a.requests, tokens, pages, flags, sm, &own);
  else place_requests<kPer>(P, 0, a.requests, tokens, pages, flags, sm);
  if (threadIdx.x == 0) finish_sums(a, tokens, pages, flags);
  if (flags && a.status) atomicOr(reinterpret_cast<unsigned *>(a.status), flags);
  if constexpr (kFill) {
    // A decoding step: a thread places the few tokens of its request itself.
    if (!__syncthreads_or(own.end - own.first > 4)) {
      for (int64_t t = own.first; t < own.end; ++t) {
        const int64_t slot = place_token(P, own, t);
        if (t < a.max_tokens) a.slot_map[t] = slot;
      }
      for (int64_t t = tokens + threadIdx.x; t < a.max_tokens; t += kScanThreads) a.slot_map[t] = -1;
      return;
    }
    const int64_t end = tokens > a.max_tokens ? tokens : a.max_tokens;
    const int64_t each = ((end + 31) / 32 + kStep - 1) / kStep * kStep, lo = (threadIdx.x >> 5) * each;
    if (lo < end) fill_stretch(P, tokens, lo, lo + each < end ? lo + each : end, threadIdx.x & 31);
  }
}

__global__ void __launch_bounds__(kScanThreads) layout_sums_kernel(const __grid_constant__ LayoutParams P) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ int64_t sm[2][32];
  int64_t x = 0, y = 0, tx, ty;
  unsigned flags = 0;
  const int64_t r0 = static_cast<int64_t>(blockIdx.x) * kBlock;
#pragma unroll
  for (int k = 0; k < kBlock / kScanThreads; ++k) {
    const int64_t r = r0 + threadIdx.x + k * kScanThreads;
    int64_t past, n, have, need;
    if (r < P.a.requests) {
      request_need(P, r, past, n, have, need, flags);
      x += n;
      y += need;
    }
  }
  block_sums(x, y, tx, ty, sm);
  if (threadIdx.x == 0) {
    P.sums[blockIdx.x] = tx;
    P.sums[P.blocks + blockIdx.x] = ty;
  }
}

__global__ void __launch_bounds__(kScanThreads) layout_offsets_kernel(const __grid_constant__ LayoutParams P) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ int64_t sm[2][32];
  int64_t x = 0, y = 0, tokens, pages;
  for (int64_t b = threadIdx.x; b < blockIdx.x; b += kScanThreads) {
    x += P.sums[b];
    y += P.sums[P.blocks + b];
  }
  block_sums(x, y, tokens, pages, sm);
  // used_out, which may be the same word, is written by the fill, when all CTAs of this launch have ended
  pages += used_before(P.a);
  unsigned flags = 0;
  const int64_t r0 = static_cast<int64_t>(blockIdx.x) * kBlock, end = r0 + kBlock < P.a.requests ? r0 + kBlock : P.a.requests;
  place_requests<kBlock / kScanThreads>(P, r0, end, tokens, pages, flags, sm);
  if (threadIdx.x == 0 && blockIdx.x == gridDim.x - 1) {
    P.a.offsets[P.a.requests] = tokens;
    P.sums[2 * P.blocks] = pages;
  }
  if (flags && P.a.status) atomicOr(reinterpret_cast<unsigned *>(P.a.status), flags);
}

__global__ void __launch_bounds__(kFillThreads, kFillCtas) layout_fill_kernel(const __grid_constant__ LayoutParams P) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const gearb_layout_args &a = P.a;
  const int64_t total = a.offsets[a.requests];
  if (P.blocks && blockIdx.x == 0 && threadIdx.x == 0) {
    unsigned flags = 0;
    finish_sums(a, total, P.sums[2 * P.blocks], flags);
    if (flags && a.status) atomicOr(reinterpret_cast<unsigned *>(a.status), flags);
  }
  const int64_t end = total > a.max_tokens ? total : a.max_tokens;
  const int64_t warps = static_cast<int64_t>(gridDim.x) * (kFillThreads / 32);
  const int64_t each = ((end + warps - 1) / warps + kStep - 1) / kStep * kStep;
  const int64_t lo = (static_cast<int64_t>(blockIdx.x) * (kFillThreads / 32) + (threadIdx.x >> 5)) * each;
  if (lo < end) fill_stretch(P, total, lo, lo + each < end ? lo + each : end, threadIdx.x & 31);
}

int launch_after(void (*kernel)(LayoutParams), unsigned grid, unsigned threads, const LayoutParams &p, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  GEARB_CUDA(cudaLaunchKernelEx(&cfg, kernel, p));
  return GEARB_OK;
}

}  // namespace
}  // namespace gearb

using namespace gearb;

extern "C" {

int64_t gearb_layout_scratch_bytes(int64_t requests) {
  return requests > 0 ? requests * 8 + 16 * ((requests + kBlock - 1) / kBlock) + 8 : 0;
}

int gearb_layout_paged(const gearb_layout_args *args, void *stream) {
  TraceRange trace("gearb:layout");
  GEARB_REQUIRE(args, "layout: null argument");
  LayoutParams p;
  p.a = *args;
  const gearb_layout_args &a = p.a;
  GEARB_REQUIRE(a.requests >= 0 && a.max_tokens >= 0 && a.num_pages >= 0, "layout: negative size");
  GEARB_REQUIRE(a.page > 0 && a.max_blocks > 0, "layout: page and max_blocks must be positive");
  // keeps positions in 32 bits and every sum of lengths inside 64
  GEARB_REQUIRE(a.page <= (int64_t(1) << 31) / a.max_blocks && a.requests < (int64_t(1) << 31) &&
                    a.num_pages <= (int64_t(1) << 31),
                "layout: page * max_blocks, requests and num_pages are limited to 2^31");
  GEARB_REQUIRE(a.used_in && a.used_out && a.offsets, "layout: null argument");
  GEARB_REQUIRE(a.requests == 0 || (a.lengths && a.block_table), "layout: null argument");
  GEARB_REQUIRE(a.max_tokens == 0 || a.slot_map, "layout: max_tokens without a slot map");
  GEARB_REQUIRE(a.scratch_bytes >= gearb_layout_scratch_bytes(a.requests) && (a.requests == 0 || a.scratch),
                "layout: scratch of %lld bytes needed", (long long)gearb_layout_scratch_bytes(a.requests));
  GEARB_REQUIRE(reinterpret_cast<uintptr_t>(a.scratch) % 8 == 0, "layout: scratch must start on 8 bytes");
  p.first_page = static_cast<int64_t *>(a.scratch);
  p.blocks = a.requests > kScanMost ? (a.requests + kBlock - 1) / kBlock : 0;
  p.sums = p.first_page + a.requests;
  p.page_shift = -1;
  for (int s = 0; s <= 31; ++s)
    if (a.page == int64_t(1) << s) p.page_shift = s;
  p.vector = reinterpret_cast<uintptr_t>(a.slot_map) % 16 == 0;
  cudaStream_t st = as_stream(stream);
  if (p.blocks == 0) {
    if (a.max_tokens > 0 && a.max_tokens <= kFusedSlots && a.requests <= kScanThreads) {
      layout_scan_kernel<true><<<1, kScanThreads, 0, st>>>(p);
      GEARB_CUDA(cudaGetLastError());
      return GEARB_OK;
    }
    layout_scan_kernel<false><<<1, kScanThreads, 0, st>>>(p);
    GEARB_CUDA(cudaGetLastError());
  } else {
    layout_sums_kernel<<<static_cast<unsigned>(p.blocks), kScanThreads, 0, st>>>(p);
    GEARB_CUDA(cudaGetLastError());
    const int rc = launch_after(layout_offsets_kernel, static_cast<unsigned>(p.blocks), kScanThreads, p, st);
    if (rc != GEARB_OK) return rc;
  }
  return launch_after(layout_fill_kernel, static_cast<unsigned>(sm_count() * kFillCtas), kFillThreads, p, st);
}

}  // extern "C"
