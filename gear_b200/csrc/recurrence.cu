// Linear recurrences over sequences, forward and backward.
//
//   h_t = a_t * h_(t-1) + x_t                      h_(-1) = h0
//   g_t = dh_t + a_(t+1) * g_(t+1)                 g_last = dh_last + dstate
//   dx_t = g_t,  da_t = sum over the gate's channels of g_t * h_(t-1),  dh0 = a_0 * g_0
//
// with a_t = gate, or exp(gate) (then dgate = da * a).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.h"

namespace gearb {
namespace {

constexpr int kThreads = 128;

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f(float v) { return v; }
template <> __device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f(float v) { return v; }
template <> __device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }

struct Span {
  int64_t first, count;  // rows of a sequence
};

__device__ __forceinline__ Span sequence_span(const gearb_recurrence_args &A, int64_t s) {
  const int64_t rows = A.batch * A.time;
  Span r;
  if (A.offsets) {
    int64_t lo = A.offsets[s], hi = A.offsets[s + 1];
    lo = lo < 0 ? 0 : (lo > rows ? rows : lo);
    hi = hi < lo ? lo : (hi > rows ? rows : hi);
    r.first = lo;
    r.count = hi - lo;
  } else {
    r.first = s * A.time;
    int64_t n = A.lengths ? A.lengths[s] : A.time;
    r.count = n < 0 ? 0 : (n > A.time ? A.time : n);
  }
  return r;
}

__device__ __forceinline__ int64_t place(const gearb_recurrence_args &A, int64_t row, int64_t sb, int64_t sr) {
  const int64_t b = row / A.time;
  return b * sb + (row - b * A.time) * sr;
}

// One thread per sequence and channel.
template <typename TX, typename TA>
__global__ void __launch_bounds__(kThreads) forward_kernel(const __grid_constant__ gearb_recurrence_args A) {
  const int64_t d = static_cast<int64_t>(blockIdx.y) * kThreads + threadIdx.x;
  if (d >= A.width) return;
  const int64_t k = d / (A.width / A.gates);
  const TX *x = static_cast<const TX *>(A.x);
  const TA *gate = static_cast<const TA *>(A.gate);
  for (int64_t s = blockIdx.x; s < A.sequences; s += gridDim.x) {
    const Span sp = sequence_span(A, s);
    float h = A.h0 ? A.h0[s * A.width + d] : 0.0f;
    for (int64_t j = 0; j < sp.count; ++j) {
      const int64_t row = sp.first + (A.reverse ? sp.count - 1 - j : j);
      float a = to_f(gate[place(A, row, A.gate_batch_stride, A.gate_row_stride) + k]);
      if (A.gate_log) a = expf(a);
      const float xv = to_f(x[place(A, row, A.x_batch_stride, A.x_row_stride) + d]);
      if (A.carry) A.carry[row * A.width + d] = h;
      h = (j > 0 || A.h0) ? fmaf(a, h, xv) : xv;
      static_cast<TX *>(A.out)[row * A.width + d] = from_f<TX>(h);
    }
    if (A.state_out) A.state_out[s * A.width + d] = h;
  }
}

template <typename TX, typename TA>
__global__ void __launch_bounds__(kThreads) backward_kernel(const __grid_constant__ gearb_recurrence_args A,
                                                            float *da_rows) {
  const int64_t d = static_cast<int64_t>(blockIdx.y) * kThreads + threadIdx.x;
  if (d >= A.width) return;
  const int64_t k = d / (A.width / A.gates);
  const TA *gate = static_cast<const TA *>(A.gate);
  const TX *dout = static_cast<const TX *>(A.dout);
  for (int64_t s = blockIdx.x; s < A.sequences; s += gridDim.x) {
    const Span sp = sequence_span(A, s);
    float c = A.dstate ? A.dstate[s * A.width + d] : 0.0f;
    for (int64_t j = sp.count; j-- > 0;) {
      const int64_t row = sp.first + (A.reverse ? sp.count - 1 - j : j);
      float a = to_f(gate[place(A, row, A.gate_batch_stride, A.gate_row_stride) + k]);
      if (A.gate_log) a = expf(a);
      const float g = to_f(dout[place(A, row, A.dout_batch_stride, A.dout_row_stride) + d]) + c;
      static_cast<TX *>(A.dx)[row * A.width + d] = from_f<TX>(g);
      float da = (j > 0 || A.h0) ? g * A.carry[row * A.width + d] : 0.0f;
      if (A.gate_log) da *= a;
      da_rows[row * A.width + d] = da;
      c = a * g;
    }
    if (A.dh0) A.dh0[s * A.width + d] = c;
  }
}

// Zeros in the rows that no sequence owns.
template <typename TX, typename TA>
__global__ void rest_kernel(const __grid_constant__ gearb_recurrence_args A, bool backward) {
  const int64_t rows = A.batch * A.time;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    bool owned;
    if (A.offsets) owned = row >= A.offsets[0] && row < A.offsets[A.sequences];
    else owned = !A.lengths || row % A.time < A.lengths[row / A.time];
    if (owned) continue;
    TX *o = static_cast<TX *>(backward ? A.dx : A.out) + row * A.width;
    for (int64_t d = threadIdx.x; d < A.width; d += blockDim.x) o[d] = from_f<TX>(0.0f);
    if (backward)
      for (int64_t d = threadIdx.x; d < A.gates; d += blockDim.x)
        static_cast<TA *>(A.dgate)[row * A.gates + d] = from_f<TA>(0.0f);
  }
}

template <typename TA>
__global__ void gate_sum_kernel(const __grid_constant__ gearb_recurrence_args A, const float *da_rows) {
  const int64_t rows = A.batch * A.time, per = A.width / A.gates;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < rows * A.gates;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t row = i / A.gates;
    bool owned;
    if (A.offsets) owned = row >= A.offsets[0] && row < A.offsets[A.sequences];
    else owned = !A.lengths || row % A.time < A.lengths[row / A.time];
    if (!owned) continue;
    const float *p = da_rows + row * A.width + (i - row * A.gates) * per;
    float sum = 0.0f;
    for (int64_t d = 0; d < per; ++d) sum += p[d];
    static_cast<TA *>(A.dgate)[i] = from_f<TA>(sum);
  }
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
    GEARB_REQUIRE(!rows || (a->dout && a->dx && a->dgate && a->carry), "recurrence: null argument");
  else
    GEARB_REQUIRE(!rows || a->out, "recurrence: null argument");
  return GEARB_OK;
}

template <typename TX, typename TA>
int launch(const gearb_recurrence_args &a, bool backward, cudaStream_t stream) {
  const int64_t rows = a.batch * a.time;
  const dim3 grid(static_cast<unsigned>(a.sequences < 65535 ? (a.sequences > 0 ? a.sequences : 1) : 65535),
                  static_cast<unsigned>((a.width + kThreads - 1) / kThreads));
  if (a.zero_rest && rows > 0 && (a.offsets || a.lengths))
    rest_kernel<TX, TA><<<static_cast<unsigned>(rows < 65535 ? rows : 65535), 128, 0, stream>>>(a, backward);
  if (!backward) {
    forward_kernel<TX, TA><<<grid, kThreads, 0, stream>>>(a);
  } else {
    float *da = static_cast<float *>(a.scratch);
    backward_kernel<TX, TA><<<grid, kThreads, 0, stream>>>(a, da);
    if (rows > 0) gate_sum_kernel<TA><<<sm_count() * 16, 256, 0, stream>>>(a, da);
  }
  GEARB_CUDA(cudaGetLastError());
  return GEARB_OK;
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
  const int64_t all = args->batch * args->time * args->width * 4;
  *scratch_bytes = backward ? all : 0;
  *carry_bytes = all;
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
