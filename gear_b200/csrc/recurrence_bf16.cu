// Recurrences over x of type __nv_bfloat16.
#include "recurrence_stream.cuh"

namespace gearb {
namespace rec {

int launch_bf16(Params &p, bool backward, cudaStream_t stream) {
  return p.A.gate_dtype == GEARB_DT_F32 ? launch_any<__nv_bfloat16, float>(p, backward, stream)
                                        : launch_any<__nv_bfloat16, __nv_bfloat16>(p, backward, stream);
}

}  // namespace rec
}  // namespace gearb
