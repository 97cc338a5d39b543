// Recurrences over x of type __half.
#include "recurrence_stream.cuh"

namespace gearb {
namespace rec {

int launch_f16(Params &p, bool backward, cudaStream_t stream) {
  return p.A.gate_dtype == GEARB_DT_F32 ? launch_any<__half, float>(p, backward, stream)
                                        : launch_any<__half, __half>(p, backward, stream);
}

}  // namespace rec
}  // namespace gearb
