// Recurrences over x of type float.
#include "recurrence_stream.cuh"

namespace gearb {
namespace rec {

int launch_f32(Params &p, bool backward, cudaStream_t stream) {
  return launch_any<float, float>(p, backward, stream);
}

}  // namespace rec
}  // namespace gearb
