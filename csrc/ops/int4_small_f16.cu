#include "int4_small_impl.cuh"

namespace fluxb {
int int4_small_f16(const Int4Params& p, int rb, int group, cudaStream_t stream) {
  return launch_small<true>(p, rb, group, stream);
}
}  // namespace fluxb
