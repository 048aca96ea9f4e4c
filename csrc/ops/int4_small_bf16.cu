#include "int4_small_impl.cuh"

namespace fluxb {
int int4_small_bf16(const Int4Params& p, int rb, int group, cudaStream_t stream) {
  return launch_small<false>(p, rb, group, stream);
}
}  // namespace fluxb
