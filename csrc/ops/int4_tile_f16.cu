#include "int4_tile_impl.cuh"

namespace fluxb {
int int4_tile_f16(Int4TileParams& tp, int tok, int group, int grid, cudaStream_t stream) {
  return launch_int4_tile<true>(tp, tok, group, grid, stream);
}
}  // namespace fluxb
