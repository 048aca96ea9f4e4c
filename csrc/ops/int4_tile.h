// Launches of the TMEM kernel of the 4-bit products (gemm_int4_tile.cuh), compiled by type in files of their own.
#pragma once

#include "../runtime/host_common.h"
#include "../sm100/gemm_int4_tile.cuh"

namespace fluxb {

// tok: rows of x per tile (32, 64, 128, 256); group: 32, 64, 128. tp.p is complete but for `tiles`.
int int4_tile_bf16(Int4TileParams& tp, int tok, int group, int grid, cudaStream_t stream);
int int4_tile_f16(Int4TileParams& tp, int tok, int group, int grid, cudaStream_t stream);

}  // namespace fluxb
