// Launches of the kernels of the 4-bit products, compiled by type in files of their own.
#pragma once

#include "../runtime/host_common.h"
#include "../sm100/gemm_int4_tile.cuh"

namespace fluxb {

// Few rows (gemm_int4.cuh). rb: 16-row blocks of the weights per CTA (2, 4); p is complete.
int int4_small_bf16(const Int4Params& p, int rb, int group, cudaStream_t stream);
int int4_small_f16(const Int4Params& p, int rb, int group, cudaStream_t stream);

// More (gemm_int4_tile.cuh). tok: rows of x per tile (32, 64, 128, 256); group: 32, 64, 128; grid: CTAs. tp is complete but
// for the tensor map.
int int4_tile_bf16(Int4TileParams& tp, int tok, int group, int grid, cudaStream_t stream);
int int4_tile_f16(Int4TileParams& tp, int tok, int group, int grid, cudaStream_t stream);

}  // namespace fluxb
