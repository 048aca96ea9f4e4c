#pragma once

#include "int4_launch.h"

#include <atomic>

namespace fluxb {
extern std::atomic<uint64_t> g_launches;

namespace {

template <class Cfg>
int launch_int4_tile(Int4TileParams& tp, int grid, cudaStream_t stream) {
  static bool configured[64] = {false};
  int dev = 0, rc;
  FLUXB_CUDA_OK(cudaGetDevice(&dev));
  if (dev >= 64 || !configured[dev]) {
    FLUXB_CUDA_OK(cudaFuncSetAttribute(int4_tile_kernel<Cfg>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM_BYTES));
    if (dev < 64) configured[dev] = true;
  }
  uint64_t dims[2] = {static_cast<uint64_t>(tp.p.K), static_cast<uint64_t>(tp.p.M)};
  uint64_t str[1] = {static_cast<uint64_t>(tp.p.ldx) * 2};
  uint32_t box[2] = {64, Cfg::TOK};
  if ((rc = encode_tmap(&tp.tm_x, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, tp.p.x, dims, str, box, Swz::B128))) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid, 1, 1);
  cfg.blockDim = dim3(Cfg::THREADS, 1, 1);
  cfg.dynamicSmemBytes = Cfg::SMEM_BYTES;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = tp.p.splits_k;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = tp.p.splits_k > 1 ? 1 : 0;
  FLUXB_CUDA_OK(cudaLaunchKernelEx(&cfg, int4_tile_kernel<Cfg>, tp));
  FLUXB_CUDA_OK(cudaGetLastError());
  g_launches.fetch_add(1, std::memory_order_relaxed);
  note_gemm({FLUXB_KERNEL_INT4_TILES, Cfg::TOK, 128, 1, tp.p.splits_k, 0});
  return kOk;
}

template <int G, bool F16>
int launch_int4_tile(Int4TileParams& tp, int tok, int grid, cudaStream_t stream) {
  if (tok == 32) return launch_int4_tile<Int4TileCfg<32, G, F16>>(tp, grid, stream);
  if (tok == 64) return launch_int4_tile<Int4TileCfg<64, G, F16>>(tp, grid, stream);
  if (tok == 128) return launch_int4_tile<Int4TileCfg<128, G, F16>>(tp, grid, stream);
  return launch_int4_tile<Int4TileCfg<256, G, F16>>(tp, grid, stream);
}

template <bool F16>
int launch_int4_tile(Int4TileParams& tp, int tok, int group, int grid, cudaStream_t stream) {
  if (group == 32) return launch_int4_tile<32, F16>(tp, tok, grid, stream);
  if (group == 64) return launch_int4_tile<64, F16>(tp, tok, grid, stream);
  return launch_int4_tile<128, F16>(tp, tok, grid, stream);
}

}  // namespace
}  // namespace fluxb
