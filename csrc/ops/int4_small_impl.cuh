#pragma once

#include "int4_launch.h"

#include <atomic>

namespace fluxb {
extern std::atomic<uint64_t> g_launches;

namespace {

template <bool F16, bool SF16, int G, int NT, int RB>
int launch_small(const Int4Params& p, cudaStream_t stream) {
  using Cfg = Int4SmallCfg<G, NT, RB>;
  static bool configured[64] = {false};
  int dev = 0;
  FLUXB_CUDA_OK(cudaGetDevice(&dev));
  if (dev >= 64 || !configured[dev]) {
    FLUXB_CUDA_OK(cudaFuncSetAttribute(int4_small_kernel<F16, SF16, G, NT, RB>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       Cfg::SMEM_BYTES));
    if (dev < 64) configured[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.tiles * p.splits_k, 1, 1);
  cfg.blockDim = dim3(kInt4Warps * 32, 1, 1);
  cfg.dynamicSmemBytes = Cfg::SMEM_BYTES;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.splits_k;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.splits_k > 1 ? 1 : 0;
  FLUXB_CUDA_OK(cudaLaunchKernelEx(&cfg, int4_small_kernel<F16, SF16, G, NT, RB>, p));
  FLUXB_CUDA_OK(cudaGetLastError());
  g_launches.fetch_add(1, std::memory_order_relaxed);
  note_gemm({FLUXB_KERNEL_INT4_ROWS, Cfg::TOK, Cfg::ROWS, 1, p.splits_k, 0});
  return kOk;
}

template <bool F16, bool SF16, int G>
int launch_small(const Int4Params& p, int rb, cudaStream_t stream) {
  if (rb == 2) return p.M <= 8 ? launch_small<F16, SF16, G, 1, 2>(p, stream) : launch_small<F16, SF16, G, 2, 2>(p, stream);
  return p.M <= 8 ? launch_small<F16, SF16, G, 1, 4>(p, stream) : launch_small<F16, SF16, G, 2, 4>(p, stream);
}

template <bool F16, bool SF16>
int launch_small(const Int4Params& p, int rb, int G, cudaStream_t stream) {
  if (G == 32) return launch_small<F16, SF16, 32>(p, rb, stream);
  if (G == 64) return launch_small<F16, SF16, 64>(p, rb, stream);
  return launch_small<F16, SF16, 128>(p, rb, stream);
}

template <bool F16>
int launch_small(const Int4Params& p, int rb, int G, cudaStream_t stream) {
  return p.scale_f16 ? launch_small<F16, true>(p, rb, G, stream) : launch_small<F16, false>(p, rb, G, stream);
}

}  // namespace
}  // namespace fluxb
