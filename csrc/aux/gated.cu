// Gated activation between the two products of an MLP or of a layer's experts, and its gradient:
//   y = r * a(g) * u          dg = r * dy * u * a'(g)      du = r * dy * a(g)      dr = sum over the row of dy * a(g) * u
// with a = silu, gelu (tanh form) or relu, r one weight per row (the routing weight of a sorted row) or 1.
// silu and gelu are g * sigmoid(z), z = g or 2 sqrt(2/pi) (g + 0.044715 g^3): no cancellation for negative g, and
// a' = sigmoid(z) + g z' sigmoid(z) sigmoid(-z). Everything between loads and stores is fp32, dr is summed in a
// fixed order.
//
// Rows past a device-side count are left as they are, or zeroed in a buffer that the caller has just made.
//
// One pass over memory in the widest pieces that every tensor's rows allow, 32 to 256 threads per row so that each has one
// piece: 32768 x 2048 bf16 with the row weights' gradient 186 us in two kernels, 5.8 TB/s over the eight values read or written
// (88 % of a plain copy; the backward has to read gate and up again). Rows that start on any 2 bytes have only 2-byte pieces,
// four of them in flight per thread: 5000 x 1001 fp16 13.7 us, 2.2 TB/s, bound by instruction issue (one at a time: 19.6 us).
// 512 x 1536 takes 2.8 us, little more than an empty kernel.
#include "../include/fluxb.h"
#include "../runtime/host_common.h"
#include "../sm100/ptx.cuh"

#include <atomic>

namespace fluxb {
extern std::atomic<uint64_t> g_launches;

namespace {

constexpr int kGatedThreads = 256;
constexpr float kGeluA = 1.5957691216057308f;     // 2 sqrt(2 / pi)
constexpr float kGeluB = 0.044715f;

enum : int { kGelu = 1, kRelu = 2, kSilu = 3 };

struct GatedParams {
  const void* gate;
  const void* up;
  const float* row_weight;
  const void* num_rows;
  void* out;
  const void* grad;
  void* dgate;
  void* dup;
  float* drow;
  int64_t rows, gate_stride, up_stride, out_stride, grad_stride, dgate_stride, dup_stride;
  int32_t cols, num_rows_64, zero_rest;
  int32_t tpr;                   // threads per row: 32 .. 256, a power of two
};

template <typename T, int V>
struct alignas(sizeof(T) * V) Piece { T v[V]; };

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// sigmoid(z) and 1 - sigmoid(z) from exp(-|z|): nothing overflows, neither loses digits. (The fast exponential is good to
// 2 + 1.2 |z| roundings of fp32, far below those of a 16-bit result; fp32 results take the exact one.)
template <typename T>
__device__ __forceinline__ float2 sigmoids(float z) {
  const float e = sizeof(T) == 2 ? __expf(-fabsf(z)) : expf(-fabsf(z));
  const float big = __fdividef(1.f, 1.f + e), small = e * big;
  return z >= 0.f ? make_float2(big, small) : make_float2(small, big);
}
template <typename T, int ACT>
__device__ __forceinline__ float act(float g) {
  if constexpr (ACT == kRelu) return g < 0.f ? 0.f : g;           // (NaN stays)
  const float z = ACT == kSilu ? g : kGeluA * (g + kGeluB * g * g * g);
  return g * sigmoids<T>(z).x;
}
// a(g) and a'(g)
template <typename T, int ACT>
__device__ __forceinline__ float2 act_slope(float g) {
  if constexpr (ACT == kRelu) return make_float2(g < 0.f ? 0.f : g, g > 0.f ? 1.f : 0.f);
  const float z = ACT == kSilu ? g : kGeluA * (g + kGeluB * g * g * g);
  const float dz = ACT == kSilu ? 1.f : kGeluA * (1.f + 3.f * kGeluB * g * g);
  const float2 s = sigmoids<T>(z);
  const float q = s.x * s.y;
  return make_float2(g * s.x, q == 0.f ? s.x : s.x + g * dz * q);  // (dz may be infinite there)
}

__device__ __forceinline__ int64_t rows_in_use(const GatedParams& p) {
  if (p.num_rows == nullptr) return p.rows;
  const int64_t n = p.num_rows_64 ? *static_cast<const int64_t*>(p.num_rows) : *static_cast<const int32_t*>(p.num_rows);
  return n < 0 ? 0 : n < p.rows ? n : p.rows;
}

template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kGatedThreads) gated_kernel(const GatedParams p) {
  const int64_t used = rows_in_use(p);
  const int64_t last = p.zero_rest ? p.rows : used;
  const int rpb = kGatedThreads / p.tpr, t = threadIdx.x % p.tpr;
  const int chunks = p.cols / V;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * rpb + threadIdx.x / p.tpr; row < last;
       row += static_cast<int64_t>(gridDim.x) * rpb) {
    using P = Piece<T, V>;
    P* out = reinterpret_cast<P*>(static_cast<T*>(p.out) + row * p.out_stride);
    if (row >= used) {
      P zero;
#pragma unroll
      for (int j = 0; j < V; ++j) zero.v[j] = from_f32<T>(0.f);
      for (int c = t; c < chunks; c += p.tpr) out[c] = zero;
      continue;
    }
    const P* gate = reinterpret_cast<const P*>(static_cast<const T*>(p.gate) + row * p.gate_stride);
    const P* up = reinterpret_cast<const P*>(static_cast<const T*>(p.up) + row * p.up_stride);
    const float r = p.row_weight != nullptr ? p.row_weight[row] : 1.f;
    // (narrow pieces: several at a time, all loads before the first use)
    constexpr int U = V * sizeof(T) >= 16 ? 1 : V * sizeof(T) >= 8 ? 2 : 4;
    for (int c0 = t; c0 < chunks; c0 += U * p.tpr) {
      P g[U], u[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int c = c0 + i * p.tpr;
        if (U == 1 || c < chunks) {
          g[i] = gate[c];
          u[i] = up[c];
        }
      }
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int c = c0 + i * p.tpr;
        if (U > 1 && c >= chunks) break;
        P y;
#pragma unroll
        for (int j = 0; j < V; ++j) y.v[j] = from_f32<T>(r * (act<T, ACT>(to_f32(g[i].v[j])) * to_f32(u[i].v[j])));
        out[c] = y;
      }
    }
  }
}

template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kGatedThreads) gated_bwd_kernel(const GatedParams p) {
  __shared__ float part[kGatedThreads / 32];
  const int64_t used = rows_in_use(p);
  const int rpb = kGatedThreads / p.tpr, t = threadIdx.x % p.tpr;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int chunks = p.cols / V;
  // (every thread of the block takes part in each step: the row sums meet in shared memory)
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * rpb; base < p.rows; base += static_cast<int64_t>(gridDim.x) * rpb) {
    const int64_t row = base + threadIdx.x / p.tpr;
    using P = Piece<T, V>;
    float sum = 0.f;
    if (row < p.rows) {
      P* dgate = reinterpret_cast<P*>(static_cast<T*>(p.dgate) + row * p.dgate_stride);
      P* dup = reinterpret_cast<P*>(static_cast<T*>(p.dup) + row * p.dup_stride);
      if (row >= used) {
        P zero;
#pragma unroll
        for (int j = 0; j < V; ++j) zero.v[j] = from_f32<T>(0.f);
        for (int c = t; c < chunks; c += p.tpr) dgate[c] = dup[c] = zero;
      } else {
        const P* gate = reinterpret_cast<const P*>(static_cast<const T*>(p.gate) + row * p.gate_stride);
        const P* up = reinterpret_cast<const P*>(static_cast<const T*>(p.up) + row * p.up_stride);
        const P* grad = reinterpret_cast<const P*>(static_cast<const T*>(p.grad) + row * p.grad_stride);
        const float r = p.row_weight != nullptr ? p.row_weight[row] : 1.f;
        constexpr int U = V * sizeof(T) >= 16 ? 1 : V * sizeof(T) >= 8 ? 2 : 4;
        for (int c0 = t; c0 < chunks; c0 += U * p.tpr) {
          P g[U], u[U], d[U];
#pragma unroll
          for (int i = 0; i < U; ++i) {
            const int c = c0 + i * p.tpr;
            if (U == 1 || c < chunks) {
              g[i] = gate[c];
              u[i] = up[c];
              d[i] = grad[c];
            }
          }
#pragma unroll
          for (int i = 0; i < U; ++i) {
            const int c = c0 + i * p.tpr;
            if (U > 1 && c >= chunks) break;
            P dg, du;
#pragma unroll
            for (int j = 0; j < V; ++j) {
              const float uj = to_f32(u[i].v[j]), dj = to_f32(d[i].v[j]);
              const float2 a = act_slope<T, ACT>(to_f32(g[i].v[j]));
              sum += dj * (a.x * uj);
              dg.v[j] = from_f32<T>(r * (dj * (uj * a.y)));
              du.v[j] = from_f32<T>(r * (dj * a.x));
            }
            dgate[c] = dg;
            dup[c] = du;
          }
        }
      }
    }
    if (p.drow != nullptr) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (p.tpr > 32) {
        if (lane == 0) part[warp] = sum;
        __syncthreads();
        if (t == 0) {
          sum = 0.f;
          for (int w = 0; w < p.tpr / 32; ++w) sum += part[warp + w];
        }
        __syncthreads();
      }
      if (t == 0 && row < p.rows) p.drow[row] = sum;
    }
  }
}

template <typename T, int V, int ACT>
int launch_gated(GatedParams& p, bool backward, cudaStream_t stream) {
  int sms = 0, rc;
  if ((rc = device_sm_count(&sms))) return rc;
  p.tpr = 32;
  constexpr int U = V * sizeof(T) >= 16 ? 1 : V * sizeof(T) >= 8 ? 2 : 4;
  while (p.tpr < kGatedThreads && p.tpr * V * U < p.cols) p.tpr *= 2;
  const int rpb = kGatedThreads / p.tpr;
  int64_t grid = (p.rows + rpb - 1) / rpb;
  if (grid > sms * 32ll) grid = sms * 32ll;
  if (backward)
    gated_bwd_kernel<T, V, ACT><<<static_cast<unsigned>(grid), kGatedThreads, 0, stream>>>(p);
  else
    gated_kernel<T, V, ACT><<<static_cast<unsigned>(grid), kGatedThreads, 0, stream>>>(p);
  FLUXB_CUDA_OK(cudaGetLastError());
  g_launches.fetch_add(1, std::memory_order_relaxed);
  return kOk;
}

template <typename T, int V>
int launch_gated(GatedParams& p, int act, bool backward, cudaStream_t stream) {
  switch (act) {
    case kGelu: return launch_gated<T, V, kGelu>(p, backward, stream);
    case kRelu: return launch_gated<T, V, kRelu>(p, backward, stream);
    case kSilu: return launch_gated<T, V, kSilu>(p, backward, stream);
    default: return fail(kErrInvalid, "gated activation: gelu, relu or silu");
  }
}

// The widest pieces (up to 16 bytes) that every row of every tensor starts on and consists of.
template <typename T>
int launch_gated(GatedParams& p, int act, bool backward, cudaStream_t stream) {
  uint64_t mix = static_cast<uint64_t>(p.cols) * sizeof(T) | 16u;
  auto add = [&](const void* base, int64_t stride) {
    mix |= reinterpret_cast<uintptr_t>(base) | static_cast<uint64_t>(stride) * sizeof(T);
  };
  add(p.gate, p.gate_stride);
  add(p.up, p.up_stride);
  if (backward) {
    add(p.grad, p.grad_stride);
    add(p.dgate, p.dgate_stride);
    add(p.dup, p.dup_stride);
  } else {
    add(p.out, p.out_stride);
  }
  const int v = static_cast<int>((mix & (~mix + 1)) / sizeof(T));
  if constexpr (sizeof(T) == 2)
    if (v >= 8) return launch_gated<T, 8>(p, act, backward, stream);
  if (v >= 4) return launch_gated<T, 4>(p, act, backward, stream);
  if (v >= 2) return launch_gated<T, 2>(p, act, backward, stream);
  return launch_gated<T, 1>(p, act, backward, stream);
}

int gated(const fluxb_gated_args_t* a, bool backward) {
  FLUXB_REQUIRE(a != nullptr, "null arguments");
  FLUXB_REQUIRE(a->rows >= 0 && a->cols >= 0, "gated activation sizes");
  if (a->rows == 0) return kOk;
  if (a->cols == 0) {
    if (backward && a->drow)
      FLUXB_CUDA_OK(cudaMemsetAsync(a->drow, 0, sizeof(float) * a->rows, reinterpret_cast<cudaStream_t>(a->stream)));
    return kOk;
  }
  FLUXB_REQUIRE(a->gate && a->up, "null inputs");
  FLUXB_REQUIRE(backward ? a->grad && a->dgate && a->dup : a->out != nullptr, "null outputs");
  FLUXB_REQUIRE(!a->drow || a->row_weight, "gradient of row weights that are not there");
  GatedParams p = {};
  p.gate = a->gate;
  p.up = a->up;
  p.row_weight = a->row_weight;
  p.num_rows = a->num_rows;
  p.out = a->out;
  p.grad = a->grad;
  p.dgate = a->dgate;
  p.dup = a->dup;
  p.drow = a->drow;
  p.rows = a->rows;
  p.gate_stride = a->gate_stride;
  p.up_stride = a->up_stride;
  p.out_stride = a->out_stride;
  p.grad_stride = a->grad_stride;
  p.dgate_stride = a->dgate_stride;
  p.dup_stride = a->dup_stride;
  p.cols = a->cols;
  p.num_rows_64 = a->num_rows_64;
  p.zero_rest = a->zero_rest;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(a->stream);
  switch (a->dtype) {
    case FLUXB_FP32: return launch_gated<float>(p, a->act, backward, stream);
    case FLUXB_BF16: return launch_gated<__nv_bfloat16>(p, a->act, backward, stream);
    case FLUXB_FP16: return launch_gated<__half>(p, a->act, backward, stream);
    default: return fail(kErrUnsupported, "gated activation takes fp32, bf16 or fp16");
  }
}

}  // namespace
}  // namespace fluxb

using namespace fluxb;

extern "C" int fluxb_gated_act(const fluxb_gated_args_t* args) { return gated(args, false); }
extern "C" int fluxb_gated_act_bwd(const fluxb_gated_args_t* args) { return gated(args, true); }
