// Routing of tokens to experts: scores of the router's logits, choice of the k experts of a token, their weights, and
// the gradient of the weights with respect to the logits.
//
//   s = softmax(l) over the E experts, or sigmoid(l) of each          c = s + bias  (the bias steers the choice only)
//   G groups of E / G consecutive experts: a group's score is the sum of its `group_top` largest c; the `topk_groups`
//   best groups stay. Of their experts the k with the largest c are chosen, largest first.
//   w = scale * s[chosen] / sum(s[chosen])   (renormalised), or scale * s[chosen]
// Equal values go to the lower index, NaN counts as the lowest value there is. A row that masks every expert (all -inf)
// gets the lowest indices with weights of zero: the k indices of a token are always valid and different.
//
// Backward, with g = dL/dw and D = sum_j g_j w_j:
//   sigmoid, renormalised    dl_i = w_i (g_i - D / scale) (1 - s_i)      sigmoid, plain   dl_i = w_i g_i (1 - s_i)
//   softmax, renormalised    dl_i = w_i (g_i - D / scale)                softmax, plain   dl_e = [e chosen] w_e g_e - p_e D
// (the renormalised softmax is the softmax over the chosen experts alone, which is why p drops out).
//
// One warp per token; a lane holds PER consecutive experts, so that the lowest lane with the largest value holds the
// lowest index, and a row is read in 16-byte pieces.
//
// The choice is exact: it is the one that scores in real numbers give. Without a bias experts are compared by their logits.
// Otherwise scores are computed in 32 bits with a bound on their error, and a token two of whose candidates (or groups) next to
// each other in the order are closer than that is decided again in 64 bits, by the warp that found it (about 3 tokens in a
// thousand with normal logits over 256 experts).
//
// Bound by instructions, not by memory (kernels alone, the L2 holding the logits): 64 tokens over 64 experts 2.8 us, little more
// than an empty kernel; 8192 x 256, 8 of them from 4 of 8 groups, bias: 16.6 us (0.5 TB/s, 67 % of the issue slots), 4 of them for
// the tail of warps that decide close tokens again (12.3 without one), where scores in 64 bits throughout took 37; 16384 x 120
// bf16, 6 of them, with the gradient: 19.8 us in two kernels.
#include "../include/fluxb.h"
#include "../runtime/host_common.h"
#include "../sm100/ptx.cuh"

#include <atomic>

namespace fluxb {
extern std::atomic<uint64_t> g_launches;

namespace {

constexpr int kRouteWarps = 4;
constexpr int kRouteMaxExperts = 512;
constexpr int kRouteMaxGroups = 32;
constexpr unsigned kFull = 0xffffffffu;

struct RouteParams {
  const void* logits;
  int64_t row_stride;            // elements
  const float* bias;             // [E] or null
  int32_t* experts;              // [tokens, k]
  float* weights;                // [tokens, k]
  const float* grad;             // backward: [tokens, k]
  void* dlogits;                 // backward: [tokens, E], type of the logits
  int64_t tokens;
  int32_t E, k, groups, topk_groups, group_top, sigmoid, renorm, vec;
  float scale;
};

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// Unsigned keys in the order of the values. 0: no candidate, 1: NaN, then -inf and up; both zeros have one key.
__device__ __forceinline__ uint64_t key_of(double v) {
  if (isnan(v)) return 1ull;
  const int64_t b = __double_as_longlong(v + 0.0);
  return static_cast<uint64_t>(b) ^ (static_cast<uint64_t>(b >> 63) | 0x8000000000000000ull);
}
__device__ __forceinline__ double value_of(uint64_t key) {
  const uint64_t b = key >> 63 ? key ^ 0x8000000000000000ull : ~key;
  return __longlong_as_double(static_cast<int64_t>(b));
}
__device__ __forceinline__ uint32_t key_of(float v) {
  if (isnan(v)) return 1u;
  const int32_t b = __float_as_int(v + 0.f);
  return static_cast<uint32_t>(b) ^ (static_cast<uint32_t>(b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key >> 31 ? key ^ 0x80000000u : ~key);
}
// largest key of the warp
__device__ __forceinline__ uint32_t warp_max(uint32_t key) { return __reduce_max_sync(kFull, key); }
__device__ __forceinline__ uint64_t warp_max(uint64_t key) {
  const uint32_t hi = static_cast<uint32_t>(key >> 32);
  const uint32_t top = __reduce_max_sync(kFull, hi);
  const uint32_t low = __reduce_max_sync(kFull, hi == top ? static_cast<uint32_t>(key) : 0u);
  return static_cast<uint64_t>(top) << 32 | low;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}
// (fmaxf passes NaN over)
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kFull, v, o));
  return v;
}

// The arithmetic of a choice. 32 bits: errors of the scores, fast exponential and division included. exp is good to
// 2^-21 + |x| 2^-23 relative, and both x s (1 - s) and x exp(-x) stay below 0.4, so two sigmoids differ by what they should to
// 2^-19, two softmax values (whose sum adds its own error) to 2^-18; sums of two to twice that.
template <typename F>
struct Num;
template <>
struct Num<float> {
  using Key = uint32_t;
  static constexpr bool kChecked = true;
  static __device__ __forceinline__ float sigmoid(float l) {
    const float s = __fdividef(1.f, 1.f + __expf(fminf(-l, 80.f)));
    return isnan(l) ? l : s;
  }
  static __device__ __forceinline__ float power(float l, float top) { return __expf(l - top); }
};
template <>
struct Num<double> {
  using Key = uint64_t;
  static constexpr bool kChecked = false;
  static __device__ __forceinline__ double sigmoid(float l) { return 1.0 / (1.0 + exp(-static_cast<double>(l))); }
  static __device__ __forceinline__ double power(float l, float top) {
    return exp(static_cast<double>(l) - static_cast<double>(top));
  }
};

// This lane's PER logits of one row; -inf past the last expert.
template <typename T, int PER>
__device__ __forceinline__ void load_row(const RouteParams& p, int64_t token, int lane, float (&l)[PER]) {
  constexpr int V = 16 / sizeof(T) < PER ? 16 / sizeof(T) : PER;
  const T* row = static_cast<const T*>(p.logits) + token * p.row_stride;
  const int e0 = lane * PER;
  if (p.vec) {
#pragma unroll
    for (int i = 0; i < PER; i += V) {
      struct alignas(sizeof(T) * V) Piece { T v[V]; };
      Piece piece;
      const bool in = e0 + i < p.E;            // (E is a multiple of V then)
      if (in) piece = *reinterpret_cast<const Piece*>(row + e0 + i);
#pragma unroll
      for (int j = 0; j < V; ++j) l[i + j] = in ? to_f32(piece.v[j]) : -INFINITY;
    }
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i) l[i] = e0 + i < p.E ? to_f32(row[e0 + i]) : -INFINITY;
  }
}

// Whether two values that follow each other in the order are too close to be sure of it.
__device__ __forceinline__ bool uncertain(float v, float next, float tau) { return v - next <= tau + fabsf(v) * 0x1p-22f; }

// The k largest of the lanes' keys, largest first; lane j < k returns the j-th expert. `tau` >= 0: also whether neighbours in the
// order, the first one that is left among them, are uncertain.
// The (k + 1)-th largest of the lanes' own maxima bounds from below what can be among the first k + 1: the few keys that reach
// it are packed into the first lanes, which then count the larger ones. About 200 instructions; taking one key after the other
// costs 16 + 6 PER each, so it is left for a few experts out of up to 128 (16384 tokens, 6 of 120, with the gradient: 18.4 us
// against 20.5; 8192 tokens, 8 of 256: 21 against 16.5), and for rows where more than 32 keys reach the bound.
template <typename K, int PER>
__device__ __forceinline__ int take_best(const K (&key)[PER], int k, int lane, float tau, K* buf /* shared, 32 */, bool& close) {
  int mine = 0;
  if (PER > 4 || k > 8) {
    K own = key[0];
#pragma unroll
    for (int i = 1; i < PER; ++i) own = max(own, key[i]);
    buf[lane] = own;
    __syncwarp();
    int rank = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const K other = buf[i];
      rank += other > own || (other == own && i < lane) ? 1 : 0;
    }
    __syncwarp();
    const unsigned at_k = __ballot_sync(kFull, rank == k);              // (none: k = 32)
    const K bound = at_k ? __shfl_sync(kFull, own, __ffs(at_k) - 1) : K(0);
    int count = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) count += key[i] >= bound && key[i] != 0 ? 1 : 0;
    int end = count;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(kFull, end, o);
      if (lane >= o) end += v;
    }
    const int total = __shfl_sync(kFull, end, 31);
    if (bound != 0 && total <= 32) {
      int to = end - count, which = 0;
      K value = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        if (key[i] >= bound && key[i] != 0) {
          buf[to] = key[i];
          reinterpret_cast<int*>(buf + 32)[to] = lane * PER + i;
          ++to;
        }
      }
      __syncwarp();
      if (lane < total) {
        value = buf[lane];
        which = reinterpret_cast<int*>(buf + 32)[lane];
      }
      int place = 0;
      for (int i = 0; i < total; ++i) {
        const K other = buf[i];
        place += other > value || (other == value && i < lane) ? 1 : 0;
      }
      __syncwarp();
      if (lane < total) {
        buf[place] = value;
        reinterpret_cast<int*>(buf + 32)[place] = which;
      }
      __syncwarp();
      mine = lane < total ? reinterpret_cast<int*>(buf + 32)[lane] : 0;
      if (tau >= 0.f) {
        const K v = lane < total ? buf[lane] : K(0), next = lane + 1 < total ? buf[lane + 1] : K(0);
        // (nothing left: certain; NaN: for the other path to say)
        const float a = static_cast<float>(value_of(v)), b = static_cast<float>(value_of(next));
        if (lane < k && next != 0 && (next == 1 || uncertain(a, b, tau))) close = true;
      }
      __syncwarp();
      return mine;
    }
  }
  uint32_t taken = 0;
  float before = INFINITY;
#pragma unroll 1
  for (int j = 0; j <= k; ++j) {
    K best = 0;
    int at = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (!(taken >> i & 1u) && key[i] > best) {
        best = key[i];
        at = i;
      }
    }
    const K top = warp_max(best);
    if (tau >= 0.f) {
      const float v = top > 1 ? static_cast<float>(value_of(top)) : -INFINITY;
      if (top == 1 || (j > 0 && top != 0 && uncertain(before, v, tau))) close = true;
      before = v;
    }
    if (j == k) break;
    const int winner = __ffs(__ballot_sync(kFull, best == top)) - 1;
    const int e = __shfl_sync(kFull, lane * PER + at, winner);
    if (lane == j) mine = e;
    if (lane == winner) taken |= 1u << at;
  }
  return mine;
}

// The choice in F; `close` (float): some comparison may have come out wrong.
template <typename F, int PER>
__device__ __forceinline__ int choose(const RouteParams& p, const float (&l)[PER], float row_max, int lane,
                                      typename Num<F>::Key* keys /* shared: [E] with groups, 48 without */, bool& close) {
  using N = Num<F>;
  using K = typename N::Key;
  const int e0 = lane * PER;
  const bool by_logit = p.bias == nullptr, sums = p.groups > 1 && p.group_top == 2;
  const float tau = p.sigmoid ? 0x1p-19f : 0x1p-18f;
  K key[PER], gkey[PER];               // experts, and for the groups' scores
#pragma unroll
  for (int i = 0; i < PER; ++i) gkey[i] = key[i] = e0 + i < p.E ? static_cast<K>(key_of(static_cast<F>(l[i]))) : K(0);
  if (!by_logit || sums) {
    F s[PER];
    if (p.sigmoid) {
#pragma unroll
      for (int i = 0; i < PER; ++i) s[i] = N::sigmoid(l[i]);
    } else {
      F sum = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        s[i] = row_max == -INFINITY ? (isnan(l[i]) ? static_cast<F>(NAN) : F(0)) : N::power(l[i], row_max);
        sum += s[i];
      }
      sum = warp_sum(sum);
      const F inv = sum == F(0) ? F(0) : F(1) / sum;
#pragma unroll
      for (int i = 0; i < PER; ++i) s[i] *= inv;
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const bool in = e0 + i < p.E;
      if (!by_logit && in) s[i] += static_cast<F>(p.bias[e0 + i]);
      if (in) gkey[i] = key_of(s[i]);
      if (!by_logit) key[i] = gkey[i];
    }
  }
  if (p.groups > 1) {
    const int size = p.E / p.groups, span = size / PER;           // experts of a group; lanes, if it begins and ends with lanes
    K mine = 0;                                                   // lane g: key of group g's score
    const bool whole = size % PER == 0 && (span & (span - 1)) == 0;
    if (whole) {
      K a = 0, b = 0;                                             // the two largest of this lane, then of its group
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        b = max(b, min(a, gkey[i]));
        a = max(a, gkey[i]);
      }
      for (int o = 1; o < span; o <<= 1) {
        const K a2 = __shfl_xor_sync(kFull, a, o), b2 = __shfl_xor_sync(kFull, b, o);
        b = max(min(a, a2), max(b, b2));
        a = max(a, a2);
      }
      K total = a;
      // (key 1 stands for NaN, which makes the sum the lowest too)
      if (p.group_top == 2) total = b <= 1 ? K(1) : static_cast<K>(key_of(value_of(a) + value_of(b)));
      mine = __shfl_sync(kFull, total, min(lane * span, 31));
      if (lane >= p.groups) mine = 0;
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (e0 + i < p.E) keys[e0 + i] = gkey[i];
      __syncwarp();
#pragma unroll 1
      for (int g = 0; g < p.groups; ++g) {
        K a = 0, b = 0;
        for (int i = lane; i < size; i += 32) {
          const K x = keys[g * size + i];
          b = max(b, min(a, x));
          a = max(a, x);
        }
        const K first = warp_max(a);
        K total = first;
        if (p.group_top == 2) {
          const int winner = __ffs(__ballot_sync(kFull, a == first)) - 1;
          const K second = warp_max(lane == winner ? b : a);
          total = second <= 1 ? K(1) : static_cast<K>(key_of(value_of(first) + value_of(second)));
        }
        if (lane == g) mine = total;
      }
      __syncwarp();
    }
    int rank = 0;
    for (int g = 0; g < p.groups; ++g) {
      const K other = __shfl_sync(kFull, mine, g);
      rank += other > mine || (other == mine && g < lane) ? 1 : 0;
    }
    const bool group = lane < p.groups;
    const unsigned kept = __ballot_sync(kFull, group && rank < p.topk_groups);
    if (N::kChecked && (!by_logit || sums) && p.topk_groups < p.groups) {
      // the last group that stays and the first that goes
      const K in = __shfl_sync(kFull, mine, __ffs(__ballot_sync(kFull, group && rank == p.topk_groups - 1)) - 1);
      const K out = __shfl_sync(kFull, mine, __ffs(__ballot_sync(kFull, group && rank == p.topk_groups)) - 1);
      const float v = static_cast<float>(value_of(in)), w = static_cast<float>(value_of(out));
      if (in <= 1 || out <= 1 || !(v - w > 2.f * tau + fabsf(v) * 0x1p-21f)) close = true;
    }
    if (whole) {
      const bool out = !(kept >> min(lane / span, 31) & 1u);
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (out) key[i] = 0;
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (e0 + i < p.E && !(kept >> ((e0 + i) / size) & 1u)) key[i] = 0;
    }
  }
  return take_best<K, PER>(key, p.k, lane, N::kChecked && !by_logit ? tau : -1.f, keys, close);
}

template <typename T, int PER>
__global__ void __launch_bounds__(kRouteWarps * 32) route_kernel(const RouteParams p) {
  extern __shared__ uint64_t key_space[];           // [warps][max(E, 48)]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t token = static_cast<int64_t>(blockIdx.x) * kRouteWarps + warp;
  if (token >= p.tokens) return;
  float l[PER];
  load_row<T, PER>(p, token, lane, l);
  float top = l[0];
#pragma unroll
  for (int i = 1; i < PER; ++i) top = fmaxf(top, l[i]);
  const float row_max = warp_max(top);
  bool close = false;
  uint64_t* const keys = key_space + warp * max(p.E, 48);
  int e = choose<float, PER>(p, l, row_max, lane, reinterpret_cast<uint32_t*>(keys), close);
  if (__any_sync(kFull, close)) e = choose<double, PER>(p, l, row_max, lane, keys, close);

  // weights: lane j holds the j-th expert
  const bool live = lane < p.k;
  const float le = live ? to_f32(static_cast<const T*>(p.logits)[token * p.row_stride + e]) : -INFINITY;
  float w;
  if (p.sigmoid) {
    // sigmoid(l) exp(-c) with c the largest chosen logit if that is negative: the quotient keeps its digits where all
    // the sigmoids are close to zero
    const float c = p.renorm ? fminf(warp_max(le), 0.f) : 0.f;
    w = le >= 0.f ? 1.f / (1.f + expf(-le)) : expf(le - c) / (1.f + expf(le));
    if (live && le == -INFINITY) w = 0.f;
  } else {
    // (a NaN in the row reaches every weight, as in any softmax)
    float sum = 0.f;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      nan |= isnan(l[i]);
      sum += p.renorm || row_max == -INFINITY ? 0.f : expf(l[i] - row_max);
    }
    if (!p.renorm) sum = warp_sum(sum);
    if (__any_sync(kFull, nan)) sum = NAN;
    const float c = p.renorm ? warp_max(le) : row_max;
    w = c == -INFINITY ? 0.f : expf(le - c);
    if (isnan(sum)) w = NAN;
    else if (!p.renorm) w = sum > 0.f ? w / sum : 0.f;
  }
  if (p.renorm) {
    const float total = warp_sum(live ? w : 0.f);
    w = total == 0.f ? 0.f : w / total;
  }
  if (live) {
    p.experts[token * p.k + lane] = e;
    p.weights[token * p.k + lane] = w * p.scale;
  }
}

template <typename T, int PER>
__global__ void __launch_bounds__(kRouteWarps * 32) route_bwd_kernel(const RouteParams p) {
  constexpr int V = 16 / sizeof(T) < PER ? 16 / sizeof(T) : PER;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t token = static_cast<int64_t>(blockIdx.x) * kRouteWarps + warp;
  if (token >= p.tokens) return;
  const bool live = lane < p.k;
  const int e = live ? p.experts[token * p.k + lane] : 0;
  const float w = live ? p.weights[token * p.k + lane] : 0.f;
  const float g = live ? p.grad[token * p.k + lane] : 0.f;
  const float dot = warp_sum(w * g);
  const T* row = static_cast<const T*>(p.logits) + token * p.row_stride;
  T* out = static_cast<T*>(p.dlogits) + token * p.E;
  const int e0 = lane * PER;
  float d[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) d[i] = 0.f;
  if (!p.sigmoid && !p.renorm) {
    float l[PER];
    load_row<T, PER>(p, token, lane, l);
    float top = l[0];
#pragma unroll
    for (int i = 1; i < PER; ++i) top = fmaxf(top, l[i]);
    const float row_max = warp_max(top);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      d[i] = row_max == -INFINITY ? (isnan(l[i]) ? l[i] : 0.f) : expf(l[i] - row_max);
      sum += d[i];
    }
    sum = warp_sum(sum);
    const float f = sum == 0.f ? 0.f : -dot / sum;
#pragma unroll
    for (int i = 0; i < PER; ++i) d[i] *= f;
  }
  // the chosen experts' terms, added where they belong
  float mine;
  if (p.renorm) {
    mine = w * (g - dot / p.scale);
  } else {
    mine = w * g;
  }
  if (p.sigmoid && live) {
    const float le = to_f32(row[e]);
    mine *= le >= 0.f ? expf(-le) / (1.f + expf(-le)) : 1.f / (1.f + expf(le));
  }
  for (int j = 0; j < p.k; ++j) {
    const int ej = __shfl_sync(kFull, e, j);
    const float v = __shfl_sync(kFull, mine, j);
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (e0 + i == ej) d[i] += v;
  }
  if (p.E % V == 0) {
#pragma unroll
    for (int i = 0; i < PER; i += V) {
      struct alignas(sizeof(T) * V) Piece { T v[V]; };
      Piece piece;
#pragma unroll
      for (int j = 0; j < V; ++j) piece.v[j] = from_f32<T>(d[i + j]);
      if (e0 + i < p.E) *reinterpret_cast<Piece*>(out + e0 + i) = piece;
    }
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (e0 + i < p.E) out[e0 + i] = from_f32<T>(d[i]);
  }
}

template <typename T, int PER>
int launch_route(RouteParams& p, bool backward, cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T) < PER ? 16 / sizeof(T) : PER;
  p.vec = p.E % V == 0 && p.row_stride % V == 0 && reinterpret_cast<uintptr_t>(p.logits) % (V * sizeof(T)) == 0;
  const int64_t grid = (p.tokens + kRouteWarps - 1) / kRouteWarps;
  FLUXB_REQUIRE(grid <= 0x7fffffff, "too many tokens");
  if (backward) {
    route_bwd_kernel<T, PER><<<static_cast<unsigned>(grid), kRouteWarps * 32, 0, stream>>>(p);
  } else {
    const size_t smem = sizeof(uint64_t) * kRouteWarps * (p.E > 48 ? p.E : 48);
    route_kernel<T, PER><<<static_cast<unsigned>(grid), kRouteWarps * 32, smem, stream>>>(p);
  }
  FLUXB_CUDA_OK(cudaGetLastError());
  g_launches.fetch_add(1, std::memory_order_relaxed);
  return kOk;
}

template <typename T>
int launch_route(RouteParams& p, bool backward, cudaStream_t stream) {
  if (p.E <= 64) return launch_route<T, 2>(p, backward, stream);
  if (p.E <= 128) return launch_route<T, 4>(p, backward, stream);
  if (p.E <= 256) return launch_route<T, 8>(p, backward, stream);
  return launch_route<T, 16>(p, backward, stream);
}

int route(const fluxb_route_args_t* a, bool backward) {
  FLUXB_REQUIRE(a != nullptr, "null arguments");
  FLUXB_REQUIRE(a->tokens >= 0 && a->num_experts >= 1 && a->num_experts <= kRouteMaxExperts, "routing sizes");
  FLUXB_REQUIRE(a->num_groups >= 1 && a->num_groups <= kRouteMaxGroups && a->num_experts % a->num_groups == 0,
                "experts must divide over at most 32 groups");
  const int size = a->num_experts / a->num_groups;
  FLUXB_REQUIRE(a->topk_groups >= 1 && a->topk_groups <= a->num_groups, "groups to keep");
  FLUXB_REQUIRE(a->group_top == 1 || (a->group_top == 2 && size >= 2), "group scores sum one or two experts");
  FLUXB_REQUIRE(a->topk >= 1 && a->topk <= 32 && a->topk <= a->topk_groups * size, "experts per token");
  if (a->tokens == 0) return kOk;
  FLUXB_REQUIRE(a->logits && a->experts && a->weights, "null routing tensors");
  FLUXB_REQUIRE(!backward || (a->grad && a->dlogits), "null gradients");
  FLUXB_REQUIRE(!backward || (reinterpret_cast<uintptr_t>(a->dlogits) & 15) == 0, "dlogits must be 16-byte aligned");
  FLUXB_REQUIRE(a->row_stride >= 0, "row stride");
  FLUXB_REQUIRE(a->scale != 0.f && a->scale - a->scale == 0.f, "scale must be finite and not zero");
  RouteParams p = {};
  p.logits = a->logits;
  p.row_stride = a->row_stride;
  p.bias = a->bias;
  p.experts = a->experts;
  p.weights = a->weights;
  p.grad = a->grad;
  p.dlogits = a->dlogits;
  p.tokens = a->tokens;
  p.E = a->num_experts;
  p.k = a->topk;
  p.groups = a->num_groups;
  p.topk_groups = a->topk_groups;
  p.group_top = a->group_top;
  p.sigmoid = a->score == FLUXB_SCORE_SIGMOID;
  p.renorm = a->renormalize != 0;
  p.scale = a->scale;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(a->stream);
  switch (a->dtype) {
    case FLUXB_FP32: return launch_route<float>(p, backward, stream);
    case FLUXB_BF16: return launch_route<__nv_bfloat16>(p, backward, stream);
    case FLUXB_FP16: return launch_route<__half>(p, backward, stream);
    default: return fail(kErrUnsupported, "routing takes fp32, bf16 or fp16 logits");
  }
}

}  // namespace
}  // namespace fluxb

using namespace fluxb;

extern "C" int fluxb_moe_route(const fluxb_route_args_t* args) { return route(args, false); }
extern "C" int fluxb_moe_route_bwd(const fluxb_route_args_t* args) { return route(args, true); }
