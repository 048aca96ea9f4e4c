// Host side of the products with 4-bit weights: layout of the weights, argument checks, choice of the kernel, launches.
#include "int4_launch.h"

#include <atomic>
#include <cmath>

namespace fluxb {
extern std::atomic<uint64_t> g_launches;

namespace {

// One thread per word: two 16-bit reads (four neighbouring values of rows g and g + 8), one 32-bit write.
__global__ void int4_layout_kernel(const fluxb_int4_layout_t a, int Np, int Kp, int64_t words) {
  const int64_t stride = static_cast<int64_t>(gridDim.x) * blockDim.x;
  const int64_t blocks = Kp / 128;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < words; i += stride) {
    const int s = static_cast<int>(i % 4), lane = static_cast<int>(i / 4 % 32), u = static_cast<int>(i / 128 % 2);
    const int64_t rest = i / 2048;
    const int kb = static_cast<int>(rest % blocks), nb = static_cast<int>(rest / blocks % (Np / 128));
    const int block = nb * 8 + static_cast<int>(i / 256 % 8), e = static_cast<int>(rest / blocks / (Np / 128));
    const int k = kb * 128 + u * 64 + s * 16 + lane % 4 * 4;
    uint32_t word = 0;
    for (int h = 0; h < 2; ++h) {
      const int n = block * 16 + lane / 4 + h * 8;
      uint32_t v = 0x8888u;                                      // (with zero points: the scale of zero makes them zero)
      if (n < a.N && k < a.K)
        v = *reinterpret_cast<const uint16_t*>(a.q + (static_cast<int64_t>(e) * a.N + n) * (a.K / 2) + k / 2);
      word |= ((v & 0xfu) | (v >> 8 & 0xfu) << 4 | (v >> 4 & 0xfu) << 16 | (v >> 12 & 0xfu) << 20) << (8 * h);
    }
    static_cast<uint32_t*>(a.packed)[i] = word;
  }
}

__global__ void int4_layout_scales_kernel(const fluxb_int4_layout_t a, int Np, int Kp, int G, int64_t count) {
  const int64_t stride = static_cast<int64_t>(gridDim.x) * blockDim.x;
  const int groups = Kp / G, given = a.K / a.group;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < count; i += stride) {
    const int n = static_cast<int>(i % Np), j = static_cast<int>(i / Np % groups), e = static_cast<int>(i / Np / groups);
    const int64_t to = (static_cast<int64_t>(e) * groups + j) * Np + n / 64 * 64 + int4_scale_slot(n % 64);
    const bool in = n < a.N && j * G < a.K;
    const int64_t from = (static_cast<int64_t>(e) * a.N + n) * given + static_cast<int64_t>(j) * G / a.group;
    static_cast<uint16_t*>(a.scales_out)[to] = in ? static_cast<const uint16_t*>(a.scales)[from] : 0;
    if (a.zeros_out != nullptr) a.zeros_out[to] = in ? a.zeros[from] & 15 : 8;
  }
}

int round128(int v) { return (v + 127) / 128 * 128; }

// What a product on the tile kernel takes in us: `ctas` tiles (times CTAs that share K) of 32 << i rows of x, `blocks` blocks of
// 128 columns each, clusters of `splits`. Start, time per block and cost of a cluster as measured on 256 x 1024, 512 x 8192,
// 32 .. 100 x 1024 / 4096 at K = 128 .. 8192 (blocks: K = 8192 less 4096); two CTAs on an SM take 1.5 times as long each.
// What it decides, in us: 256 x 1024 x 1024 7.5 on tiles of 32 (64: 8.0, 128: 9.1, 256: 12.6, on clusters of two 12.8);
// 100 x 1024 x 8192 9.4 on 32 and clusters of eight (128: 36.5, clusters of eight 13.5); 512 x 8192 x 4096 30.8 on 256 (128: 39.3,
// 64: 56, 32: 69); groups of 64 make large tiles wait for more sums: 512 x 8192 x 4096 41, 50, 64, 79.
double int4_tile_us(int i, int splits, int G, double ctas, int blocks, int sms) {
  static const double start[4] = {4.8, 4.8, 5.6, 7.0};
  static const double block[3][4] = {{0.70, 0.75, 1.09, 1.63}, {0.37, 0.43, 0.65, 1.02}, {0.33, 0.38, 0.50, 0.70}};
  static const double cluster[4][4] = {{0.0, 1.4, 1.5, 2.5}, {0.0, 1.4, 2.0, 2.6}, {0.0, 1.8, 3.0, 4.4}, {0.0, 3.2, 5.0, 8.4}};
  // clusters of 1, 2, 4, 8; those between are in the middle
  const int j = splits >= 8 ? 3 : splits >= 4 ? 2 : splits >= 2 ? 1 : 0;
  const double extra = splits == 3 || splits == 6 ? 0.5 * (cluster[i][j] + cluster[i][j + 1]) : cluster[i][j];
  double one = block[G == 32 ? 0 : G == 64 ? 1 : 2][i], rounds = ctas / sms;
  if (i == 0 && rounds > 1.0) {
    one *= 1.5;
    rounds /= 2.0;
  }
  return start[i] + extra + one * blocks * (rounds <= 1.0 ? 1.0 : ceil(rounds));
}

bool shape_ok(int experts, int N, int K, int group) {
  return experts >= 1 && experts <= 512 && N >= 1 && N <= (1 << 24) && K >= 32 && K <= (1 << 24) &&
         (group == 32 || group == 64 || (group >= 128 && group % 128 == 0)) && K % group == 0;
}

}  // namespace
}  // namespace fluxb

using namespace fluxb;

extern "C" int fluxb_int4_layout(const fluxb_int4_layout_t* a) {
  FLUXB_REQUIRE(a && a->q && a->scales && a->packed && a->scales_out, "null arguments");
  FLUXB_REQUIRE((a->zeros != nullptr) == (a->zeros_out != nullptr), "zero points need both arrays");
  FLUXB_REQUIRE(shape_ok(a->experts, a->N, a->K, a->group), "4-bit weights: sizes");
  FLUXB_REQUIRE((reinterpret_cast<uintptr_t>(a->q) & 1) == 0 && (reinterpret_cast<uintptr_t>(a->packed) & 15) == 0 &&
                    (reinterpret_cast<uintptr_t>(a->scales_out) & 15) == 0 && (reinterpret_cast<uintptr_t>(a->zeros_out) & 15) == 0,
                "4-bit weights: alignment");
  const int Np = round128(a->N), Kp = round128(a->K), G = a->group < 128 ? a->group : 128;
  const int64_t words = static_cast<int64_t>(a->experts) * Np * (Kp / 8);
  const int64_t count = static_cast<int64_t>(a->experts) * (Kp / G) * Np;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(a->stream);
  int sms = 0, rc;
  if ((rc = device_sm_count(&sms))) return rc;
  int4_layout_kernel<<<sms * 8, 256, 0, stream>>>(*a, Np, Kp, words);
  int4_layout_scales_kernel<<<sms * 8, 256, 0, stream>>>(*a, Np, Kp, G, count);
  FLUXB_CUDA_OK(cudaGetLastError());
  g_launches.fetch_add(2, std::memory_order_relaxed);
  return kOk;
}

extern "C" int fluxb_int4_gemm(const fluxb_int4_gemm_t* a) {
  FLUXB_REQUIRE(a != nullptr, "null arguments");
  FLUXB_REQUIRE(shape_ok(a->experts, a->N, a->K, a->group), "4-bit product: sizes");
  FLUXB_REQUIRE(a->splits != nullptr || a->experts == 1, "several experts need their row counts");
  FLUXB_REQUIRE(a->M >= 0 && a->M < (1ll << 31), "4-bit product: rows");
  if (a->M == 0) return kOk;
  FLUXB_REQUIRE(a->x && a->packed && a->scales && a->out, "null tensors");
  FLUXB_REQUIRE(a->dtype == FLUXB_BF16 || a->dtype == FLUXB_FP16, "activations must be bf16 or fp16");
  FLUXB_REQUIRE(a->scale_dtype == FLUXB_BF16 || a->scale_dtype == FLUXB_FP16, "scales must be bf16 or fp16");
  FLUXB_REQUIRE(((reinterpret_cast<uintptr_t>(a->x) | reinterpret_cast<uintptr_t>(a->packed) |
                  reinterpret_cast<uintptr_t>(a->scales) | reinterpret_cast<uintptr_t>(a->zeros)) & 15) == 0,
                "4-bit product: 16-byte aligned tensors");
  FLUXB_REQUIRE(a->ldx % 8 == 0 && a->ldx >= 0 && a->ldo >= 0, "rows of the activations must be 16-byte aligned");
  Int4Params p = {};
  p.x = static_cast<const uint16_t*>(a->x);
  p.packed = static_cast<const uint4*>(a->packed);
  p.scales = static_cast<const uint16_t*>(a->scales);
  p.zeros = a->zeros;
  p.bias = static_cast<const uint16_t*>(a->bias);
  p.splits = a->splits;
  p.out = static_cast<uint16_t*>(a->out);
  p.M = a->M;
  p.ldx = a->ldx;
  p.ldo = a->ldo;
  p.E = a->experts;
  p.N = a->N;
  p.K = a->K;
  p.Np = round128(a->N);
  p.Kp = round128(a->K);
  p.scale_f16 = a->scale_dtype == FLUXB_FP16;
  int sms = 0, rc;
  if ((rc = device_sm_count(&sms))) return rc;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(a->stream);
  const int G = a->group < 128 ? a->group : 128;
  const int steps = p.Kp / 128;
  if (a->splits == nullptr && a->M <= 16) {
    // Rows of the weights per CTA, and CTAs that share K (a cluster costs 1 - 2 us to start):
    //  * 64 where that fills the chip: 1 x 16384 x 4096 12.2 us, with 32 rows 13.3, on clusters of two 14.4;
    //  * 32 where it does not: 1 x 4096 x 4096 5.1, with 64 rows and clusters of four 6.0; 16 x 4096 x 4096 7.2 and 7.8;
    //  * 64 and clusters again for a long K: 16 x 4096 x 16384 17.7, with 32 rows 20.7, on clusters of two 21.6.
    const int t64 = (a->N + 63) / 64, t32 = (a->N + 31) / 32;
    const int rb = t64 > sms || steps > 64 ? 4 : 2;
    p.tiles = rb == 4 ? t64 : t32;
    const int room = rb == 4 ? 2 * sms : sms;
    int s = 1;
    while (s < 4 && 2 * s * p.tiles <= room && steps >= 16 * s) s *= 2;
    p.splits_k = s;
    return a->dtype == FLUXB_FP16 ? int4_small_f16(p, rb, G, stream) : int4_small_bf16(p, rb, G, stream);
  }
  Int4TileParams tp = {};
  p.tiles = p.Np / 128;
  int tok = 0;
  double best = 1e30;
  for (int i = 0; i < 4; ++i) {
    const int t = 32 << i, resident = sms * (t == 32 ? 2 : 1);
    // row tiles: at most, and about so many (an expert's last tile is half full on average)
    const int64_t most = (a->M + t - 1) / t + (a->splits ? p.E : 0);
    double about = static_cast<double>((a->M + t - 1) / t);
    if (a->splits) {
      const double each = static_cast<double>(a->M) / p.E;
      about = each < 1.0 ? static_cast<double>(a->M) : p.E * (each < 0.5 * t ? 1.0 : each / t + 0.5);
    }
    if (most * p.tiles >= (1ll << 31)) continue;
    for (int splits : {1, 2, 3, 4, 6, 8}) {
      // (large clusters need that many free SMs in one part of the chip: half of the CTAs that fit have to do)
      if (splits > 1 && (most * p.tiles * splits > (splits > 4 ? resident / 2 : resident) || steps < 2 * splits)) break;
      const double us = int4_tile_us(i, splits, G, about * p.tiles * splits, (steps + splits - 1) / splits, sms);
      if (us < best) {
        best = us;
        tok = t;
        p.splits_k = splits;
      }
    }
  }
  FLUXB_REQUIRE(tok != 0, "4-bit product: too many tiles");
  const int64_t items = ((a->M + tok - 1) / tok + (a->splits ? p.E : 0)) * p.tiles;
  const int resident = sms * (tok == 32 ? 2 : 1);
  tp.p = p;
  tp.out_vec = a->ldo % 8 == 0 && (reinterpret_cast<uintptr_t>(a->out) & 15) == 0;
  tp.timeout_ns = 2000000000ull;
  tp.status = reinterpret_cast<Status*>(a->status);
  const int grid = p.splits_k > 1 ? static_cast<int>(items) * p.splits_k : static_cast<int>(items < resident ? items : resident);
  return a->dtype == FLUXB_FP16 ? int4_tile_f16(tp, tok, G, grid, stream) : int4_tile_bf16(tp, tok, G, grid, stream);
}
