// Products with 4-bit weights and group scales: out[m, n] = sum_k x[m, k] * (q[n, k] - z[n, g]) * s[n, g], g = k / G.
//
// The integers q - z are exact in 16-bit floats, so the tensor cores multiply them with the activations as they are; a
// group's sum is exact up to fp32 rounding, and is multiplied by its scale in fp32 when the group is complete. No weight is
// ever rounded.
//
// Weights are laid out once, in the order in which the lanes of a warp hold the A fragment of a 16 x 16 tile:
//   packed [Np / 16][Kp / 64][32 lanes][4 words]: lane (g, t) = (lane / 4, lane % 4), word s holds rows g and g + 8 of the
//   16-row block at k = 64 u + 16 s + 4 t + {0, 1, 2, 3}, as four pairs i = 0..3 of nibbles at bits 4 i and 16 + 4 i:
//   row g k {0, 1}, row g k {2, 3}, row g + 8 k {0, 1}, row g + 8 k {2, 3}.
// A lane's four k are neighbours (instead of the pairs 2t and 2t + 8 of the instruction's own numbering: the order of the
// terms of a sum is free as long as both operands agree), so that it also reads its activations 8 bytes at a time.
// (w >> 4 i) & 0x000f000f | magic is then a pair of 16-bit floats 128 + q (bf16) or 1024 + q (fp16), and one packed
// subtraction of magic + z gives the pair q - z: 11 instructions for 8 weights.
//   scales [Kp / G][Np], zeros likewise: inside 64 rows the order is (row % 8, row / 16, row / 8 % 2), so that a lane reads
//   the eight values of its rows in four row blocks with one load.
// Rows and columns up to Np and Kp are zero weights (q = z) with zero scales.
#pragma once

#include "ptx.cuh"

namespace fluxb {

struct Int4Params {
  const uint16_t* x;             // [M, K]
  const uint4* packed;
  const uint16_t* scales;
  const uint8_t* zeros;          // null: 8
  const uint16_t* bias;
  const int32_t* splits;         // null: one expert that owns all rows
  uint16_t* out;
  int64_t M, ldx, ldo;
  int32_t E, N, K, Np, Kp;
  int32_t scale_f16;
  int32_t tiles, splits_k;       // 64-row tiles of the weights; CTAs (of one cluster) that share K
};

// position of row n's scale inside its 64 rows
__host__ __device__ constexpr int int4_scale_slot(int n) { return (n % 8) * 8 + (n / 16 % 4) * 2 + n / 8 % 2; }

namespace int4 {

template <bool F16>
struct Half;
template <>
struct Half<false> {
  static constexpr uint32_t kMagic = 0x43004300u;
  static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b) {
    __nv_bfloat162 r = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<uint32_t*>(&r);
  }
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
template <>
struct Half<true> {
  static constexpr uint32_t kMagic = 0x64006400u;
  static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b) {
    __half2 r = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<uint32_t*>(&r);
  }
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

__device__ __forceinline__ uint4 ld_stream(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// First row and row count of expert e, by all lanes of a warp. Counts are taken as they come from the device: negative ones
// count as zero, and rows past the input do not exist.
__device__ __forceinline__ void expert_rows(const Int4Params& p, int e, int lane, int64_t& row0, int& rows) {
  if (p.splits == nullptr) {
    row0 = 0;
    rows = static_cast<int>(p.M);
    return;
  }
  uint32_t before = 0;
  for (int i = lane; i < e; i += 32) before += static_cast<uint32_t>(max(p.splits[i], 0));
  const int mine = max(p.splits[e], 0);
  // (at most 512 experts of at most 2^31 rows: in two halves)
  const uint64_t sum = static_cast<uint64_t>(__reduce_add_sync(0xffffffffu, before & 0xffffu)) +
                       (static_cast<uint64_t>(__reduce_add_sync(0xffffffffu, before >> 16)) << 16);
  row0 = static_cast<int64_t>(sum) < p.M ? static_cast<int64_t>(sum) : p.M;
  rows = static_cast<int>(row0 + mine <= p.M ? mine : p.M - row0);
}

}  // namespace int4

// ----------------------------------------------------------------------------------------
// Few rows. A CTA owns 64 rows of the weights, its eight warps take 128 columns of k in turn: every weight is read and
// converted once, every activation goes to the one warp that needs it, and the warps' sums meet in shared memory, those of
// the `splits_k` CTAs of a cluster in distributed shared memory, always in the same order. 8 * NT rows of x at a time.
// ----------------------------------------------------------------------------------------
constexpr int kInt4Warps = 8;
constexpr int kInt4Rows = 64;

template <int NT>
struct Int4SmallCfg {
  static constexpr int TOK = 8 * NT;
  static constexpr int PITCH = kInt4Rows + 4;                        // floats per token of a staged tile
  static constexpr int SMEM_BYTES = (kInt4Warps + 1) * TOK * PITCH * 4;
};

template <bool F16, int G, int NT>
__global__ void __launch_bounds__(kInt4Warps * 32) int4_small_kernel(const __grid_constant__ Int4Params p) {
  using H = int4::Half<F16>;
  using Cfg = Int4SmallCfg<NT>;
  constexpr int TOK = Cfg::TOK, PITCH = Cfg::PITCH;
  constexpr int GPS = 128 / G;                                       // groups per step of 128 columns
  extern __shared__ float smem[];                                    // [warps + 1][TOK][PITCH]
  const int lane = threadIdx.x & 31, warp = ptx::warp_index();
  const int g = lane >> 2, t = lane & 3;
  const int S = p.splits_k;
  const int rank = S > 1 ? static_cast<int>(ptx::cluster_ctarank()) : 0;
  const int item = blockIdx.x / S;
  const int e = item / p.tiles, tile = item % p.tiles;
  int64_t row0;
  int rows;
  int4::expert_rows(p, e, lane, row0, rows);
  const int steps = p.Kp / 128;
  const int s0 = static_cast<int>(static_cast<int64_t>(steps) * rank / S);
  const int s1 = static_cast<int>(static_cast<int64_t>(steps) * (rank + 1) / S);
  const int64_t units = p.Kp / 64;
  const uint4* wbase = p.packed + ((static_cast<int64_t>(e) * (p.Np / 16) + tile * 4) * units) * 32 + lane;
  const int64_t scale_base = static_cast<int64_t>(e) * (p.Kp / G) * p.Np + tile * 64 + g * 8;

  for (int m0 = 0; m0 < rows; m0 += TOK) {
    float acc[4][NT][4];
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[r][n][i] = 0.f;
    for (int st = s0 + warp; st < s1; st += kInt4Warps) {
      uint4 w[4][2];
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int u = 0; u < 2; ++u) w[r][u] = int4::ld_stream(wbase + (r * units + st * 2 + u) * 32);
      uint4 sc[GPS];
      uint2 zp[GPS];
#pragma unroll
      for (int j = 0; j < GPS; ++j) {
        const int64_t at = scale_base + (static_cast<int64_t>(st) * GPS + j) * p.Np;
        sc[j] = *reinterpret_cast<const uint4*>(p.scales + at);
        zp[j] = p.zeros != nullptr ? *reinterpret_cast<const uint2*>(p.zeros + at) : make_uint2(0x08080808u, 0x08080808u);
      }
      uint2 xf[NT][8];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int m = m0 + n * 8 + g;
        const uint16_t* xr = p.x + (row0 + m) * p.ldx + st * 128 + t * 4;
#pragma unroll
        for (int s = 0; s < 8; ++s)                                  // (K is a multiple of 32: four columns at once are in or out)
          xf[n][s] = m < rows && st * 128 + s * 16 + t * 4 < p.K ? *reinterpret_cast<const uint2*>(xr + s * 16) : make_uint2(0u, 0u);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float part[NT][4];
#pragma unroll
        for (int s = 0; s < 8; ++s) {
          constexpr int SPG = G / 16;                                // k16 steps per group
          const int j = s / SPG;
          if (s % SPG == 0) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int i = 0; i < 4; ++i) part[n][i] = 0.f;
          }
          const uint4 wu = w[r][s / 4];
          const uint32_t word = s % 4 == 0 ? wu.x : s % 4 == 1 ? wu.y : s % 4 == 2 ? wu.z : wu.w;
          const uint32_t zz = (r < 2 ? zp[j].x : zp[j].y) >> (r % 2 * 16);
          const uint32_t z0 = H::kMagic + (zz & 0xffu) * 0x00010001u;
          const uint32_t z1 = H::kMagic + (zz >> 8 & 0xffu) * 0x00010001u;
          uint32_t a[4];
          a[0] = H::sub((word & 0x000f000fu) | H::kMagic, z0);
          a[2] = H::sub((word >> 4 & 0x000f000fu) | H::kMagic, z0);
          a[1] = H::sub((word >> 8 & 0x000f000fu) | H::kMagic, z1);
          a[3] = H::sub((word >> 12 & 0x000f000fu) | H::kMagic, z1);
#pragma unroll
          for (int n = 0; n < NT; ++n) H::mma(part[n], a, xf[n][s].x, xf[n][s].y);
          if (s % SPG == SPG - 1) {
            const uint32_t pair = r == 0 ? sc[j].x : r == 1 ? sc[j].y : r == 2 ? sc[j].z : sc[j].w;
            const float f0 = ptx::half_bits_to_float(static_cast<uint16_t>(pair), p.scale_f16);
            const float f1 = ptx::half_bits_to_float(static_cast<uint16_t>(pair >> 16), p.scale_f16);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              acc[r][n][0] = fmaf(part[n][0], f0, acc[r][n][0]);
              acc[r][n][1] = fmaf(part[n][1], f0, acc[r][n][1]);
              acc[r][n][2] = fmaf(part[n][2], f1, acc[r][n][2]);
              acc[r][n][3] = fmaf(part[n][3], f1, acc[r][n][3]);
            }
          }
        }
      }
    }
    // the warps' sums: D fragment rows are weights (g, g + 8), columns are tokens (2 t, 2 t + 1)
    float* mine = smem + (warp + 1) * TOK * PITCH;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) mine[(n * 8 + 2 * t + (i & 1)) * PITCH + r * 16 + g + (i >> 1) * 8] = acc[r][n][i];
    __syncthreads();
    for (int i = threadIdx.x; i < TOK * kInt4Rows; i += kInt4Warps * 32) {
      const int at = (i / kInt4Rows) * PITCH + i % kInt4Rows;
      float v = 0.f;
#pragma unroll
      for (int wv = 1; wv <= kInt4Warps; ++wv) v += smem[wv * TOK * PITCH + at];
      smem[at] = v;
    }
    if (S > 1) ptx::cluster_sync();
    else __syncthreads();
    const int last = min(rows - m0, TOK);
    for (int i = rank * kInt4Warps * 32 + threadIdx.x; i < last * kInt4Rows; i += S * kInt4Warps * 32) {
      const int m = i / kInt4Rows, n = tile * 64 + i % kInt4Rows;
      if (n >= p.N) continue;
      const uint32_t at = ptx::smem_u32(smem + m * PITCH + i % kInt4Rows);
      float v = 0.f;
      if (S > 1) {
        for (int c = 0; c < S; ++c) {
          float part;
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(part) : "r"(ptx::mapa_u32(at, c)));
          v += part;
        }
      } else {
        v = smem[m * PITCH + i % kInt4Rows];
      }
      if (p.bias != nullptr) v += ptx::half_bits_to_float(p.bias[n], F16);
      p.out[(row0 + m0 + m) * p.ldo + n] = static_cast<uint16_t>(ptx::pack_half2(F16, v, 0.f));
    }
    // the others may still read this tile
    if (S > 1) ptx::cluster_sync();
    else __syncthreads();
  }
}

}  // namespace fluxb
