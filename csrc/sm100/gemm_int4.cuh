// Products with 4-bit weights and group scales: out[m, n] = sum_k x[m, k] * (q[n, k] - z[n, g]) * s[n, g], g = k / G.
//
// The integers q - z are exact in 16-bit floats, so the tensor cores multiply them with the activations as they are; a
// group's sum is exact up to fp32 rounding, and is multiplied by its scale in fp32 when the group is complete. No weight is
// ever rounded.
//
// Weights are laid out once, in the order in which the lanes of a warp hold the A fragment of a 16 x 16 tile:
//   packed [Np / 128][Kp / 128][8 row blocks][2 halves u][32 lanes][4 words]: lane (g, t) = (lane / 4, lane % 4), word s
//   holds rows g and g + 8 of its 16-row block at columns 64 u + 16 s + 4 t + {0, 1, 2, 3} of the 128, as four pairs
//   i = 0..3 of nibbles at bits 4 i and 16 + 4 i: row g {0, 1}, row g {2, 3}, row g + 8 {0, 1}, row g + 8 {2, 3}.
// A lane's four k are neighbours (instead of the pairs 2t and 2t + 8 of the instruction's own numbering: the order of the
// terms of a sum is free as long as both operands agree), so that it also reads its activations 8 bytes at a time.
// (w >> 4 i) & 0x000f000f | magic is then a pair of 16-bit floats 128 + q (bf16) or 1024 + q (fp16), and one packed
// subtraction of magic + z gives the pair q - z: 11 instructions for 8 weights (9 in fp16).
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
  int32_t tiles, splits_k;       // tiles of the weights (64 or 128 rows); CTAs (of one cluster) that share K
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
  // d = a * b + c
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, float c0, float c1,
                                             float c2, float c3) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%10, %11, %12, %13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
  }
};
template <>
struct Half<true> {
  static constexpr uint32_t kMagic = 0x64006400u;
  static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b) {
    __half2 r = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<uint32_t*>(&r);
  }
  // a / 16 + b
  static __device__ __forceinline__ uint32_t sixteenth(uint32_t a, uint32_t b) {
    const __half2 f = __half2half2(__ushort_as_half(static_cast<unsigned short>(0x2c00)));
    __half2 r = __hfma2(*reinterpret_cast<__half2*>(&a), f, *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<uint32_t*>(&r);
  }
  // d = a * b + c
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, float c0, float c1,
                                             float c2, float c3) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%10, %11, %12, %13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
  }
};

// The four pairs of 16-bit floats q - z of one word; z0, z1: magic + zero point of rows g and g + 8, in both halves.
// (Written as one three-input operation, since the compiler splits an AND and an OR with two constants: 13 ALU instructions
// per word instead of 7, and the ALU, at half rate, is what limits the unpacking.)
// fp16 has ten bits of mantissa: a nibble at bit 4 makes 1024 + 16 q there, and one multiply-add q - z, exactly. That saves two
// of the three shifts; bf16's seven bits leave no room for it.
template <bool F16>
__device__ __forceinline__ void unpack(uint32_t w, uint32_t z0, uint32_t z1, uint32_t& r0a, uint32_t& r0b, uint32_t& r8a,
                                       uint32_t& r8b) {
  using H = Half<F16>;
  auto pick = [](uint32_t v, uint32_t mask) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(v), "r"(mask), "r"(H::kMagic));          // (v & mask) | magic
    return r;
  };
  if constexpr (F16) {
    const uint32_t n0 = H::sub(0x63806380u, z0), n1 = H::sub(0x63806380u, z1);                    // 960 - (1024 + z)
    r0a = H::sub(pick(w, 0x000f000fu), z0);
    r0b = H::sixteenth(pick(w, 0x00f000f0u), n0);
    r8a = H::sub(pick(w >> 8, 0x000f000fu), z1);
    r8b = H::sixteenth(pick(w >> 8, 0x00f000f0u), n1);
  } else {
    r0a = H::sub(pick(w, 0x000f000fu), z0);
    r0b = H::sub(pick(w >> 4, 0x000f000fu), z0);
    r8a = H::sub(pick(w >> 8, 0x000f000fu), z1);
    r8b = H::sub(pick(w >> 12, 0x000f000fu), z1);
  }
}

// magic + zero point, in both halves; I: which byte of zz
template <bool F16, int I>
__device__ __forceinline__ uint32_t magic_zero(uint32_t zz) {
  return __byte_perm(zz, Half<F16>::kMagic >> 8, I | 0x40 | I << 8 | 0x4000);
}
template <bool F16>
__device__ __forceinline__ float half_to_float(uint32_t bits16) {
  if constexpr (F16) return __half2float(__ushort_as_half(static_cast<uint16_t>(bits16)));
  else return __uint_as_float(bits16 << 16);
}

}  // namespace int4

// ----------------------------------------------------------------------------------------
// Few rows. A CTA owns 64 (or 32) rows of the weights, its eight warps take 64 columns of k in turn: every weight is read and
// converted once, every activation goes to the one warp that needs it, and the warps' sums meet in shared memory, those of
// the `splits_k` CTAs of a cluster in distributed shared memory, always in the same order. Up to 8 * NT rows of x.
// What a lane needs for a step it copies itself into a ring of its own in shared memory (cp.async) while it works on the
// steps before: no barriers, few registers, and 50 KB and more in flight per SM, which is what 6.5 TB/s take.
//
// Measured, bf16, groups of 128 (L2 cold): 1 x 16384 x 4096 11.6 us, 3.0 TB/s, of which 4 are start, first loads and the last
// sums; a longer K adds weights at 4.3 TB/s. 16 x 4096 x 16384 fp16, groups of 64, zero points: 17.4 us, 2.2 TB/s. Bound by
// the ALU, which takes 7 of the 11 instructions of each 8 weights (fp16: 5 of 9) at half rate - issue slots 56 % busy, ALU 54 %,
// tensor pipe 14 % -, and by 256 tiles on 148 SMs.
// ----------------------------------------------------------------------------------------
constexpr int kInt4Warps = 8;

template <int G, int NT, int RB_>
struct Int4SmallCfg {
  static constexpr int RB = RB_, ROWS = 16 * RB_;                    // row blocks and rows of the weights
  static constexpr int TOK = 8 * NT;
  static constexpr int GPS = G < 64 ? 64 / G : 1;                    // groups per step of 64 columns
  static constexpr int DEPTH = 2;                                    // steps in the ring
  static constexpr int CTAS = NT == 1 ? 3 : 2;                       // per SM
  // one step of one warp: weights [RB][lane] 16 bytes, scales [GPS][lane] 4 RB, x [NT][4][lane] 8, zeros [GPS][lane] 2 RB
  static constexpr int SC_OFF = RB * 512, X_OFF = SC_OFF + GPS * RB * 128, Z_OFF = X_OFF + NT * 1024,
                       STEP = Z_OFF + GPS * RB * 64;
  static constexpr int PITCH = ROWS + 4;                             // floats per token of a staged tile
  static constexpr int RING_BYTES = kInt4Warps * DEPTH * STEP, TILE_BYTES = (kInt4Warps + 1) * TOK * PITCH * 4;
  static constexpr int SMEM_BYTES = RING_BYTES > TILE_BYTES ? RING_BYTES : TILE_BYTES;
};

template <bool F16, bool SF16, int G, int NT, int RB>
__global__ void __launch_bounds__(kInt4Warps * 32, Int4SmallCfg<G, NT, RB>::CTAS)
    int4_small_kernel(const __grid_constant__ Int4Params p) {
  using H = int4::Half<F16>;
  using Cfg = Int4SmallCfg<G, NT, RB>;
  constexpr int ROWS = Cfg::ROWS;
  constexpr int TOK = Cfg::TOK, PITCH = Cfg::PITCH, GPS = Cfg::GPS, DEPTH = Cfg::DEPTH;
  constexpr int SPG = 4 / GPS;                                       // MMAs per group and step
  extern __shared__ __align__(16) float smem[];                      // the rings, then [warps + 1][TOK][PITCH]
  const int lane = threadIdx.x & 31, warp = ptx::warp_index();
  const int g = lane >> 2, t = lane & 3;
  const int S = p.splits_k;
  const int rank = S > 1 ? static_cast<int>(ptx::cluster_ctarank()) : 0;
  const int tile = blockIdx.x / S, rows = static_cast<int>(p.M);
  const int units = p.Kp / 64;
  const int u0 = static_cast<int>(static_cast<int64_t>(units) * rank / S);
  const int u1 = static_cast<int>(static_cast<int64_t>(units) * (rank + 1) / S);
  const uint4* const wbase =
      p.packed + static_cast<int64_t>(tile * ROWS / 128) * (p.Kp / 128) * 512 + tile * ROWS % 128 / 16 * 64 + lane;
  const int scale_base = tile * ROWS / 64 * 64 + g * 8 + tile * ROWS % 64 / 8;      // (slot of the first row block)
  const uint32_t ring = ptx::smem_u32(smem) + warp * (DEPTH * Cfg::STEP);

  const uint16_t* const x0 = p.x + g * p.ldx + t * 4;
  auto fetch = [&](int u, int slot) {
    const uint32_t to = ring + slot * Cfg::STEP;
    if (u < u1) {
      const uint4* const wu = wbase + static_cast<int64_t>(u >> 1) * 512 + (u & 1) * 32;
#pragma unroll
      for (int r = 0; r < RB; ++r) ptx::cp_async_16(to + r * 512 + lane * 16, wu + r * 64, 16);
#pragma unroll
      for (int j = 0; j < GPS; ++j) {
        const int64_t at = scale_base + static_cast<int64_t>(u * 64 / G + j) * p.Np;
        ptx::cp_async<RB * 4>(to + Cfg::SC_OFF + (j * 32 + lane) * RB * 4, p.scales + at);
        if (p.zeros != nullptr) ptx::cp_async<RB * 2>(to + Cfg::Z_OFF + (j * 32 + lane) * RB * 2, p.zeros + at);
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const uint16_t* const xr = x0 + static_cast<int64_t>(n) * 8 * p.ldx + u * 64;
        const bool in = n * 8 + g < rows;
        // (K is a multiple of 32: the first and the second half of the step are in or out as a whole)
        const bool lo = in && u * 64 < p.K, hi = in && u * 64 + 32 < p.K;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          const bool ok = s < 2 ? lo : hi;
          ptx::cp_async_8(to + Cfg::X_OFF + (n * 4 + s) * 256 + lane * 8, ok ? xr + s * 16 : p.x, ok ? 8 : 0);
        }
      }
    }
    ptx::cp_async_commit();
  };
  float acc[RB][NT][4];
#pragma unroll
  for (int r = 0; r < RB; ++r)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[r][n][i] = 0.f;
#pragma unroll
  for (int d = 0; d < DEPTH; ++d) fetch(u0 + warp + d * kInt4Warps, d);
  int slot = 0;
#pragma unroll 1
  for (int u = u0 + warp; u < u1; u += kInt4Warps) {
    ptx::cp_async_wait<DEPTH - 1>();
    const uint32_t from = ring + slot * Cfg::STEP;
    uint32_t w[RB][4];
#pragma unroll
    for (int r = 0; r < RB; ++r) ptx::ld_shared(from + r * 512 + lane * 16, w[r]);
    uint32_t sc[GPS][RB], zp[GPS][RB / 2], xf[NT][4][2];
#pragma unroll
    for (int j = 0; j < GPS; ++j) {
      ptx::ld_shared(from + Cfg::SC_OFF + (j * 32 + lane) * RB * 4, sc[j]);
#pragma unroll
      for (int r = 0; r < RB / 2; ++r) zp[j][r] = 0x08080808u;
      if (p.zeros != nullptr) ptx::ld_shared(from + Cfg::Z_OFF + (j * 32 + lane) * RB * 2, zp[j]);
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int s = 0; s < 4; ++s) ptx::ld_shared(from + Cfg::X_OFF + (n * 4 + s) * 256 + lane * 8, xf[n][s]);
    fetch(u + DEPTH * kInt4Warps, slot);
    slot = slot + 1 == DEPTH ? 0 : slot + 1;
#pragma unroll
    for (int r = 0; r < RB; ++r) {
#pragma unroll
      for (int j = 0; j < GPS; ++j) {
        const uint32_t zz = zp[j][r / 2];
        const uint32_t z0 = r % 2 ? int4::magic_zero<F16, 2>(zz) : int4::magic_zero<F16, 0>(zz);
        const uint32_t z1 = r % 2 ? int4::magic_zero<F16, 3>(zz) : int4::magic_zero<F16, 1>(zz);
        float part[NT][4];
#pragma unroll
        for (int s = j * SPG; s < (j + 1) * SPG; ++s) {
          uint32_t a[4];
          int4::unpack<F16>(w[r][s], z0, z1, a[0], a[2], a[1], a[3]);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            if (s == j * SPG) H::mma(part[n], a, xf[n][s][0], xf[n][s][1], 0.f, 0.f, 0.f, 0.f);
            else H::mma(part[n], a, xf[n][s][0], xf[n][s][1], part[n][0], part[n][1], part[n][2], part[n][3]);
          }
        }
        const float f0 = int4::half_to_float<SF16>(sc[j][r] & 0xffffu), f1 = int4::half_to_float<SF16>(sc[j][r] >> 16);
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
  ptx::cp_async_wait<0>();
  __syncthreads();                                                 // (the tiles lie over the rings)
  // the warps' sums: D fragment rows are weights (g, g + 8), columns are tokens (2 t, 2 t + 1)
  float* mine = smem + (warp + 1) * TOK * PITCH;
#pragma unroll
  for (int r = 0; r < RB; ++r)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) mine[(n * 8 + 2 * t + (i & 1)) * PITCH + r * 16 + g + (i >> 1) * 8] = acc[r][n][i];
  __syncthreads();
  for (int i = threadIdx.x; i < TOK * ROWS; i += kInt4Warps * 32) {
    const int at = (i / ROWS) * PITCH + i % ROWS;
    float v = 0.f;
#pragma unroll
    for (int wv = 1; wv <= kInt4Warps; ++wv) v += smem[wv * TOK * PITCH + at];
    smem[at] = v;
  }
  if (S > 1) ptx::cluster_sync();
  else __syncthreads();
  for (int i = rank * kInt4Warps * 32 + threadIdx.x; i < rows * ROWS; i += S * kInt4Warps * 32) {
    const int m = i / ROWS, n = tile * ROWS + i % ROWS;
    if (n >= p.N) continue;
    const uint32_t at = ptx::smem_u32(smem + m * PITCH + i % ROWS);
    float v = 0.f;
    if (S > 1) {
      for (int c = 0; c < S; ++c) {
        float part;
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(part) : "r"(ptx::mapa_u32(at, c)));
        v += part;
      }
    } else {
      v = smem[m * PITCH + i % ROWS];
    }
    if (p.bias != nullptr) v += ptx::half_bits_to_float(p.bias[n], F16);
    p.out[m * p.ldo + n] = static_cast<uint16_t>(ptx::pack_half2(F16, v, 0.f));
  }
  if (S > 1) ptx::cluster_sync();                                    // the others may still read this tile
}

}  // namespace fluxb
