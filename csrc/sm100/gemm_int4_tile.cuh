// Products with 4-bit weights for more than a few rows: the weights' integers go through TMEM.
//
// A tile is 128 rows of the weights (the M of the MMA) times TOK rows of x (its N). Four warps unpack the weights of the
// next 128 columns of k and store them into TMEM, where the MMA reads its A operand: the 32 KB of 16-bit integers never pass
// through shared memory, whose bandwidth (128 bytes a cycle for writing and reading both) would bound the kernel at half the
// speed at which memory delivers the packed weights. x tiles arrive by TMA as the B operand.
// Every group's product lands in a fresh accumulator; eight warps multiply it with the group's scale (a thread owns one row
// of the weights, so that is one number) and add it to their fp32 sums in registers. With TOK = 256 the accumulator is two
// halves of 128 columns: the sums of one half are taken while the other is multiplied, and one unpacked weight serves 256
// rows. Smaller TOK alternate two accumulators between groups.
//
//   warps 0 .. 7    sums: TMEM lanes 32 (warp % 4), the first or second half of the columns (warp / 4); epilogue
//   warps 8 .. 11   weights: packed words by cp.async into a ring of their own (a lane reads back what it copied, so the
//                   ring needs no barriers), unpacked into TMEM
//   warp 12         TMA of x, warp 13 MMA issue
// One CTA per SM walks the tiles of all experts; the loads of a tile run ahead into the one before. With splits_k > 1 a
// cluster shares one tile, each CTA with its part of k, and the sums meet in distributed shared memory in rank order.
#pragma once

#include "gemm_int4.cuh"

namespace fluxb {

struct Int4TileParams {
  CUtensorMap tm_x;              // x [M, K], box {64, TOK}
  Int4Params p;                  // tiles: 128-row tiles of the weights
  int32_t out_vec;               // 16-byte stores are aligned
  uint64_t timeout_ns;
  Status* status;
};

constexpr int kInt4MaxExperts = 512;

template <int TOK_, int G_, bool F16_>
struct Int4TileCfg {
  static constexpr int TOK = TOK_, G = G_;
  static constexpr bool F16 = F16_;
  static constexpr int THREADS = 512;
  static constexpr int HALVES = TOK_ == 256 ? 2 : 1;
  static constexpr int NMMA = TOK_ / HALVES;
  static constexpr int CPT = TOK_ / 2;                   // columns of a thread
  static constexpr int GPS = 128 / G_;                   // groups per 128 columns of k
  static constexpr int A_BUFS = 4, A_COL = 256;          // TMEM: accumulators in columns 0 .. 255, weights behind them
  static constexpr int XS_BYTES = TOK_ * 128;            // one stage: 64 columns of k
  static constexpr int X_STAGES = TOK_ == 256 ? 5 : TOK_ == 128 ? 6 : 12;
  static constexpr int PF = TOK_ == 256 ? 4 : 8;         // blocks of 128 columns in the ring of packed weights
  static constexpr int W_BYTES = PF * 8192, Z_BYTES = PF * GPS * 512;
  static constexpr int EPI_BYTES = 2 * 16 * 128 * 4;     // 16 rows of the output at a time for each half
  static constexpr int TAB_BYTES = (2 * (kInt4MaxExperts + 1) * 4 + 15) / 16 * 16;
  static constexpr int BAR_BYTES = 512;
  static constexpr int X_OFF = 0, W_OFF = X_STAGES * XS_BYTES, Z_OFF = W_OFF + W_BYTES, EPI_OFF = Z_OFF + Z_BYTES,
                       TAB_OFF = EPI_OFF + EPI_BYTES, BAR_OFF = TAB_OFF + TAB_BYTES;
  static constexpr int SMEM_BYTES = BAR_OFF + BAR_BYTES + 1024;
  static_assert(SMEM_BYTES <= 227 * 1024, "shared memory");
  static_assert(X_STAGES * XS_BYTES >= TOK_ * 512, "the staged tile of a split product reuses the ring");
};

template <class Cfg>
__global__ void __launch_bounds__(Cfg::THREADS, 1) int4_tile_kernel(const __grid_constant__ Int4TileParams tp) {
  using H = int4::Half<Cfg::F16>;
  constexpr int TOK = Cfg::TOK, G = Cfg::G, GPS = Cfg::GPS, NMMA = Cfg::NMMA, CPT = Cfg::CPT;
  extern __shared__ uint8_t smem_raw[];
  const Int4Params& p = tp.p;
  const uint32_t raw = ptx::smem_u32(smem_raw);
  const uint32_t pad = (1024u - (raw & 1023u)) & 1023u;
  const uint32_t base = raw + pad;
  uint8_t* const sm = smem_raw + pad;
  auto bar = [&](int i) { return base + Cfg::BAR_OFF + 8u * i; };
  auto xfull = [&](int s) { return bar(s); };
  auto xempty = [&](int s) { return bar(Cfg::X_STAGES + s); };
  auto afull = [&](int b) { return bar(2 * Cfg::X_STAGES + b); };
  auto aempty = [&](int b) { return bar(2 * Cfg::X_STAGES + Cfg::A_BUFS + b); };
  auto dfull = [&](int d) { return bar(2 * Cfg::X_STAGES + 2 * Cfg::A_BUFS + d); };
  auto dempty = [&](int d) { return bar(2 * Cfg::X_STAGES + 2 * Cfg::A_BUFS + 2 + d); };
  constexpr int kBars = 2 * Cfg::X_STAGES + 2 * Cfg::A_BUFS + 4;
  static_assert(8 * kBars + 8 <= Cfg::BAR_BYTES, "barrier block too small");
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(sm + Cfg::BAR_OFF + 8 * kBars);
  volatile uint32_t* abort_word = tmem_slot + 1;
  int32_t* const row_of = reinterpret_cast<int32_t*>(sm + Cfg::TAB_OFF);       // [E + 1] first row of each expert
  int32_t* const tile_of = row_of + kInt4MaxExperts + 1;                       // [E + 1] first tile of rows

  const int warp = ptx::warp_index(), lane = threadIdx.x & 31;
  const int S = p.splits_k;
  const int rank = S > 1 ? static_cast<int>(ptx::cluster_ctarank()) : 0;
  const int steps = p.Kp / 128;
  const int kb0 = static_cast<int>(static_cast<int64_t>(steps) * rank / S);
  const int kb1 = static_cast<int>(static_cast<int64_t>(steps) * (rank + 1) / S);

  if (threadIdx.x == 0) {
    for (int s = 0; s < Cfg::X_STAGES; ++s) {
      ptx::mbar_init(xfull(s), 1);
      ptx::mbar_init(xempty(s), 1);
    }
    for (int b = 0; b < Cfg::A_BUFS; ++b) {
      ptx::mbar_init(afull(b), 4);
      ptx::mbar_init(aempty(b), 1);
    }
    for (int d = 0; d < 2; ++d) {
      ptx::mbar_init(dfull(d), 1);
      ptx::mbar_init(dempty(d), Cfg::HALVES == 2 ? 4 : 8);
    }
    *abort_word = 0;
    ptx::fence_mbar_init();
  }
  if (warp == 12 && lane == 0) ptx::prefetch_tmap(&tp.tm_x);
  if (warp == 13) {
    ptx::tmem_alloc<1>(ptx::smem_u32(const_cast<uint32_t*>(tmem_slot)), 512);
    ptx::tmem_relinquish<1>();
  }
  if (warp == 14) {
    // rows and tiles of the experts; negative counts are none, rows past the input do not exist
    int64_t rows = 0;
    int tiles = 0;
    for (int c = 0; c < p.E; c += 32) {
      const int e = c + lane;
      int64_t n = 0;
      if (e < p.E) n = p.splits == nullptr ? p.M : max(p.splits[e], 0);
      int64_t end = n;
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t v = __shfl_up_sync(0xffffffffu, end, o);
        if (lane >= o) end += v;
      }
      const int64_t r0 = min(rows + end - n, p.M), r1 = min(rows + end, p.M);
      const int t = static_cast<int>((r1 - r0 + TOK - 1) / TOK);
      int te = t;
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, te, o);
        if (lane >= o) te += v;
      }
      if (e < p.E) {
        row_of[e] = static_cast<int32_t>(r0);
        tile_of[e] = tiles + te - t;
      }
      rows += __shfl_sync(0xffffffffu, end, 31);
      tiles += __shfl_sync(0xffffffffu, te, 31);
    }
    if (lane == 0) {
      row_of[p.E] = static_cast<int32_t>(min(rows, p.M));
      tile_of[p.E] = tiles;
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  const WaitCtx wc{tp.status, abort_word, tp.timeout_ns};
  const int items = tile_of[p.E] * p.tiles;
  const int first = blockIdx.x / S, stride = gridDim.x / S;

  struct Item {
    int e, n0, row, last;        // expert, first row of the weights, first row of x, end of the expert's rows
  };
  auto item_of = [&](int item) {
    const int t = item / p.tiles;
    int lo = 0, hi = p.E;        // tile_of[lo] <= t < tile_of[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (tile_of[mid] <= t) lo = mid;
      else hi = mid;
    }
    return Item{lo, (item - t * p.tiles) * 128, row_of[lo] + (t - tile_of[lo]) * TOK, row_of[lo + 1]};
  };

  // eight sums of one row of x, bias added
  auto store8 = [&](float (&v)[8], int64_t row, int n) {
    uint16_t* out = p.out + row * p.ldo + n;
    if (p.bias != nullptr) {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (n + k < p.N) v[k] += ptx::half_bits_to_float(p.bias[n + k], Cfg::F16);
    }
    const uint32_t w[4] = {ptx::pack_half2(Cfg::F16, v[0], v[1]), ptx::pack_half2(Cfg::F16, v[2], v[3]),
                           ptx::pack_half2(Cfg::F16, v[4], v[5]), ptx::pack_half2(Cfg::F16, v[6], v[7])};
    if (tp.out_vec && n + 8 <= p.N) {
      ptx::st_global_v4(out, make_uint4(w[0], w[1], w[2], w[3]));
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (n + k < p.N) out[k] = static_cast<uint16_t>(w[k >> 1] >> (16 * (k & 1)));
    }
  };
  // a wait gave up: let copies and MMAs in flight land before this CTA's shared memory and TMEM go away
  auto drain = [&] {
    __syncwarp();
    if (*abort_word) {
      const uint64_t t0 = ptx::globaltimer_ns();
      while (ptx::globaltimer_ns() - t0 < 200000ull) __nanosleep(2000);
    }
    __syncwarp();
  };

  if (warp < 8) {
    // ------------------------------------------------------------------ sums and epilogue
    if constexpr (TOK == 256) ptx::setmaxnreg_inc<200>();
    const int set = warp >> 2, quad = warp & 3, r = quad * 32 + lane;
    const int groups = p.Kp / G, g0 = kb0 * GPS, ng = (kb1 - kb0) * GPS;
    const int slot = (r / 64) * 64 + int4_scale_slot(r % 64);
    const uint32_t lanes = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    float* const stage = reinterpret_cast<float*>(sm + Cfg::EPI_OFF) + set * (16 * 128);
    uint32_t count = 0;          // groups so far
    bool ok = true;
    uint16_t next[4];
    auto fetch = [&](int item, int j) {          // scales of groups j .. j + 3
      if (item >= items) return;
      const Item it = item_of(item);
      const uint16_t* s = p.scales + (static_cast<int64_t>(it.e) * groups + g0) * p.Np + it.n0 + slot;
#pragma unroll
      for (int i = 0; i < 4; ++i) next[i] = j + i < ng ? s[static_cast<int64_t>(j + i) * p.Np] : static_cast<uint16_t>(0);
    };
    fetch(first, 0);
    for (int item = first; item < items && ok; item += stride) {
      const Item it = item_of(item);
      uint64_t acc[CPT / 2];
#pragma unroll
      for (int i = 0; i < CPT / 2; ++i) acc[i] = 0ull;
      for (int j0 = 0; j0 < ng && ok; j0 += 4) {
        uint16_t now[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) now[i] = next[i];
        if (j0 + 4 < ng) fetch(item, j0 + 4);
        else fetch(item + stride, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (j0 + i >= ng) break;
          const uint32_t d = Cfg::HALVES == 2 ? static_cast<uint32_t>(set) : count & 1u;
          const uint32_t phase = Cfg::HALVES == 2 ? count & 1u : count >> 1 & 1u;
          ++count;
          const float f = ptx::half_bits_to_float(now[i], p.scale_f16);
          const uint64_t ff = ptx::pack_f32x2(f, f);
          if (!mbar_wait_warp(wc, dfull(d), phase, kSiteTmemFull)) {
            ok = false;
            break;
          }
          ptx::tc_fence_after();
          const uint32_t at = lanes + (Cfg::HALVES == 2 ? set * NMMA : d * NMMA + set * CPT);
          constexpr int W = CPT == 128 || CPT < 32 ? 16 : 32;  // (128 sums leave room for 16 more registers)
#pragma unroll
          for (int c = 0; c < CPT; c += W) {
            uint32_t v[W];
            if constexpr (W == 32) ptx::tmem_ld_32x32b_x32(at + c, v);
            else ptx::tmem_ld_32x32b_x16(at + c, v);
            ptx::tmem_ld_wait();
            if (c + W == CPT) {
              ptx::tc_fence_before();
              __syncwarp();
              if (lane == 0) ptx::mbar_arrive_relaxed(dempty(d));
            }
#pragma unroll
            for (int k = 0; k < W / 2; ++k)
              acc[c / 2 + k] = ptx::ffma2(ptx::pack_b32x2(v[2 * k], v[2 * k + 1]), ff, acc[c / 2 + k]);
          }
        }
      }
      if (!ok) break;
      if (S > 1) {
        // (everything in the ring has been multiplied: the whole tile goes there, one row of x after the other)
        float* tile = reinterpret_cast<float*>(sm + Cfg::X_OFF);
#pragma unroll
        for (int c = 0; c < CPT / 2; ++c) {
          tile[(set * CPT + 2 * c) * 128 + r] = __uint_as_float(static_cast<uint32_t>(acc[c]));
          tile[(set * CPT + 2 * c + 1) * 128 + r] = __uint_as_float(static_cast<uint32_t>(acc[c] >> 32));
        }
        continue;
      }
      const int live = it.last - it.row - set * CPT;       // rows of x that this half holds
#pragma unroll
      for (int c0 = 0; c0 < CPT; c0 += 16) {
        if (c0 >= live) break;
#pragma unroll
        for (int c = 0; c < 16; c += 2) {
          stage[c * 128 + r] = __uint_as_float(static_cast<uint32_t>(acc[(c0 + c) / 2]));
          stage[(c + 1) * 128 + r] = __uint_as_float(static_cast<uint32_t>(acc[(c0 + c) / 2] >> 32));
        }
        asm volatile("bar.sync %0, 128;" ::"r"(1 + set) : "memory");
        for (int u = quad * 32 + lane; u < 256; u += 128) {
          const int m = u / 16, n = it.n0 + u % 16 * 8;
          if (c0 + m >= live || n >= p.N) continue;
          const float4 a = *reinterpret_cast<const float4*>(stage + m * 128 + u % 16 * 8);
          const float4 b = *reinterpret_cast<const float4*>(stage + m * 128 + u % 16 * 8 + 4);
          float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
          store8(v, static_cast<int64_t>(it.row) + set * CPT + c0 + m, n);
        }
        asm volatile("bar.sync %0, 128;" ::"r"(1 + set) : "memory");
      }
    }
    ptx::tc_fence_before();
    drain();
    if (S > 1) {
      // one tile per cluster: its sums, eight columns of one row of x at a time, dealt out over the CTAs, ranks in order
      ptx::cluster_sync();
      if (first < items) {
        const Item it = item_of(first);
        const int live = min(TOK, it.last - it.row);
        for (int u = rank * 256 + static_cast<int>(threadIdx.x); u < live * 16; u += S * 256) {
          const int m = u / 16, n = it.n0 + u % 16 * 8;
          if (n >= p.N) continue;
          const uint32_t at = base + Cfg::X_OFF + (m * 128 + u % 16 * 8) * 4;
          float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
          for (int c = 0; c < S; ++c) {
            const uint32_t from = ptx::mapa_u32(at, c);
            const uint4 a = ptx::ld_cluster_v4(from), b = ptx::ld_cluster_v4(from + 16);
            v[0] += __uint_as_float(a.x), v[1] += __uint_as_float(a.y);
            v[2] += __uint_as_float(a.z), v[3] += __uint_as_float(a.w);
            v[4] += __uint_as_float(b.x), v[5] += __uint_as_float(b.y);
            v[6] += __uint_as_float(b.z), v[7] += __uint_as_float(b.w);
          }
          store8(v, static_cast<int64_t>(it.row) + m, n);
        }
      }
      __syncwarp();
      ptx::cluster_sync();                       // the others may still be reading this CTA's sums
    } else {
      __syncthreads();
    }
  } else if (warp < 12) {
    // ------------------------------------------------------------------ weights
    if constexpr (TOK == 256) ptx::setmaxnreg_dec<72>();
    const int q = warp - 8, g = lane >> 2;
    const int64_t units = p.Kp / 64;
    const int groups = p.Kp / G;
    const uint32_t wring = base + Cfg::W_OFF + (q * 4 * 32 + lane) * 16;       // [PF][warp][4][lane]
    const uint32_t zring = base + Cfg::Z_OFF + (q * GPS * 32 + lane) * 4;      // [PF][warp][GPS][lane]
    int fetch_item = first, fetch_kb = kb0;
    const uint4* wsrc = nullptr;
    const uint8_t* zsrc = nullptr;
    auto aim = [&] {
      if (fetch_item >= items) return;
      const Item it = item_of(fetch_item);
      wsrc = p.packed + ((static_cast<int64_t>(it.e) * (p.Np / 16) + it.n0 / 16 + 2 * q) * units) * 32 + lane;
      if (p.zeros != nullptr)
        zsrc = p.zeros + static_cast<int64_t>(it.e) * groups * p.Np + it.n0 + (q / 2) * 64 + g * 8 + (q % 2) * 4;
    };
    auto fetch = [&](int slot) {                 // the next block, if there is one, into a slot of the ring
      if (fetch_item < items) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          ptx::cp_async_16(wring + slot * 8192 + i * 512, wsrc + ((i >> 1) * units + fetch_kb * 2 + (i & 1)) * 32, 16);
        if (p.zeros != nullptr) {
#pragma unroll
          for (int j = 0; j < GPS; ++j)
            ptx::cp_async_4(zring + slot * (GPS * 512) + j * 128, zsrc + (static_cast<int64_t>(fetch_kb) * GPS + j) * p.Np);
        }
        if (++fetch_kb == kb1) {
          fetch_kb = kb0;
          fetch_item += stride;
          aim();
        }
      }
      ptx::cp_async_commit();
    };
    aim();
    for (int s = 0; s < Cfg::PF; ++s) fetch(s);
    int slot = 0;
    uint32_t count = 0;
    bool ok = true;
    for (int item = first; item < items && ok; item += stride) {
      for (int kb = kb0; kb < kb1; ++kb, ++count) {
        ptx::cp_async_wait<Cfg::PF - 1>();
        const uint32_t buf = count % Cfg::A_BUFS;
        if (!mbar_wait_warp(wc, aempty(buf), (count / Cfg::A_BUFS & 1u) ^ 1u, kSiteTmemEmpty)) {
          ok = false;
          break;
        }
        ptx::tc_fence_after();
        uint32_t zz[GPS];
#pragma unroll
        for (int j = 0; j < GPS; ++j) {
          zz[j] = 0x08080808u;
          if (p.zeros != nullptr)
            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(zz[j]) : "r"(zring + slot * (GPS * 512) + j * 128));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {            // row block i / 2 of the warp's two, 64 columns i % 2
          uint32_t w[4];
          asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                       : "r"(wring + slot * 8192 + i * 512));
          uint32_t a[16];
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            const uint32_t z = zz[((i & 1) * 64 + s * 16) / G] >> (i >> 1) * 16;
            const uint32_t z0 = H::kMagic + (z & 0xffu) * 0x00010001u;
            const uint32_t z1 = H::kMagic + (z >> 8 & 0xffu) * 0x00010001u;
            a[4 * s] = H::sub((w[s] & 0x000f000fu) | H::kMagic, z0);
            a[4 * s + 1] = H::sub((w[s] >> 4 & 0x000f000fu) | H::kMagic, z0);
            a[4 * s + 2] = H::sub((w[s] >> 8 & 0x000f000fu) | H::kMagic, z1);
            a[4 * s + 3] = H::sub((w[s] >> 12 & 0x000f000fu) | H::kMagic, z1);
          }
          ptx::tmem_st_16x256b_x4(tmem + (static_cast<uint32_t>(q * 32 + (i >> 1) * 16) << 16) + Cfg::A_COL + buf * 64 + (i & 1) * 32,
                                  a);
        }
        ptx::tmem_st_wait();
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(afull(buf));
        fetch(slot);
        slot = slot + 1 == Cfg::PF ? 0 : slot + 1;
      }
    }
    ptx::cp_async_wait<0>();
    drain();
    if (S > 1) ptx::cluster_sync();
    else __syncthreads();
    if (S > 1) ptx::cluster_sync();
  } else {
    if constexpr (TOK == 256) ptx::setmaxnreg_dec<40>();
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    if (warp == 12) {
      // ------------------------------------------------------------------ x
      for (int item = first; item < items && ok; item += stride) {
        const Item it = item_of(item);
        for (int u = 2 * kb0; u < 2 * kb1; ++u) {
          if (!mbar_wait_warp(wc, xempty(stage), phase ^ 1u, kSiteSmemEmpty)) {
            ok = false;
            break;
          }
          if (ptx::elect_one()) {
            ptx::mbar_arrive_expect_tx(xfull(stage), Cfg::XS_BYTES);
            ptx::tma_load_2d(base + Cfg::X_OFF + stage * Cfg::XS_BYTES, &tp.tm_x, xfull(stage), u * 64, it.row);
          }
          __syncwarp();
          if (++stage == Cfg::X_STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
    } else if (warp == 13) {
      // ------------------------------------------------------------------ MMA
      constexpr uint32_t kFmt = Cfg::F16 ? 0u : 1u;
      const uint32_t idesc = ptx::umma_idesc(kFmt, kFmt, 128, NMMA);
      constexpr int SPG = G / 16;                  // MMAs of one group
      uint32_t blocks = 0, count = 0;              // (stage: that of the block's first 64 columns)
      for (int item = first; item < items && ok; item += stride) {
        for (int kb = kb0; kb < kb1 && ok; ++kb, ++blocks) {
          const uint32_t buf = blocks % Cfg::A_BUFS;
          if (!mbar_wait_warp(wc, afull(buf), blocks / Cfg::A_BUFS & 1u, kSiteSmemFull)) {
            ok = false;
            break;
          }
          const int stage1 = stage + 1 == Cfg::X_STAGES ? 0 : stage + 1;
          const uint32_t phase1 = stage1 == 0 ? phase ^ 1u : phase;
#pragma unroll
          for (int j = 0; j < GPS; ++j, ++count) {
            if (j == 0 && !mbar_wait_warp(wc, xfull(stage), phase, kSiteSmemFull)) ok = false;
            if ((j + 1) * G > 64 && j * G <= 64 && !mbar_wait_warp(wc, xfull(stage1), phase1, kSiteSmemFull)) ok = false;
            if (!ok) break;
#pragma unroll
            for (int h = 0; h < Cfg::HALVES; ++h) {
              const uint32_t d = Cfg::HALVES == 2 ? static_cast<uint32_t>(h) : count & 1u;
              const uint32_t use = Cfg::HALVES == 2 ? count : count >> 1;
              if (!mbar_wait_warp(wc, dempty(d), (use & 1u) ^ 1u, kSiteTmemEmpty)) {
                ok = false;
                break;
              }
              ptx::tc_fence_after();
              if (ptx::elect_one()) {
#pragma unroll
                for (int s = j * SPG; s < (j + 1) * SPG; ++s) {
                  const uint32_t xs = base + Cfg::X_OFF + (s < 4 ? stage : stage1) * Cfg::XS_BYTES + h * NMMA * 128;
                  ptx::umma_ts_f16(tmem + d * NMMA, tmem + Cfg::A_COL + buf * 64 + s * 8,
                                   ptx::umma_desc_k_sw128(xs) + 2u * (s % 4), idesc, s != j * SPG ? 1u : 0u);
                }
                ptx::umma_commit(dfull(d));
                if (h == Cfg::HALVES - 1) {
                  if (j * G < 64 && (j + 1) * G >= 64) ptx::umma_commit(xempty(stage));
                  if (j == GPS - 1) {
                    ptx::umma_commit(xempty(stage1));
                    ptx::umma_commit(aempty(buf));
                  }
                }
              }
              __syncwarp();
            }
            if (!ok) break;
          }
          stage = stage1 + 1 == Cfg::X_STAGES ? 0 : stage1 + 1;
          phase = stage == 0 ? phase1 ^ 1u : phase1;
        }
      }
    }
    drain();
    if (S > 1) ptx::cluster_sync();
    else __syncthreads();
    if (warp == 13) {
      ptx::tc_fence_after();
      ptx::tmem_dealloc<1>(tmem, 512);
    }
    __syncwarp();
    if (S > 1) ptx::cluster_sync();
  }
}

}  // namespace fluxb
