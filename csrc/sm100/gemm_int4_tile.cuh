// Products with 4-bit weights for more than a few rows: the weights' integers go through TMEM.
//
// A tile is 128 rows of the weights (the M of the MMA) times TOK rows of x (its N). Four warps unpack the weights of the
// next 128 columns of k and store them into TMEM, where the MMA reads its A operand: the 32 KB of 16-bit integers never pass
// through shared memory, whose bandwidth (128 bytes a cycle for writing and reading both) would bound the kernel at half the
// speed at which memory delivers the packed weights. x tiles arrive by TMA as the B operand.
// Every group's product lands in a fresh accumulator; eight warps multiply it with the group's scale (a thread owns one row
// of the weights, so that is one number) and add it to their fp32 sums in registers. With TOK = 256 the tile is two
// halves of 128 columns that take turns at two or three accumulators, and one unpacked weight serves 256 rows. Smaller TOK have
// two to four accumulators for consecutive groups.
//
//   warps 0 .. 7    sums: TMEM lanes 32 (warp % 4), the first or second half of the columns (warp / 4); epilogue
//                   (TOK = 32: warps 0 .. 3)
//   the next 4 (8)  unpack the weights into TMEM
//   the next three  loads of x and scales, MMA issue, loads of packed weights and zero points
// One CTA per SM (two with TOK = 32) walks the tiles of all experts; the loads of a tile run ahead into the one before. With
// splits_k > 1 a cluster shares one tile, each CTA with its part of k, and the sums meet in distributed shared memory in rank
// order.
//
// Measured (kernels alone, weights from DRAM):
//   TOK = 32    512 rows over 64 experts, 4096 x 4096, groups of 128: 132 us, 4.3 TB/s of 564 MB; unpacking is the bound (ALU 59 %,
//               issue slots 72 % busy; without it, its stores included, 91 us)
//   TOK = 64    45 x 5003 x 4128, groups of 32, zero points, clusters of three: 15.6 us, a third of it start and end
//   TOK = 256   2048 x 12288 x 4096, groups of 128: 165 us, 1.25 PFLOP/s, tensor pipe 58 % busy. 6 rounds of tiles where 5.2
//               would do, epilogues 10 us; no other part alone is the bound: without the sums, the unpacking or the loads of x
//               160 us, with one MMA in eight 134. Groups of 64 take 220 us, of 32 410: a hand-over costs about 500 cycles.
//               9216 rows over 32 experts, 4096 x 2048, groups of 64: 215 us, 719 TFLOP/s; without epilogues 24 less, without
//               sums 35, without unpacking 23
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
template <int I>
struct IntC {
  static constexpr int value = I;
};

template <int TOK_, int G_, bool F16_>
struct Int4TileCfg {
  static constexpr int TOK = TOK_, G = G_;
  static constexpr bool F16 = F16_;
  static constexpr int HALVES = TOK_ == 256 ? 2 : 1;
  static constexpr int NMMA = TOK_ / HALVES;
  static constexpr int GPS = 128 / G_;                   // groups per block of 128 columns of k
  // The smallest tiles wait for weights, and what a CTA does once per block (waits, issue) would hold them up: two CTAs share
  // an SM. With TOK = 64, which needs the shared memory, two sets of warps unpack instead.
  static constexpr int CTAS = TOK_ == 32 ? 2 : 1;
  static constexpr int SUM_WARPS = CTAS == 2 ? 4 : 8, SETS = SUM_WARPS / 4, UNPACK_SETS = TOK_ <= 64 ? 2 : 1;
  static constexpr int UNPACK_WARP0 = SUM_WARPS, X_WARP = SUM_WARPS + 4 * UNPACK_SETS, MMA_WARP = X_WARP + 1,
                       W_WARP = X_WARP + 2, TABLE_WARP = X_WARP + 3;
  static constexpr int THREADS = 32 * (X_WARP + 4);
  static constexpr int CPD = NMMA / SETS;                // columns of an accumulator that a thread reads
  static constexpr int CPT = CPD * HALVES;               // columns that it sums
  // TMEM: accumulators in the first half of the CTA's columns, blocks of weights in the second; with TOK = 256 and small
  // groups three accumulators and two blocks: an accumulator comes round after about 850 cycles, a group of 64 columns
  // multiplies in 260 (9216 rows over 32 experts, groups of 64: 229 us with two, 217 with three; 2048 x 12288 x 4096, groups
  // of 128: 166 and 169)
  static constexpr int TMEM_COLS = 512 / CTAS, A_COL = TOK_ == 256 && G_ < 128 ? 384 : TMEM_COLS / 2,
                       A_BUFS = (TMEM_COLS - A_COL) / 64, D_BUFS = A_COL / NMMA;
  // x arrives in blocks of 128 columns, with TOK = 256 in halves of a block (shared memory holds two and a half of them)
  static constexpr int XS_PER_BLOCK = TOK_ == 256 ? 2 : 1;
  static constexpr int XS_BYTES = TOK_ * 256 / XS_PER_BLOCK;
  static constexpr int X_STAGES = TOK_ == 256 ? 5 : TOK_ == 64 ? 8 : 4;
  // One commit per group or block hands its product over; the last one of a block also frees its weights and its x. The
  // barriers are a ring of RING blocks. (TOK = 256: one per accumulator, and commits of their own for x and weights.)
  static constexpr int RING = TOK_ == 256 ? 1 : X_STAGES;
  // Groups that are handed over at once: those of a block where the accumulators hold two blocks, else one. (HALVES == 2:
  // one half of one group.) A wait that finds its phase complete still costs a warp about 110 cycles.
  static constexpr int GRAN = HALVES == 1 && D_BUFS >= 2 * GPS ? GPS : 1;
  static constexpr int HPB = GPS / GRAN;                 // hand-overs per block (and half)
  static constexpr int UNITS = D_BUFS / GRAN;
  static constexpr int D_BARS = TOK_ == 256 ? UNITS : RING * HPB;
  static constexpr int SC_SLOTS = TOK_ == 256 ? 8 : RING + (D_BUFS + GPS - 1) / GPS;  // blocks of scales, see the x warp
  static constexpr int SC_BYTES = GPS * 256;
  static constexpr int W_STAGES = TOK_ == 64 ? 6 : TOK_ == 256 ? 3 : 4;        // blocks of packed weights and zero points
  static constexpr int W_BYTES = 8192, Z_BYTES = GPS * 128;
  static constexpr int EPI_PITCH = 40;                   // 16-bit values; a warp stages 16 rows of the output at a time
  static constexpr int EPI_BYTES = SUM_WARPS * 16 * EPI_PITCH * 2;
  static constexpr int TAB_BYTES = (2 * (kInt4MaxExperts + 1) * 4 + 15) / 16 * 16;
  static constexpr int BAR_BYTES = 640;
  static constexpr int X_OFF = 0, SC_OFF = X_STAGES * XS_BYTES, W_OFF = SC_OFF + SC_SLOTS * SC_BYTES,
                       Z_OFF = W_OFF + W_STAGES * W_BYTES, TAB_OFF = Z_OFF + W_STAGES * Z_BYTES,
                       BAR_OFF = TAB_OFF + TAB_BYTES, END = BAR_OFF + BAR_BYTES;
  static constexpr int EPI_OFF = END;
  static constexpr int SMEM_BYTES = EPI_OFF + EPI_BYTES + 1024;
  static_assert(CTAS * (SMEM_BYTES + 1024) <= 228 * 1024, "shared memory");
  static_assert(X_STAGES * XS_BYTES >= TOK_ * 512, "the staged tile of a split product reuses the ring");
};

template <class Cfg>
__global__ void __launch_bounds__(Cfg::THREADS, Cfg::CTAS) int4_tile_kernel(const __grid_constant__ Int4TileParams tp) {
  constexpr int TOK = Cfg::TOK, G = Cfg::G, GPS = Cfg::GPS, GRAN = Cfg::GRAN, HPB = Cfg::HPB;
  constexpr int NMMA = Cfg::NMMA, CPD = Cfg::CPD, CPT = Cfg::CPT;
  extern __shared__ uint8_t smem_raw[];
  const Int4Params& p = tp.p;
  const uint32_t raw = ptx::smem_u32(smem_raw);
  const uint32_t pad = (1024u - (raw & 1023u)) & 1023u;
  const uint32_t base = raw + pad;
  uint8_t* const sm = smem_raw + pad;
  auto bar = [&](int i) { return base + Cfg::BAR_OFF + 8u * i; };
  auto xfull = [&](int s) { return bar(s); };
  auto xempty = [&](int s) { return bar(Cfg::X_STAGES + s); };                 // (TOK = 256)
  auto afull = [&](int b) { return bar(2 * Cfg::X_STAGES + b); };
  auto aempty = [&](int b) { return bar(2 * Cfg::X_STAGES + Cfg::A_BUFS + b); };       // (TOK = 256)
  auto dempty = [&](int d) { return bar(2 * Cfg::X_STAGES + 2 * Cfg::A_BUFS + d); };
  auto dfull = [&](int d) { return bar(2 * Cfg::X_STAGES + 2 * Cfg::A_BUFS + Cfg::UNITS + d); };
  constexpr int kWBar = 2 * Cfg::X_STAGES + 2 * Cfg::A_BUFS + Cfg::UNITS + Cfg::D_BARS;
  auto wfull = [&](int s) { return bar(kWBar + s); };
  auto wempty = [&](int s) { return bar(kWBar + Cfg::W_STAGES + s); };
  constexpr int kBars = kWBar + 2 * Cfg::W_STAGES;
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
    for (int s = 0; s < Cfg::W_STAGES; ++s) {
      ptx::mbar_init(wfull(s), 1);
      ptx::mbar_init(wempty(s), 4);
    }
    for (int d = 0; d < Cfg::UNITS; ++d) ptx::mbar_init(dempty(d), Cfg::SUM_WARPS);
    for (int d = 0; d < Cfg::D_BARS; ++d) ptx::mbar_init(dfull(d), 1);
    *abort_word = 0;
    ptx::fence_mbar_init();
  }
  if (warp == Cfg::X_WARP && lane == 0) ptx::prefetch_tmap(&tp.tm_x);
  if (warp == Cfg::MMA_WARP) {
    ptx::tmem_alloc<1>(ptx::smem_u32(const_cast<uint32_t*>(tmem_slot)), Cfg::TMEM_COLS);
    ptx::tmem_relinquish<1>();
  }
  if (warp == Cfg::TABLE_WARP) {
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
  const int items = __shfl_sync(0xffffffffu, tile_of[p.E], 0) * p.tiles;    // (known to be the same in all lanes)
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

  if (warp < Cfg::SUM_WARPS) {
    // ------------------------------------------------------------------ sums and epilogue
    if constexpr (TOK == 256) ptx::setmaxnreg_inc<200>();
    const int set = warp >> 2, quad = warp & 3, r = quad * 32 + lane;
    const int slot = (r / 64) * 64 + int4_scale_slot(r % 64);
    const uint32_t lanes = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    uint16_t* const stage = reinterpret_cast<uint16_t*>(sm + Cfg::EPI_OFF) + warp * (16 * Cfg::EPI_PITCH);
    const uint16_t* const scales = reinterpret_cast<const uint16_t*>(sm + Cfg::SC_OFF) + slot;
    uint32_t blocks = 0, turn = 0, lap = 0;
    bool ok = true;
    for (int item = first; item < items && ok; item += stride) {
      const Item it = item_of(item);
      uint64_t acc[CPT / 2];
#pragma unroll
      for (int i = 0; i < CPT / 2; ++i) acc[i] = 0ull;
      const bool both = it.last - it.row > NMMA;           // (TOK = 256) the second half has rows
      for (int kb = kb0; kb < kb1 && ok; ++kb, ++blocks) {
#pragma unroll
        for (int j = 0; j < GPS; ++j) {
          float f = 0.f;
#pragma unroll
          for (int h = 0; h < Cfg::HALVES; ++h) {
            if (h == 1 && !both) break;
            const uint32_t count = blocks * HPB + j / GRAN;      // of hand-overs (TOK = 256: `turn` and `lap` tell)
            const uint32_t unit = Cfg::HALVES == 2 ? turn : count % Cfg::UNITS;
            const uint32_t d = unit * GRAN + j % GRAN;
            if (j % GRAN == 0) {
              const uint32_t full = Cfg::HALVES == 2 ? turn : count % Cfg::D_BARS;
              const uint32_t phase = (Cfg::HALVES == 2 ? lap : count / Cfg::D_BARS) & 1u;
              if (!mbar_wait_all_warp(wc, MbarPhase{dfull(full), phase, kSiteTmemFull})) {
                ok = false;
                break;
              }
              ptx::tc_fence_after();
            }
            if (h == 0)
              f = ptx::half_bits_to_float(scales[(blocks % Cfg::SC_SLOTS) * (Cfg::SC_BYTES / 2) + j * 128], p.scale_f16);
            const uint64_t ff = ptx::pack_f32x2(f, f);
            const uint32_t at = lanes + d * NMMA + set * CPD;
            constexpr int W = Cfg::CTAS == 2 ? 16 : 32;      // columns at a time, as registers allow
#pragma unroll
            for (int c = 0; c < CPD; c += W) {
              uint32_t v[W];
              if constexpr (W == 32) ptx::tmem_ld_32x32b_x32(at + c, v);
              else ptx::tmem_ld_32x32b_x16(at + c, v);
              ptx::tmem_ld_wait(v);
              if (c + W == CPD && j % GRAN == GRAN - 1) {
                ptx::tc_fence_before();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(dempty(unit));
              }
#pragma unroll
              for (int k = 0; k < W / 2; ++k)
                acc[(h * CPD + c) / 2 + k] =
                    ptx::ffma2(ptx::pack_b32x2(v[2 * k], v[2 * k + 1]), ff, acc[(h * CPD + c) / 2 + k]);
            }
            if (Cfg::HALVES == 2 && ++turn == Cfg::UNITS) {
              turn = 0;
              ++lap;
            }
          }
          if (!ok) break;
        }
      }
      if (!ok) break;
      if (S > 1) {
        // (everything in the ring has been multiplied: the whole tile goes there, one row of x after the other)
        float* tile = reinterpret_cast<float*>(sm + Cfg::X_OFF);
#pragma unroll
        for (int c = 0; c < CPT / 2; ++c) {
          const int m = c * 2 / CPD * NMMA + set * CPD + c * 2 % CPD;
          tile[m * 128 + r] = __uint_as_float(static_cast<uint32_t>(acc[c]));
          tile[(m + 1) * 128 + r] = __uint_as_float(static_cast<uint32_t>(acc[c] >> 32));
        }
        continue;
      }
      // 16 rows of x by this warp's 32 rows of the weights, turned around in shared memory (nobody waits for other warps)
      const float bias = p.bias != nullptr && it.n0 + r < p.N ? ptx::half_bits_to_float(p.bias[it.n0 + r], Cfg::F16) : 0.f;
#pragma unroll
      for (int c0 = 0; c0 < CPT; c0 += 16) {
        const int m0 = c0 / CPD * NMMA + set * CPD + c0 % CPD;
        const int live = it.last - it.row - m0;
        if (live <= 0) break;
#pragma unroll
        for (int c = 0; c < 16; c += 2) {
          const uint64_t two = acc[(c0 + c) / 2];
          const uint32_t w = ptx::pack_half2(Cfg::F16, __uint_as_float(static_cast<uint32_t>(two)) + bias,
                                             __uint_as_float(static_cast<uint32_t>(two >> 32)) + bias);
          stage[c * Cfg::EPI_PITCH + lane] = static_cast<uint16_t>(w);
          stage[(c + 1) * Cfg::EPI_PITCH + lane] = static_cast<uint16_t>(w >> 16);
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int m = i * 8 + lane / 4, n = it.n0 + quad * 32 + lane % 4 * 8;
          if (m < live && n < p.N) {
            const uint4 o = *reinterpret_cast<const uint4*>(stage + m * Cfg::EPI_PITCH + lane % 4 * 8);
            uint16_t* const out = p.out + (static_cast<int64_t>(it.row) + m0 + m) * p.ldo + n;
            if (tp.out_vec && n + 8 <= p.N) {
              ptx::st_global_v4(out, o);
            } else {
              const uint32_t w[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
              for (int k = 0; k < 8; ++k)
                if (n + k < p.N) out[k] = static_cast<uint16_t>(w[k >> 1] >> (16 * (k & 1)));
            }
          }
        }
        __syncwarp();
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
        for (int u = rank * (Cfg::SUM_WARPS * 32) + static_cast<int>(threadIdx.x); u < live * 16;
             u += S * (Cfg::SUM_WARPS * 32)) {
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
  } else if (warp < Cfg::X_WARP) {
    // ------------------------------------------------------------------ weights
    if constexpr (TOK == 256) ptx::setmaxnreg_dec<72>();
    const int q = (warp - Cfg::UNPACK_WARP0) & 3, turn = (warp - Cfg::UNPACK_WARP0) >> 2;    // blocks turn, turn + sets, ...
    const uint32_t wring = base + Cfg::W_OFF + (q * 4 * 32 + lane) * 16;
    const uint32_t zring = base + Cfg::Z_OFF + (q / 2) * 64 + (lane >> 2) * 8 + (q % 2) * 4;
    const bool zeros = p.zeros != nullptr;
    const uint32_t total = first < items ? static_cast<uint32_t>((items - 1 - first) / stride + 1) * (kb1 - kb0) : 0u;
    // 16 rows by 64 columns at a time: unpacked while the stores of those before are on their way to TMEM; a block's stores are
    // waited for, and published, at its end.
    bool ok = true;
    auto publish = [&](uint32_t buf) {
      ptx::tmem_st_wait();
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(afull(buf));
    };
    uint32_t slot = turn, wphase = 0;
    for (uint32_t count = turn; count < total; count += Cfg::UNPACK_SETS) {
      const uint32_t buf = count % Cfg::A_BUFS;
      // the packed block is here, and what was multiplied from its place in TMEM is done
      const uint32_t before = count - Cfg::A_BUFS;
      const uint32_t done = Cfg::HALVES == 2 ? aempty(buf) : dfull(before % Cfg::RING * HPB + HPB - 1);
      const uint32_t dphase = (Cfg::HALVES == 2 ? before / Cfg::A_BUFS : before / Cfg::RING) & 1u;
      if (!mbar_wait_all_warp(wc, MbarPhase{wfull(slot), wphase, kSiteSmemFull})) break;
#pragma unroll
      for (int i = 0; i < 4; ++i) {                          // row block i % 2 of the warp's two, 64 columns i / 2
        constexpr int GPH = G < 64 ? 64 / G : 1;             // groups of 64 columns
        const int u = i / 2;
        uint32_t w[4], zz[GPH], a[16];
        ptx::ld_shared(wring + slot * Cfg::W_BYTES + (2 * (i % 2) + u) * 512, w);
#pragma unroll
        for (int j = 0; j < GPH; ++j) {
          zz[j] = 0x08080808u;
          if (zeros)
            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(zz[j]) : "r"(zring + slot * Cfg::Z_BYTES + (u * 64 / G + j) * 128));
        }
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          const uint32_t z = zz[s * 16 / G % GPH];
          const uint32_t z0 = i % 2 == 0 ? int4::magic_zero<Cfg::F16, 0>(z) : int4::magic_zero<Cfg::F16, 2>(z);
          const uint32_t z1 = i % 2 == 0 ? int4::magic_zero<Cfg::F16, 1>(z) : int4::magic_zero<Cfg::F16, 3>(z);
          int4::unpack<Cfg::F16>(w[s], z0, z1, a[4 * s], a[4 * s + 1], a[4 * s + 2], a[4 * s + 3]);
        }
        if (i == 0) {
          // (the block that was here before has been multiplied)
          if (count >= Cfg::A_BUFS && !mbar_wait_all_warp(wc, MbarPhase{done, dphase, kSiteTmemEmpty})) {
            ok = false;
            break;
          }
          ptx::tc_fence_after();
        }
        ptx::tmem_st_16x256b_x4(
            tmem + (static_cast<uint32_t>(q * 32 + (i % 2) * 16) << 16) + Cfg::A_COL + buf * 64 + u * 32, a);
      }
      if (!ok) break;
      if (lane == 0) ptx::mbar_arrive(wempty(slot));       // (the words have been read: they are in the stores)
      publish(buf);
      slot += Cfg::UNPACK_SETS;
      if (slot >= Cfg::W_STAGES) {
        slot -= Cfg::W_STAGES;
        wphase ^= 1u;
      }
    }
    drain();
    if (S > 1) ptx::cluster_sync();
    else __syncthreads();
    if (S > 1) ptx::cluster_sync();
  } else {
    if constexpr (TOK == 256) ptx::setmaxnreg_dec<40>();
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    if (warp == Cfg::X_WARP) {
      // ------------------------------------------------------------------ x
      // Scales come along with x. They are read when the product is done, by when the stage of x may be in use again: their
      // ring is longer. Block b is loaded when block b - RING has been multiplied, for which the groups D_BUFS before its
      // last one had to be summed, and that many more blocks have slots of their own. (TOK = 256: x runs less than three
      // blocks ahead, sums one behind.)
      constexpr int PER = Cfg::XS_PER_BLOCK;
      const int groups = p.Kp / G;
      uint32_t blocks = 0;
      for (int item = first; item < items && ok; item += stride) {
        const Item it = item_of(item);
        const uint16_t* const scales = p.scales + static_cast<int64_t>(it.e) * groups * p.Np + it.n0;
        for (int u = PER * kb0; u < PER * kb1; ++u) {
          const uint32_t empty = Cfg::HALVES == 2 ? xempty(stage) : dfull(stage * HPB + HPB - 1);
          if (!mbar_wait_warp(wc, empty, phase ^ 1u, kSiteSmemEmpty)) {
            ok = false;
            break;
          }
          if (ptx::elect_one()) {
            const uint32_t to = base + Cfg::X_OFF + stage * Cfg::XS_BYTES;
            const bool block = PER == 1 || u % 2 == 0;       // (the first part of a block)
            ptx::mbar_arrive_expect_tx(xfull(stage), Cfg::XS_BYTES + (block ? Cfg::SC_BYTES : 0));
            ptx::tma_load_2d(to, &tp.tm_x, xfull(stage), u * (128 / PER), it.row);
            if (PER == 1) ptx::tma_load_2d(to + Cfg::XS_BYTES / 2, &tp.tm_x, xfull(stage), u * 128 + 64, it.row);
            if (block) {
#pragma unroll
              for (int j = 0; j < GPS; ++j)
                ptx::bulk_load(base + Cfg::SC_OFF + (blocks % Cfg::SC_SLOTS) * Cfg::SC_BYTES + j * 256,
                               scales + (static_cast<int64_t>(u / PER) * GPS + j) * p.Np, 256, xfull(stage));
            }
          }
          __syncwarp();
          if (PER == 1 || u % 2 == 1) ++blocks;
          if (++stage == Cfg::X_STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
    } else if (warp == Cfg::W_WARP) {
      // ------------------------------------------------------------------ packed weights
      const int groups = p.Kp / G;
      for (int item = first; item < items && ok; item += stride) {
        const Item it = item_of(item);
        const uint8_t* const from = reinterpret_cast<const uint8_t*>(p.packed) +
                                    (static_cast<int64_t>(it.e) * (p.Np / 128) + it.n0 / 128) * steps * Cfg::W_BYTES;
        const uint8_t* const zfrom = p.zeros + static_cast<int64_t>(it.e) * groups * p.Np + it.n0;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait_all_warp(wc, MbarPhase{wempty(stage), phase ^ 1u, kSiteSmemEmpty})) {
            ok = false;
            break;
          }
          if (ptx::elect_one()) {
            ptx::mbar_arrive_expect_tx(wfull(stage), Cfg::W_BYTES + (p.zeros != nullptr ? Cfg::Z_BYTES : 0));
            ptx::bulk_load(base + Cfg::W_OFF + stage * Cfg::W_BYTES, from + static_cast<int64_t>(kb) * Cfg::W_BYTES, Cfg::W_BYTES,
                           wfull(stage));
            if (p.zeros != nullptr) {
#pragma unroll
              for (int j = 0; j < GPS; ++j)
                ptx::bulk_load(base + Cfg::Z_OFF + stage * Cfg::Z_BYTES + j * 128,
                               zfrom + (static_cast<int64_t>(kb) * GPS + j) * p.Np, 128, wfull(stage));
            }
          }
          __syncwarp();
          if (++stage == Cfg::W_STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
    } else if (warp == Cfg::MMA_WARP) {
      // ------------------------------------------------------------------ MMA
      constexpr uint32_t kFmt = Cfg::F16 ? 0u : 1u;
      const uint32_t idesc = ptx::umma_idesc(kFmt, kFmt, 128, NMMA);
      constexpr int SPG = G / 16;                  // MMAs of one group
      uint32_t blocks = 0;
      if constexpr (Cfg::HALVES == 1) {
        // One block, B of the ring. All operands of the MMAs are constants beside two uniform base addresses: with addresses
        // computed from a running index, each MMA of 32 columns took 49 cycles to issue (16 to execute).
        auto multiply = [&](auto b_index) {
          constexpr int B = decltype(b_index)::value;
          const uint32_t x0 = ptx::umma_desc_k_sw128_lo(base + Cfg::X_OFF + B * Cfg::XS_BYTES);
#pragma unroll
          for (int u = 0; u < HPB; ++u) {
            const int unit = (B * HPB + u) % Cfg::UNITS;
            const uint32_t use = (blocks * HPB + u) / Cfg::UNITS;
            const MbarPhase room = {dempty(unit), (use & 1u) ^ 1u, kSiteTmemEmpty};
            const MbarPhase a = {afull(B % Cfg::A_BUFS), blocks / Cfg::A_BUFS & 1u, kSiteSmemFull};
            const MbarPhase x = {xfull(B), blocks / Cfg::RING & 1u, kSiteSmemFull};
            if (!(u == 0 ? mbar_wait_all_warp(wc, a, x, room) : mbar_wait_all_warp(wc, room))) return false;
            ptx::tc_fence_after();
            if (ptx::elect_one()) {
#pragma unroll
              for (int s = u * GRAN * SPG; s < (u + 1) * GRAN * SPG; ++s) {
                const uint32_t b_lo = x0 + (s / 4) * (TOK * 128 / 16) + 2u * (s % 4);
                const uint32_t a_col = tmem + Cfg::A_COL + B % Cfg::A_BUFS * 64 + s * 8;
                const uint32_t to = tmem + (unit * GRAN + s / SPG % GRAN) * NMMA;
                if (s % SPG == 0) ptx::umma_ts_f16<false>(to, a_col, b_lo, idesc);
                else ptx::umma_ts_f16<true>(to, a_col, b_lo, idesc);
              }
              ptx::umma_commit(dfull(B * HPB + u));
            }
            __syncwarp();
          }
          return true;
        };
        for (int item = first; item < items && ok; item += stride) {
          for (int kb = kb0; kb < kb1 && ok; ++kb, ++blocks) {
            switch (blocks % Cfg::RING) {
              case 0: ok = multiply(IntC<0>{}); break;
              case 1: ok = multiply(IntC<1>{}); break;
              case 2: ok = multiply(IntC<2>{}); break;
              case 3: ok = multiply(IntC<3>{}); break;
              default:
                if constexpr (Cfg::RING == 8) {
                  switch (blocks % Cfg::RING) {
                    case 4: ok = multiply(IntC<4>{}); break;
                    case 5: ok = multiply(IntC<5>{}); break;
                    case 6: ok = multiply(IntC<6>{}); break;
                    default: ok = multiply(IntC<7>{}); break;
                  }
                }
            }
          }
        }
      } else {
        // (stage: that of the block's first 64 columns)
        uint32_t turn = 0, lap = 0;              // accumulator, and how often it has been used
        // (lets the compiler know that all lanes have the same)
        auto uniform = [](uint32_t v) { return __shfl_sync(0xffffffffu, v, 0); };
        for (int item = first; item < items && ok; item += stride) {
          const Item it = item_of(item);
          // a tile that ends early is multiplied as far as it goes, in steps of 16 rows
          const int live = __shfl_sync(0xffffffffu, min(it.last - it.row, TOK), 0);
          const int halves = live > NMMA ? 2 : 1;
          const uint32_t idesc0 = uniform(ptx::umma_idesc(kFmt, kFmt, 128, min((live + 15) & ~15, NMMA)));
          const uint32_t idesc1 = uniform(ptx::umma_idesc(kFmt, kFmt, 128, max(min((live + 15 - NMMA) & ~15, NMMA), 16)));
          for (int kb = kb0; kb < kb1 && ok; ++kb, ++blocks) {
            const uint32_t buf = blocks % Cfg::A_BUFS;
            const int stage1 = stage + 1 == Cfg::X_STAGES ? 0 : stage + 1;
            const uint32_t phase1 = stage1 == 0 ? phase ^ 1u : phase;
            const uint32_t x0 = uniform(ptx::umma_desc_k_sw128_lo(base + Cfg::X_OFF + stage * Cfg::XS_BYTES));
            const uint32_t x1 = uniform(ptx::umma_desc_k_sw128_lo(base + Cfg::X_OFF + stage1 * Cfg::XS_BYTES));
            const uint32_t a_col = uniform(tmem + Cfg::A_COL + buf * 64);
            const MbarPhase a = {afull(buf), blocks / Cfg::A_BUFS & 1u, kSiteSmemFull};
            const MbarPhase xa = {xfull(stage), phase, kSiteSmemFull}, xb = {xfull(stage1), phase1, kSiteSmemFull};
            // (groups of 32: the hand-overs of a block in a row are more instructions than the first cache of them holds; as a
            // loop 2048 x 12288 x 4096 takes 411 us instead of 474. Two groups of 64 in a row measured the same.)
#pragma unroll(G == 32 ? 1 : GPS)
            for (int j = 0; j < GPS; ++j) {
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                if (h == halves) break;
                const MbarPhase room = {dempty(turn), (lap & 1u) ^ 1u, kSiteTmemEmpty};
                const uint32_t to = uniform(tmem + turn * NMMA);
                if (h == 0 && j == 0) ok = GPS == 1 ? mbar_wait_all_warp(wc, a, xa, xb, room) : mbar_wait_all_warp(wc, a, xa, room);
                else ok = h == 0 && j * G == 64 ? mbar_wait_all_warp(wc, xb, room) : mbar_wait_all_warp(wc, room);
                if (!ok) break;
                ptx::tc_fence_after();
                if (ptx::elect_one()) {
#pragma unroll
                  for (int s = j * SPG; s < (j + 1) * SPG; ++s) {
                    const uint32_t b_lo = (s < 4 ? x0 : x1) + h * (NMMA * 128 / 16) + 2u * (s % 4);
                    const uint32_t shape = h == 0 ? idesc0 : idesc1;
                    if (s == j * SPG) ptx::umma_ts_f16<false>(to, a_col + s * 8, b_lo, shape);
                    else ptx::umma_ts_f16<true>(to, a_col + s * 8, b_lo, shape);
                  }
                  ptx::umma_commit(dfull(turn));
                  if (h == halves - 1) {
                    if (j * G < 64 && (j + 1) * G >= 64) ptx::umma_commit(xempty(stage));
                    if (j == GPS - 1) {
                      ptx::umma_commit(xempty(stage1));
                      ptx::umma_commit(aempty(buf));
                    }
                  }
                }
                __syncwarp();
                if (++turn == Cfg::UNITS) {
                  turn = 0;
                  ++lap;
                }
              }
              if (!ok) break;
            }
            stage = stage1 + 1 == Cfg::X_STAGES ? 0 : stage1 + 1;
            phase = stage == 0 ? phase1 ^ 1u : phase1;
          }
        }
      }
    }
    drain();
    if (S > 1) ptx::cluster_sync();
    else __syncthreads();
    if (warp == Cfg::MMA_WARP) {
      ptx::tc_fence_after();
      ptx::tmem_dealloc<1>(tmem, Cfg::TMEM_COLS);
    }
    __syncwarp();
    if (S > 1) ptx::cluster_sync();
  }
}

}  // namespace fluxb
