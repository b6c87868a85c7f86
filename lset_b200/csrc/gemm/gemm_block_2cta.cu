// Block-scaled 8-bit products (block_scale.cuh) on CTA pairs: one 256 x 256 tile per pair, and the gated pair of
// projections whose epilogue activates and casts.
//
// Tiles, roles and barriers as in gemm_2cta.cu: CTA r of a pair stages its own 128 rows of A and half of B's
// 256, 256 bytes of depth a stage; one thread of the leader issues tcgen05.mma.cta_group::2 (M = 256, N = 256).
// What the scales add:
//   * four warps of each CTA (10-13) copy scale words from memory into tensor memory, 512 columns of depth at
//     a time and ahead of the issuer: the words of the CTA's 128 rows of A and of all 256 of B, which every
//     quarter of the lanes has to hold (each warp writes its own). Two groups of words are in flight.
//   * they need 2 x 16 of the 512 columns of tensor memory, so the two accumulators of 256 share 32 columns:
//     [0, 256) and [224, 480). The epilogue drains those first and says so (`tover`), and the issuer
//     waits for that before it starts the next tile.
//
//   warp 0      TMA producer                  warps 2-9    epilogue
//   warp 1      leader: MMA issuer            warps 10-13  scales
//
// DEEP: a tile's contraction is several sums (kDeepestSum says why), each in the accumulator whose turn it is; the
// epilogue adds them in 128 registers a thread, while the next one is in the making. For these the registers of the other
// warps go to those of the epilogue, so warpgroups have one role each: warps 4-7 scales, 8-15 epilogue. The gradient of
// gate and up at 4097 x 2048 x 8192 then is off fp32 sums' by 1.45e-4 of its norm for 1.66e-4, gate and up round on another
// side than in 64 bits in 4e-5 of the values for 7e-5 (8192 deep: 1.4e-4 for 3.2e-4). Measured in turn without / with,
// training steps: 4097 x 2048 x 8192 798 / 817 us, 16384 x 2560 x 9728 3754 / 3881.
//
// Measured by itself, L2 flushed: 8192 x 4096 x 4096 93 us (2.97 PFLOP/s, the tensor pipe active in 81 % of the cycles),
// 20960 x 6144 x 4096 338 us (3.12; 352 inside the layer), 16384 x 4096 x 4096 172 (3.20). Bound by the tensor cores where
// the contraction is deep, and by the power limit over seconds; by the epilogue where it is short (8192 x 8192 x 512 47 us).
// Rows stored from registers, for staging them in shared memory: 95.6 -> 92.9 us under the profiler at the first size.
#include <cuda_bf16.h>

#include "../common/pair.cuh"
#include "../common/pdl.h"
#include "../common/ptx.cuh"
#include "../common/tma_desc.h"
#include "block_gemm.h"
#include "block_glu.cuh"
#include "block_scale.cuh"

namespace lb {
namespace {

constexpr int BM = 128;                      // rows of A of a CTA
constexpr int BNp = 256, BNh = 128;          // rows of B of a pair, of a CTA
constexpr int BK = 256;                      // bytes (elements) of depth of a stage: two blocks
constexpr int kStages = 3;
constexpr int kGroup = 2;                    // stages that one group of scale words serves
constexpr int A_BYTES = BM * BK, B_BYTES = BNh * BK, STAGE_BYTES = A_BYTES + B_BYTES;
constexpr int kEpiWarps = 8;
// Warps: with DEEP the scale warps and the epilogue are whole warpgroups (warps 4-7 and 8-15), whose registers differ.
constexpr int kWarpsPlain = 2 + kEpiWarps + 4, kWarpsDeep = 16;
constexpr int kRegsLaunch = 128, kRegsFew = 48, kRegsEpi = 208;   // DEEP: of a thread, at launch and from then on
static_assert(2 * kRegsFew + 2 * kRegsEpi <= 4 * kRegsLaunch && kRegsLaunch * 32 * kWarpsDeep <= 65536, "");
constexpr int EPI_WORDS = 32 * 33;
constexpr int kBarBytes = 512;
constexpr int SMEM_BYTES = kStages * STAGE_BYTES + 1024 + kBarBytes + kEpiWarps * EPI_WORDS * 4;
constexpr int kAcc1 = 224, kScaleCols = 480, kSlots = 2;
static_assert(SMEM_BYTES <= 232448, "");

struct Block2Args {
  int M, N, K;
  const uint32_t *sa, *sb, *sb2;             // scale words of A's and B's rows; GLU: gate and up rows
  long long rows_sa, rows_sb;
  void* C;                                   // GLU: gate products (null: not wanted)
  long long ldc;
  int wide, wide_h;                          // rows of C (GLU: of both products), of h start at multiples of 32 bytes
  int accumulate;                            // fp32 only: C += result
  const __nv_bfloat16* bias;
  int a_e5m2, b_e5m2;
  int splits, stages_per_split;
  int stages_per_sum;                        // DEEP: stages of one sum in tensor memory; else those of a split
  long long split_stride;                    // elements between the outputs of two splits
  int band;                                  // rows of tiles in a band; 0: row by row
  int whole, items;                          // work items: `whole` tiles, then halves of 128 columns
  void* up_out;                              // GLU: up products, and act(gate) * up cast in blocks of a row
  uint8_t* h;
  long long ldh;
  uint32_t* h_scales;
  long long rows_h;
  int* status;
};

// D (both CTAs' tensor memory) (+)= block-scaled A * B of both CTAs' shared memory; leader thread only.
__device__ __forceinline__ void umma2_block(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                            uint32_t tmem_sa, uint32_t tmem_sb, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %6, 0;\n"
      "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n"
      "}\n"
      :
      : "r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(tmem_sa), "r"(tmem_sb), "r"(accumulate)
      : "memory");
}

// 32 bytes, a whole sector, from one lane.
__device__ __forceinline__ void st32(void* p, const uint32_t* w) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
               "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}
// A lane's WORDS words of a row, the first `bytes` of them (a multiple of 16); wide: at a multiple of 32.
template <int WORDS>
__device__ __forceinline__ void store_words(void* dst, const uint32_t (&w)[WORDS], int bytes, bool wide) {
  uint8_t* p = static_cast<uint8_t*>(dst);
  if (wide && bytes >= 4 * WORDS) {
#pragma unroll
    for (int j = 0; j < WORDS / 8; ++j) st32(p + 32 * j, w + 8 * j);
  } else {
#pragma unroll
    for (int j = 0; j < WORDS / 4; ++j)
      if (16 * j < bytes)
        *reinterpret_cast<uint4*>(p + 16 * j) = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
  }
}

// Registers of this warpgroup's threads from here on (all its warps take part).
template <int REGS>
__device__ __forceinline__ void fewer_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS));
}
template <int REGS>
__device__ __forceinline__ void more_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS));
}

template <typename OutT, int GLU, int DEEP>
__global__ void __launch_bounds__(32 * (DEEP ? kWarpsDeep : kWarpsPlain), 1)
    gemm_block_2cta_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                           const __grid_constant__ CUtensorMap tmB2, Block2Args g) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kStages * STAGE_BYTES);
  uint64_t* empty = full + kStages;
  uint64_t* tfull = empty + kStages;
  uint64_t* tempty = tfull + 2;
  uint64_t* sfull = tempty + 2;
  uint64_t* sempty = sfull + kSlots;
  uint64_t* tover = sempty + kSlots;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tover + 1);
  float* epi_stage = reinterpret_cast<float*>(smem + kStages * STAGE_BYTES + kBarBytes);

  constexpr int kEpi0 = DEEP ? 8 : 2, kScale0 = DEEP ? 4 : 2 + kEpiWarps;   // first warp of the epilogue, of the scales
  const int warp = warp_index();
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();   // 0 = leader
  const bool leader = rank == 0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], 2 * kEpiWarps);
    }
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(&sfull[s], 8);
      mbar_init(&sempty[s], 1);
    }
    mbar_init(tover, kEpiWarps);
    mbar_fence_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
    if (GLU) tma_prefetch_desc(&tmB2);
  }
  if (warp == 1) {
    tmem_alloc2(tmem_slot, 512);
    tmem_relinquish2();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();   // both CTAs' barriers exist before anything arrives on them from afar
  tc_fence_after();
  pdl_wait();
  pdl_trigger();
  const uint32_t tmem_base = *tmem_slot;

  constexpr int kTileN = GLU ? BNh : BNp;   // output columns (features) of a tile
  const int tiles_m = (g.M + 2 * BM - 1) / (2 * BM), tiles_n = (g.N + kTileN - 1) / kTileN;
  const int stages_total = (g.K + BK - 1) / BK;
  const int total = g.items;
  const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;
  // Tiles row by row or in bands (band_of in gemm_2cta.cu says why). m0: first row of this CTA's half.
  // narrow: an item of 128 columns, half a tile.
  bool narrow = false;
  auto decode = [&](int item, int& split, int& m0, int& n0, int& st0, int& st1) {
    narrow = !GLU && item >= g.whole;
    const int tile = narrow ? g.whole + (item - g.whole) / 2 : item;
    split = tile / (tiles_m * tiles_n);
    const int mn = tile - split * (tiles_m * tiles_n);
    int mt = mn / tiles_n, nt = mn - mt * tiles_n;
    if (g.band) {
      const int first = mn / (g.band * tiles_n) * g.band, at = mn - first * tiles_n;
      const int rows = min(g.band, tiles_m - first);
      nt = at / rows;
      mt = first + at - nt * rows;
    }
    m0 = mt * (2 * BM) + int(rank) * BM;
    n0 = nt * kTileN + (narrow ? ((item - g.whole) & 1) * BNh : 0);
    st0 = split * g.stages_per_split;
    st1 = min(st0 + g.stages_per_split, stages_total);
  };
  int split, m0, n0, st0, st1;

  if (DEEP && warp < kScale0) fewer_registers<kRegsFew>();
  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = pair; tile < total && ok; tile += npairs) {
        decode(tile, split, m0, n0, st0, st1);
        // (GLU: tmB2 is the up weight; else B in boxes of 64 rows, for narrow items)
        const int rows = narrow ? BNh / 2 : BNh;
        const int nb = GLU ? n0 : n0 + int(rank) * rows;
        const CUtensorMap* tb = (GLU ? !leader : narrow) ? &tmB2 : &tmB;
        for (int st = st0; st < st1; ++st) {
          if (!mbar_wait(&empty[stage], phase ^ 1u)) {
            report_status(g.status, kStatusTimeoutProducer);
            ok = false;
            break;
          }
          if (leader) mbar_expect_tx(&full[stage], 2 * (A_BYTES + rows * BK));
          uint8_t* sa = smem + stage * STAGE_BYTES;
          uint8_t* sb = sa + A_BYTES;
          const uint32_t bar = map_to_cta(&full[stage], 0);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            tma_load_2d_pair(sa + h * (BM * 128), &tmA, bar, st * BK + 128 * h, m0);
            tma_load_2d_pair(sb + h * (rows * 128), tb, bar, st * BK + 128 * h, nb);
          }
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (leader && elect_one()) {
      // ---------------------------------------------------------------- MMA issuer (leader)
      int stage = 0, group = 0, it = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = pair; tile < total && ok; tile += npairs) {
        decode(tile, split, m0, n0, st0, st1);
        const uint32_t idesc0 = umma_idesc_block(2 * BM, narrow ? BNh : BNp, g.a_e5m2, g.b_e5m2, 0);
        const uint32_t b_half = narrow ? BNh / 2 * 128 : BNh * 128;   // bytes of 128 of depth
        for (int s0 = st0; s0 < st1 && ok; s0 += g.stages_per_sum, ++it) {
          const int s1 = min(s0 + g.stages_per_sum, st1), acc = it & 1;
          if (!mbar_wait(&tempty[acc], ((it >> 1) & 1) ^ 1u) || (it > 0 && !mbar_wait(tover, (it - 1) & 1))) {
            report_status(g.status, kStatusTimeoutMma);
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t d_tmem = tmem_base + (acc ? kAcc1 : 0);
          for (int st = s0; st < s1; ++st) {
            const int at = (st - s0) % kGroup, slot = group % kSlots;
            if ((at == 0 && !mbar_wait_cluster(&sfull[slot], (group / kSlots) & 1)) || !mbar_wait(&full[stage], phase)) {
              report_status(g.status, kStatusTimeoutMma);
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t sa = smem_u32(smem + stage * STAGE_BYTES), sb = sa + A_BYTES;
            const uint32_t scales = tmem_base + kScaleCols + 16 * slot;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              if (k >= 4 && st * BK + kScaleBlock >= g.K) break;   // no second block: nor is there a scale for it
              const uint32_t sf = uint32_t(2 * at + k / 4);
              umma2_block(d_tmem, umma_smem_desc(sa + (k / 4) * (BM * 128) + (k % 4) * 32, 16, 1024),
                          umma_smem_desc(sb + (k / 4) * b_half + (k % 4) * 32, 16, 1024),
                          idesc0 | (sf << 4) | (sf << 29), scales, scales + 4, st > s0 || k > 0);
            }
            umma2_commit_both(&empty[stage], 1u);
            if (at == kGroup - 1 || st == s1 - 1) {
              umma2_commit_both(&sempty[slot], 1u);
              ++group;
            }
            if (++stage == kStages) {
              stage = 0;
              phase ^= 1u;
            }
          }
          if (ok) umma2_commit_both(&tfull[acc], 1u);
        }
      }
    }
    __syncwarp();
  } else if (warp >= kScale0 && warp < kScale0 + 4) {
    // ------------------------------------------------------------------ scale warps
    if constexpr (DEEP) fewer_registers<kRegsFew>();
    const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;
    const uint32_t arrive0 = map_to_cta(&sfull[0], 0), arrive1 = map_to_cta(&sfull[1], 0);
    uint32_t wa[4], wb[8];
    auto fetch = [&](int word) {   // words of depth 512 * word .. of this tile's rows
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int m = m0 + c * 32 + lane;
        wa[c] = m < g.M ? g.sa[word * g.rows_sa + m] : 0x7f7f7f7fu;
      }
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const int n = n0 + (GLU ? c & 3 : c) * 32 + lane;
        const uint32_t* sb = GLU && c >= 4 ? g.sb2 : g.sb;
        wb[c] = n < g.N ? sb[word * g.rows_sb + n] : 0x7f7f7f7fu;
      }
    };
    int group = 0;
    bool ok = true;
    int tile = pair;
    if (tile < total) {
      decode(tile, split, m0, n0, st0, st1);
      fetch(st0 / kGroup);
    }
    while (tile < total && ok) {
      const int first = st0 / kGroup, last = (st1 - 1) / kGroup;
      for (int w = first; w <= last; ++w, ++group) {
        const int slot = group % kSlots;
        // (all lanes take part in the store, and may see a bounded wait end differently)
        if (!__all_sync(0xffffffffu, mbar_wait(&sempty[slot], ((group / kSlots) & 1) ^ 1u))) {
          report_status(g.status, kStatusTimeoutEpilogue);
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t dst = tmem_base + lanes + kScaleCols + 16 * slot;
        tmem_st_32x32b_x4(dst, wa[0], wa[1], wa[2], wa[3]);
        tmem_st_32x32b_x8(dst + 4, wb);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(slot ? arrive1 : arrive0);
        if (w < last) {
          fetch(w + 1);
        } else if (tile + npairs < total) {
          decode(tile + npairs, split, m0, n0, st0, st1);
          fetch(st0 / kGroup);
        }
      }
      tile += npairs;
    }
  } else if (warp >= kEpi0) {
    // ------------------------------------------------------------------ epilogue
    if constexpr (DEEP) more_registers<kRegsEpi>();
    const int q = warp & 3;
    const int half = (warp - kEpi0) >> 2;
    const uint32_t tempty0 = map_to_cta(&tempty[0], 0), tempty1 = map_to_cta(&tempty[1], 0);
    const uint32_t over = map_to_cta(tover, 0);
    uint8_t* sblk = reinterpret_cast<uint8_t*>(epi_stage + (warp - kEpi0) * EPI_WORDS);
    int it = 0;
    bool ok = true;
    for (int tile = pair; tile < total; tile += npairs, ++it) {
      decode(tile, split, m0, n0, st0, st1);
      // the sum that is next in tensor memory
      auto arrived = [&] {
        ok = ok && __all_sync(0xffffffffu, mbar_wait(&tfull[it & 1], (it >> 1) & 1));
        if (!ok) report_status(g.status, kStatusTimeoutEpilogue);
        return ok;
      };
      // DEEP: all sums of the tile but the last, 32 columns a group, added in their order
      float before[DEEP ? 4 : 1][32];
      if constexpr (DEEP) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 32; ++j) before[i][j] = 0.f;
        for (int s0 = st0; ok && s0 + g.stages_per_sum < st1; s0 += g.stages_per_sum, ++it) {
          if (!arrived()) break;
          tc_fence_after();
          const int acc = it & 1;
          const uint32_t src = tmem_base + (uint32_t(q * 32) << 16) + (acc ? kAcc1 : 0);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            // (the groups of the tile's end below, in the same order)
            const int c = GLU ? 2 * half + ((i / 2 - half) & 1) + (i & 1) * (BNh / 32)
                              : (narrow ? 2 : 4) * half + ((i - half) & (narrow ? 1 : 3));
            if (GLU || !narrow || i < 2) {
              uint32_t r[32];
              tmem_ld_32x32b_x32(src + c * 32, r);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 32; ++j) before[i][j] += __uint_as_float(r[j]);
            }
            if (i == (GLU ? 1 : 0) && half != acc) {   // gate and up, or the one, of the columns that are shared
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive_remote(over);
            }
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_remote(acc ? tempty1 : tempty0);
        }
      }
      const int acc = it & 1;
      if (ok) arrived();
      if (!ok) {   // (the two warps of a row meet at a barrier for each tile, whatever either has waited for)
        if (GLU) asm volatile("bar.sync %0, 64;" ::"r"(1 + q) : "memory");
        continue;
      }
      tc_fence_after();
      const uint32_t src0 = tmem_base + (uint32_t(q * 32) << 16) + (acc ? kAcc1 : 0);
      const int row = m0 + q * 32 + lane;
      // the columns that the other accumulator shares: this one's last (acc 0) or first 32
      const bool shared_here = half != acc;
      // start with the last chunk of the half (DEEP: whichever accumulator it is, so that sums stay where they are)
      const int rot = (DEEP || acc == 0) && half == 1 ? -1 : 0;
      if constexpr (GLU) {
        uint32_t h[2][16];
        uint32_t top = 0u;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int c = 2 * half + ((i + rot) & 1);
          uint32_t rg[32], ru[32];
          tmem_ld_32x32b_x32(src0 + c * 32, rg);
          tmem_ld_32x32b_x32(src0 + BNh + c * 32, ru);
          tmem_ld_wait();
          if (i == 0 && shared_here) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_remote(over);
          }
          if constexpr (DEEP) {
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              rg[j] = __float_as_uint(before[2 * i][j] + __uint_as_float(rg[j]));
              ru[j] = __float_as_uint(before[2 * i + 1][j] + __uint_as_float(ru[j]));
            }
          }
          uint32_t w[2][16];   // gate, up
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            w[0][j] = pack_bf16x2(__uint_as_float(rg[2 * j]), __uint_as_float(rg[2 * j + 1]));
            w[1][j] = pack_bf16x2(__uint_as_float(ru[2 * j]), __uint_as_float(ru[2 * j + 1]));
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint4 v = block_glu8<GLU - 1>(
                make_uint4(w[0][4 * j], w[0][4 * j + 1], w[0][4 * j + 2], w[0][4 * j + 3]),
                make_uint4(w[1][4 * j], w[1][4 * j + 1], w[1][4 * j + 2], w[1][4 * j + 3]));
            h[i][4 * j] = v.x;
            h[i][4 * j + 1] = v.y;
            h[i][4 * j + 2] = v.z;
            h[i][4 * j + 3] = v.w;
          }
#pragma unroll
          for (int j = 0; j < 16; ++j) top = __vmaxu2(top, h[i][j] & 0x7fff7fffu);
          if (g.C != nullptr && row < g.M) {
            const long long at = row * g.ldc + n0 + c * 32;
            store_words(reinterpret_cast<OutT*>(g.C) + at, w[0], 64, g.wide);
            store_words(reinterpret_cast<OutT*>(g.up_out) + at, w[1], 64, g.wide);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_remote(acc ? tempty1 : tempty0);
        // a block of a row is this tile's 128 features: the largest magnitude of both halves
        top = max(top & 0xffffu, top >> 16);
        uint32_t* tops = reinterpret_cast<uint32_t*>(sblk) + acc * 32 + lane;   // two tiles in turn
        *tops = top;
        asm volatile("bar.sync %0, 64;" ::"r"(1 + q) : "memory");
        top = max(top, tops[half ? -4 * EPI_WORDS : 4 * EPI_WORDS]);   // the warp with the other half of the rows
        const float s = block_inverse<0>(top);
        if (row < g.M) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int f0 = n0 + (2 * half + ((i + rot) & 1)) * 32;
            uint32_t o[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float2 a = unpack_bf16x2(h[i][2 * j]), b = unpack_bf16x2(h[i][2 * j + 1]);
              o[j] = cast4<0>(a.x * s, a.y * s, b.x * s, b.y * s);
            }
            store_words(g.h + row * g.ldh + f0, o, 32, g.wide_h);
          }
          if (half == 0) {
            const int kb = n0 / kScaleBlock;
            uint8_t* p = reinterpret_cast<uint8_t*>(g.h_scales + (kb >> 2) * g.rows_h + row);
            p[kb & 3] = uint8_t(block_scale_byte<0>(top));
            if (n0 + kScaleBlock >= g.N)
              for (int k = (kb & 3) + 1; k < 4; ++k) p[k] = uint8_t(kScaleOne);
          }
        }
      } else {
        OutT* Cout = reinterpret_cast<OutT*>(g.C) + split * g.split_stride;
        const int chunks = narrow ? 2 : 4;   // of 32 columns, a half of the warps
#pragma unroll(DEEP ? 4 : 1)
        for (int i = 0; i < (DEEP ? 4 : chunks); ++i) {
          if (DEEP && i >= chunks) continue;
          const int c = chunks * half + ((i + rot) & (chunks - 1));
          uint32_t r[32];
          tmem_ld_32x32b_x32(src0 + c * 32, r);
          tmem_ld_wait();
          if (i == 0 && shared_here) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_remote(over);
          }
          if constexpr (DEEP) {
#pragma unroll
            for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(before[i][j] + __uint_as_float(r[j]));
          }
          const int col0 = n0 + c * 32;
          if (g.bias != nullptr) {
            const float b = col0 + lane < g.N ? __bfloat162float(g.bias[col0 + lane]) : 0.f;
#pragma unroll
            for (int j = 0; j < 32; ++j)
              r[j] = __float_as_uint(__uint_as_float(r[j]) + __shfl_sync(0xffffffffu, b, j));
          }
          if constexpr (sizeof(OutT) == 2) {
            uint32_t w[16];
#pragma unroll
            for (int j = 0; j < 16; ++j)
              w[j] = pack_bf16x2(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1]));
            if (row < g.M) store_words(Cout + row * g.ldc + col0, w, 2 * (g.N - col0), g.wide);
          } else if (!g.accumulate) {
            if (row < g.M) store_words(Cout + row * g.ldc + col0, r, 4 * (g.N - col0), g.wide);
          } else {
            float* st = reinterpret_cast<float*>(sblk);
#pragma unroll
            for (int j = 0; j < 32; ++j) st[lane * 33 + j] = __uint_as_float(r[j]);
            __syncwarp();
            const int rr = lane >> 3, cc = (lane & 7) * 4;
            if (col0 + cc < g.N) {
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                const int lr = k * 4 + rr, grow = m0 + q * 32 + lr;
                const float* sp = st + lr * 33 + cc;
                if (grow < g.M)   // one tile adds to an element: the order of tiles does not matter
                  red_add4(reinterpret_cast<float*>(Cout) + grow * g.ldc + col0 + cc, sp[0], sp[1], sp[2], sp[3]);
              }
            }
            __syncwarp();
          }
        }
        // this warp is done reading the accumulator
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_remote(acc ? tempty1 : tempty0);
      }
    }
  }

  // Nobody leaves while the partner may still read this CTA's shared memory, arrive on its barriers or (the
  // leader's products) write its tensor memory.
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  if (warp == 1) tmem_dealloc2(tmem_base, 512);
}

constexpr int kMaxDevices = 64;
int g_pairs[kMaxDevices];   // CTA pairs resident at once; 0: not asked yet

template <typename OutT, int GLU, int DEEP>
int launch_2cta(const CUtensorMap& tmA, const CUtensorMap& tmB, const CUtensorMap& tmB2, Block2Args& g,
                long long total, cudaStream_t stream) {
  auto kern = gemm_block_2cta_kernel<OutT, GLU, DEEP>;
  constexpr int kThreads = 32 * (DEEP ? kWarpsDeep : kWarpsPlain);
  static bool configured[kMaxDevices] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return -10;
  if (!configured[dev]) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES) != cudaSuccess)
      return -10;
    cudaFuncAttributes is{};
    // (warps that ask for more than the block was launched with would wait for good)
    if (DEEP && (cudaFuncGetAttributes(&is, kern) != cudaSuccess || is.numRegs != kRegsLaunch)) return -12;
    configured[dev] = true;
  }
  if (g_pairs[dev] == 0) {
    // not every SM has a partner that it can form a cluster with
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    int sms = 0, n = 0;
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    cfg.gridDim = dim3(sms > 1 ? sms / 2 * 2 : 2, 1, 1);
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.dynamicSmemBytes = SMEM_BYTES;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n <= 0) {
      cudaGetLastError();
      n = sms / 2 > 0 ? sms / 2 : 1;
    }
    g_pairs[dev] = n;
  }
  // The tiles of the last wave in halves, where those still fit in one. (No sum changes with it.) Measured in turn with
  // whole tiles / halves, at the power limit: a training step of the linear layer 8191 x 2560 -> 6144 (its weight gradient
  // has 240 tiles on 74 pairs) 403 / 394 us, of 16384 x 4096 -> 4096 788 / 788.
  const int rest = int(total % g_pairs[dev]);
  g.whole = g.items = int(total);
  if (!GLU && g.splits == 1 && rest > 0 && 2 * rest <= g_pairs[dev]) {
    g.whole = int(total) - rest;
    g.items = g.whole + 2 * rest;
  }
  const int pairs = g.items < g_pairs[dev] ? g.items : g_pairs[dev];
  return launch_pdl(kern, dim3(2 * pairs), dim3(kThreads), SMEM_BYTES, stream, pdl_enabled(), 2, tmA, tmB, tmB2, g);
}

constexpr int kBand = 16;
int band_of(int tiles_n, long long b_bytes) { return tiles_n > kBand && b_bytes > (32 << 20) ? kBand : 0; }

int stages_of_split(int K, int splits) {
  const int stages = (K + BK - 1) / BK;
  return ((stages + splits - 1) / splits + kGroup - 1) / kGroup * kGroup;   // whole groups of scale words
}
// Stages of one sum: equal parts of the contraction, of `deepest` at most.
int stages_of_sum(int K, int deepest) { return stages_of_split(K, block_2cta_sums(K, deepest)); }
static_assert(kDeepestSum % (kGroup * BK) == 0, "");

}  // namespace

bool block_2cta_splits_ok(int K, int splits) {
  const int stages = (K + BK - 1) / BK, each = stages_of_split(K, splits);
  return (stages + each - 1) / each == splits;
}

int block_2cta_sums(int K, int deepest) { return deepest > 0 ? (K + deepest - 1) / deepest : 1; }
int block_2cta_depth(int K, int splits) { return stages_of_split(K, splits) * BK; }

// N a multiple of 8, C 16-byte aligned, ldc a multiple of 8. splits > 1 (fp32): split s of the contraction writes its
// own sums to C + s * split_stride. deepest > 0 (bf16 without bias, splits = 1): sums of tensor memory are that deep at
// most, and added in registers.
int block_gemm_2cta(int splits, int deepest, long long split_stride, const BlockMat& A, const BlockMat& B, void* C, int M,
                    int N, int K, long long ldc, int out_fp32, int accumulate, const void* bias, int* status,
                    cudaStream_t stream) {
  const bool deep = block_2cta_sums(K, deepest) > 1;
  if (deep && (splits > 1 || out_fp32 || bias != nullptr || deepest % (kGroup * BK))) return -5;
  if ((N & 7) || (ldc & 7) || (reinterpret_cast<uintptr_t>(C) & 15)) return -5;
  if (splits > 1 && (!out_fp32 || accumulate || bias != nullptr)) return -5;
  if (splits < 1 || !block_2cta_splits_ok(K, splits)) return -5;
  CUtensorMap tmA, tmB, tmBh;
  int rc = make_tmap_2d(&tmA, A.data, 1, (uint64_t)K, (uint64_t)M, (uint64_t)A.ld, 128, BM, true);
  if (rc) return rc;
  rc = make_tmap_2d(&tmB, B.data, 1, (uint64_t)K, (uint64_t)N, (uint64_t)B.ld, 128, BNh, true);
  if (rc) return rc;
  rc = make_tmap_2d(&tmBh, B.data, 1, (uint64_t)K, (uint64_t)N, (uint64_t)B.ld, 128, BNh / 2, true);
  if (rc) return rc;
  const int tiles_m = (M + 2 * BM - 1) / (2 * BM), tiles_n = (N + BNp - 1) / BNp;
  Block2Args g{};
  g.M = M;
  g.N = N;
  g.K = K;
  g.sa = A.scales;
  g.sb = B.scales;
  g.rows_sa = A.rows_s;
  g.rows_sb = B.rows_s;
  g.C = C;
  g.ldc = ldc;
  g.wide = !(reinterpret_cast<uintptr_t>(C) & 31) && !(ldc & (out_fp32 ? 7 : 15));
  g.accumulate = accumulate;
  g.bias = static_cast<const __nv_bfloat16*>(bias);
  g.a_e5m2 = A.e5m2 ? 1 : 0;
  g.b_e5m2 = B.e5m2 ? 1 : 0;
  g.splits = splits;
  g.stages_per_split = stages_of_split(K, splits);
  g.stages_per_sum = deep ? stages_of_sum(K, deepest) : g.stages_per_split;
  g.split_stride = splits > 1 ? split_stride : 0;
  if (g.split_stride & 7) g.wide = 0;
  g.band = band_of(tiles_n, 1LL * N * K);
  g.status = status;
  const long long total = 1LL * tiles_m * tiles_n * splits;
  if (total > 0x7fff0000LL) return -3;   // (tiles are counted in steps of the grid)
  if (out_fp32) return launch_2cta<float, 0, 0>(tmA, tmB, tmBh, g, total, stream);
  return deep ? launch_2cta<__nv_bfloat16, 0, 1>(tmA, tmB, tmBh, g, total, stream)
              : launch_2cta<__nv_bfloat16, 0, 0>(tmA, tmB, tmBh, g, total, stream);
}

// gate and up weights [I, K], I a multiple of 128, with a common row stride and scale words of common groups. Both
// products, rounded to bf16, also go to gate and up (rows ld_gu elements apart) unless those are null. deepest: as above.
int block_gemm_glu(int kind, int deepest, const BlockMat& A, const BlockMat& Wg, const BlockMat& Wu, int M, int I, int K,
                   void* gate, void* up, long long ld_gu, const BlockMat& h, int* status, cudaStream_t stream) {
  const bool deep = block_2cta_sums(K, deepest) > 1;
  if (deep && deepest % (kGroup * BK)) return -5;
  if ((I % kScaleBlock) || (ld_gu & 7) || (gate == nullptr) != (up == nullptr) || Wg.rows_s != Wu.rows_s) return -3;
  CUtensorMap tmA, tmG, tmU;
  int rc = make_tmap_2d(&tmA, A.data, 1, (uint64_t)K, (uint64_t)M, (uint64_t)A.ld, 128, BM, true);
  if (rc) return rc;
  rc = make_tmap_2d(&tmG, Wg.data, 1, (uint64_t)K, (uint64_t)I, (uint64_t)Wg.ld, 128, BNh, true);
  if (rc) return rc;
  rc = make_tmap_2d(&tmU, Wu.data, 1, (uint64_t)K, (uint64_t)I, (uint64_t)Wu.ld, 128, BNh, true);
  if (rc) return rc;
  const int tiles_m = (M + 2 * BM - 1) / (2 * BM), tiles_n = I / BNh;
  Block2Args g{};
  g.M = M;
  g.N = I;
  g.K = K;
  g.sa = A.scales;
  g.sb = Wg.scales;
  g.sb2 = Wu.scales;
  g.rows_sa = A.rows_s;
  g.rows_sb = Wg.rows_s;
  g.C = gate;
  g.up_out = up;
  g.ldc = ld_gu;
  g.wide = !(reinterpret_cast<uintptr_t>(gate) & 31) && !(reinterpret_cast<uintptr_t>(up) & 31) && !(ld_gu & 15);
  g.wide_h = !(reinterpret_cast<uintptr_t>(h.data) & 31) && !(h.ld & 31);
  g.a_e5m2 = A.e5m2 ? 1 : 0;
  g.b_e5m2 = Wg.e5m2 ? 1 : 0;
  g.splits = 1;
  g.stages_per_split = stages_of_split(K, 1);
  g.stages_per_sum = deep ? stages_of_sum(K, deepest) : g.stages_per_split;
  g.band = band_of(tiles_n, 2LL * I * K);
  g.h = h.data;
  g.ldh = h.ld;
  g.h_scales = h.scales;
  g.rows_h = h.rows_s;
  g.status = status;
  const long long total = 1LL * tiles_m * tiles_n;
  if (total > 0x7fff0000LL) return -3;   // (tiles are counted in steps of the grid)
  if (deep)
    return kind == kSwiglu ? launch_2cta<__nv_bfloat16, 1 + kSwiglu, 1>(tmA, tmG, tmU, g, total, stream)
                           : launch_2cta<__nv_bfloat16, 1 + kGeglu, 1>(tmA, tmG, tmU, g, total, stream);
  return kind == kSwiglu ? launch_2cta<__nv_bfloat16, 1 + kSwiglu, 0>(tmA, tmG, tmU, g, total, stream)
                         : launch_2cta<__nv_bfloat16, 1 + kGeglu, 0>(tmA, tmG, tmU, g, total, stream);
}

}  // namespace lb
