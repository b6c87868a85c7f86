// C[M, N] = A · Bᵀ (+ bias) of 8-bit floats in blocks of 128 (block_scale.cuh): A [M, K] and B [N, K] both
// K-major, the scales applied by the tensor cores.
//
// One CTA per 128 columns of C (rows of B, the M side of the instruction, so that a warp stores
// neighbouring columns) and TN rows of C (rows of A, its N side): with few tokens the tile is filled by the
// weights, which is what such a product streams. The contraction may be split over the CTAs of a cluster; their
// sums are added through distributed shared memory in the order of their ranks, so a result never depends
// on timing.
//
//   warp 0      TMA producer: 128 bytes (one block) of B's and A's rows a stage
//   warp 1      MMA issuer: four instructions a stage; the scale words of four blocks are in TMEM
//   warps 2-5   copy scale words from memory to TMEM ahead of the issuer (the instruction reads them from
//               every quarter of the lanes: each warp writes its own), then drain the accumulator
//
// CAST: A is bf16 still, and warps 2-5 cast the blocks of its rows on their way into shared memory, each CTA those of
// its own depth. For up to 32 rows, where a launch (3 us with its gap, and the host's 4) costs more than casting the
// few rows in every CTA: 12 x 2560 x 4096 11.0 -> 8.1 us.
//
// Bound by launch, set-up and epilogue (3.6 us of an empty contraction in tiles of 16 rows, 8.2 in tiles of 128) and
// then by the weights' way from memory: 12 x 19456 x 2560 in 12.4 us (4.0 TB/s), 12 x 2560 x 9728 in 10.1 split four
// ways (19.4 whole). Sums go through shared memory so that a thread stores 16 bytes: as 2-byte stores from the
// accumulator's lanes the epilogue of 128 rows took 7 us more.
#include <cuda_bf16.h>
#include <math.h>

#include "../common/pdl.h"
#include "../common/ptx.cuh"
#include "../common/tma_desc.h"
#include "block_gemm.h"
#include "block_scale.cuh"

namespace lb {
namespace {

constexpr int kBP = 128;          // columns of C of a CTA
constexpr int kSlots = 4;         // groups of scale words in TMEM; a group serves four stages
constexpr int kThreads1 = 192;

template <int TN, int CAST = 0>
struct Cfg {
  static constexpr int kStages = TN <= 16 ? 6 : (TN <= 64 ? (TN <= 32 ? 5 : 4) : 3);
  static constexpr int kP = kBP * 128, kQ = TN * 128;    // bytes of a stage
  static constexpr int kAcc = TN < 32 ? 32 : TN;         // columns of the accumulator in TMEM
  static constexpr int kOwn = kAcc + 8 * kSlots;         // CAST: scales of A, four columns (one used) a stage
  static constexpr int kCols = TN <= 32 && !CAST ? 64 : (TN <= 64 ? 128 : 256);
  static constexpr int kBatch = TN <= 16 ? 3 : 2;        // CAST: blocks whose scales are handed over together
  static constexpr int kShare = CAST ? 2 * kBatch * TN * 4 : 0;
  static constexpr int kSmem = kStages * (kP + kQ) + 1024 + 256 + kShare;
  static_assert(kOwn + (CAST ? 4 * kStages : 0) <= kCols && 2 * kBatch <= kStages + 1, "");
  static_assert(kStages * (kP + kQ) >= kBP * TN * 4, "partial sums reuse the stages");
};

struct BlockArgs {
  int M, N, K;
  const uint32_t *sa, *sb;       // scale words of A's and B's rows
  long long rows_sa, rows_sb;    // words of a group of four blocks
  void* C;
  long long ldc;
  int out_fp32, accumulate;
  const __nv_bfloat16* bias;
  int a_e5m2, b_e5m2;
  int q_rows;                    // rows of A in a box: TN, or M where that is less
  const __nv_bfloat16* x;        // CAST: A, rows ldx elements apart
  long long ldx;
  int tiles_m;
  int vec;                       // rows of C start at multiples of eight elements and 16 bytes
  int* status;
};

__device__ __forceinline__ void cluster_sync_block() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr, uint32_t rank) {
  uint32_t at;
  float4 v;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(at)
               : "memory");
  return v;
}

// Eight columns from n on of row m of C, v their sums.
__device__ __forceinline__ void store_c8(const BlockArgs& g, int m, int n, float (&v)[8]) {
  if (g.bias != nullptr) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (n + i < g.N) v[i] += __bfloat162float(g.bias[n + i]);
  }
  const long long at = m * g.ldc + n;
  const bool whole = g.vec && n + 8 <= g.N;
  if (g.out_fp32) {
    float* p = static_cast<float*>(g.C) + at;
    if (whole) {
      float4* p4 = reinterpret_cast<float4*>(p);
      float4 a = make_float4(v[0], v[1], v[2], v[3]), b = make_float4(v[4], v[5], v[6], v[7]);
      if (g.accumulate) {
        const float4 x = p4[0], y = p4[1];
        a = make_float4(x.x + a.x, x.y + a.y, x.z + a.z, x.w + a.w);
        b = make_float4(y.x + b.x, y.y + b.y, y.z + b.z, y.w + b.w);
      }
      p4[0] = a;
      p4[1] = b;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (n + i < g.N) p[i] = g.accumulate ? p[i] + v[i] : v[i];
    }
  } else {
    __nv_bfloat16* p = static_cast<__nv_bfloat16*>(g.C) + at;
    if (whole) {
      *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]),
                                                pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (n + i < g.N) p[i] = __float2bfloat16(v[i]);
    }
  }
}

// Warps 2-5 of a CTA with CAST: rows m0 .. m0 + TN - 1 of A, blocks kb0 .. kb1 - 1, cast into the stages; put(i) stores
// group i of B's scale words. A thread has TN values of a block, 128 / TN threads a row; loads run kAhead blocks
// ahead. Scales go through shared memory to the lanes that hold their rows in tensor memory, kBatch blocks at a
// time (a block at a time took 1 us each).
template <int TN, typename Put>
__device__ __forceinline__ bool cast_rows(const BlockArgs& g, uint8_t* smem, uint64_t* full, uint64_t* empty, int m0,
                                          int kb0, int kb1, uint32_t tmem_lanes, Put&& put) {
  using F = Cfg<TN, 1>;
  constexpr int kVecs = TN / 8, kPer = 128 / TN, kBatch = F::kBatch, kAhead = 2 * kBatch;
  const int t = threadIdx.x - 64, lane = threadIdx.x & 31;
  const int r = t / kPer, c0 = t % kPer * TN, m = m0 + r;
  uint32_t* share = reinterpret_cast<uint32_t*>(smem + F::kSmem - 1024 - F::kShare);   // [2][kBatch][TN]
  uint4 x[kAhead][kVecs];
  auto load = [&](int kb, uint4 (&v)[kVecs]) {
#pragma unroll
    for (int j = 0; j < kVecs; ++j) {
      const int k = kb * kScaleBlock + c0 + 8 * j;
      v[j] = kb < kb1 && m < g.M && k < g.K ? *reinterpret_cast<const uint4*>(g.x + m * g.ldx + k)
                                            : make_uint4(0u, 0u, 0u, 0u);
    }
  };
#pragma unroll
  for (int p = 0; p < kAhead; ++p) load(kb0 + p, x[p]);
  // A wait that has run out ends the waiting, not the loop: the four warps meet at a barrier in it.
  bool ok = true;
  int stage = 0, group = 0;
  uint32_t phase = 0;
  for (int base = kb0; base < kb1; base += kAhead) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int first = stage;
      if (base + half * kBatch >= kb1) break;
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int p = half * kBatch + i, kb = base + p;
        if (kb >= kb1) break;
        if (ok && (kb == kb0 || (kb & 3) == 0)) ok = put(group++);
        ok = ok && __all_sync(0xffffffffu, mbar_wait(&empty[stage], phase ^ 1u));
        uint32_t top = 0u;
#pragma unroll
        for (int j = 0; j < kVecs; ++j) {
          const uint4& q = x[p][j];
          top = __vmaxu2(top, __vmaxu2(__vmaxu2(q.x & 0x7fff7fffu, q.y & 0x7fff7fffu),
                                       __vmaxu2(q.z & 0x7fff7fffu, q.w & 0x7fff7fffu)));
        }
        top = max(top & 0xffffu, top >> 16);
#pragma unroll
        for (int o = kPer / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float s = block_inverse<0>(top);
        uint8_t* sq = smem + stage * (F::kP + F::kQ) + F::kP;
#pragma unroll
        for (int j = 0; j < kVecs / 2; ++j) {
          uint32_t o[4];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint4& q = x[p][2 * j + h];
            const float2 a = unpack_bf16x2(q.x), b = unpack_bf16x2(q.y), c = unpack_bf16x2(q.z), d = unpack_bf16x2(q.w);
            o[2 * h] = cast4<0>(a.x * s, a.y * s, b.x * s, b.y * s);
            o[2 * h + 1] = cast4<0>(c.x * s, c.y * s, d.x * s, d.y * s);
          }
          *reinterpret_cast<uint4*>(sq + swz128_offset(r, c0 / 16 + j)) = make_uint4(o[0], o[1], o[2], o[3]);
        }
        if (t % kPer == 0) share[(half * kBatch + i) * TN + r] = block_scale_byte<0>(top) * 0x01010101u;
        load(kb + kAhead, x[p]);
        if (++stage == F::kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      fence_proxy_async_smem();
      asm volatile("bar.sync 1, 128;" ::: "memory");
      int at = first;
      tc_fence_after();   // the products of these stages' last blocks are behind (`empty`)
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        if (base + half * kBatch + i >= kb1) break;
        const uint32_t e = lane < TN ? share[(half * kBatch + i) * TN + lane] : 0x7f7f7f7fu;
        asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(tmem_lanes + F::kOwn + 4 * at), "r"(e)
                     : "memory");
        if (++at == F::kStages) at = 0;
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      at = first;
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        if (base + half * kBatch + i >= kb1) break;
        if (lane == 0) mbar_arrive(&full[at]);
        if (++at == F::kStages) at = 0;
      }
    }
  }
  return ok;
}

template <int TN, int CAST>
__global__ void __launch_bounds__(kThreads1, 2)
    gemm_block_kernel(const __grid_constant__ CUtensorMap tmP, const __grid_constant__ CUtensorMap tmQ,
                      BlockArgs g) {
  using F = Cfg<TN, CAST>;
  constexpr int kStages = F::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kStages * (F::kP + F::kQ));
  uint64_t* empty = full + kStages;
  uint64_t* sfull = empty + kStages;
  uint64_t* sempty = sfull + kSlots;
  uint64_t* tfull = sempty + kSlots;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tfull + 1);

  const int warp = warp_index();
  const int lane = threadIdx.x & 31;
  const int splits = int(cluster_size()), rank = int(cluster_rank());
  const int tile = blockIdx.x / splits;
  const int nt = tile / g.tiles_m, mt = tile - nt * g.tiles_m;
  const int n0 = nt * kBP, m0 = mt * TN;
  const int kb_total = (g.K + kScaleBlock - 1) / kScaleBlock;
  const int kb0 = int(1LL * kb_total * rank / splits), kb1 = int(1LL * kb_total * (rank + 1) / splits);

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], CAST ? 5 : 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(&sfull[s], 4);
      mbar_init(&sempty[s], 1);
    }
    mbar_init(tfull, 1);
    mbar_fence_init();
    tma_prefetch_desc(&tmP);
    if (!CAST) tma_prefetch_desc(&tmQ);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, F::kCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_wait();
  pdl_trigger();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    if (elect_one()) {
      const uint32_t bytes = F::kP + (CAST ? 0 : g.q_rows * 128);
      int stage = 0;
      uint32_t phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&empty[stage], phase ^ 1u)) {
          report_status(g.status, kStatusTimeoutProducer);
          break;
        }
        mbar_expect_tx(&full[stage], bytes);
        uint8_t* sp = smem + stage * (F::kP + F::kQ);
        tma_load_2d(sp, &tmP, &full[stage], kb * kScaleBlock, n0);
        if (!CAST) tma_load_2d(sp + F::kP, &tmQ, &full[stage], kb * kScaleBlock, m0);
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int kb = kb0; kb < kb1; ++kb) {
        const int group = (kb >> 2) - (kb0 >> 2), slot = group % kSlots;
        if ((kb == kb0 || (kb & 3) == 0) && !mbar_wait(&sfull[slot], (group / kSlots) & 1)) ok = false;
        if (!ok || !mbar_wait(&full[stage], phase)) {
          report_status(g.status, kStatusTimeoutMma);
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t sp = smem_u32(smem + stage * (F::kP + F::kQ)), sq = sp + F::kP;
        const uint32_t scales = tmem + F::kAcc + 8 * slot;
        const uint32_t scales_q = CAST ? tmem + F::kOwn + 4 * stage : scales + 4;
        const uint32_t idesc = umma_idesc_block(kBP, TN, g.b_e5m2, g.a_e5m2, kb & 3);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          umma_block(tmem, umma_smem_desc(sp + 32 * k, 16, 1024), umma_smem_desc(sq + 32 * k, 16, 1024), idesc,
                     scales, scales_q, kb > kb0 || k > 0);
        umma_commit(&empty[stage]);
        if ((kb & 3) == 3) umma_commit(&sempty[slot]);
        if (++stage == kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (ok) umma_commit(tfull);
    }
    __syncwarp();
  } else {
    const int q = warp & 3;
    const uint32_t lanes = uint32_t(q * 32) << 16;
    bool ok = true;
    if (kb1 > kb0) {
      const int g0 = kb0 >> 2, groups = ((kb1 - 1) >> 2) - g0 + 1;
      uint32_t w[8];
      auto fetch = [&](int i) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int n = n0 + c * 32 + lane, m = m0 + c * 32 + lane;
          w[c] = n < g.N ? g.sb[(g0 + i) * g.rows_sb + n] : 0x7f7f7f7fu;
          if (!CAST) w[4 + c] = c * 32 < TN && m < g.M ? g.sa[(g0 + i) * g.rows_sa + m] : 0x7f7f7f7fu;
        }
      };
      // group i of scale words into its slot; false where the wait for it ran out
      auto put = [&](int i) {
        const int slot = i % kSlots;
        // (all lanes take part in the store, and may see a bounded wait end differently)
        if (!__all_sync(0xffffffffu, mbar_wait(&sempty[slot], ((i / kSlots) & 1) ^ 1u))) return false;
        tc_fence_after();   // the products that read the slot are behind
        if (CAST)
          tmem_st_32x32b_x4(tmem + lanes + F::kAcc + 8 * slot, w[0], w[1], w[2], w[3]);
        else
          tmem_st_32x32b_x8(tmem + lanes + F::kAcc + 8 * slot, w);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sfull[slot]);
        if (i + 1 < groups) fetch(i + 1);
        return true;
      };
      fetch(0);
      if constexpr (!CAST) {
        for (int i = 0; i < groups && ok; ++i) ok = put(i);
      } else {
        ok = cast_rows<TN>(g, smem, full, empty, m0, kb0, kb1, tmem + lanes, put);
      }
      ok = ok && __all_sync(0xffffffffu, mbar_wait(tfull, 0));
      if (!ok) report_status(g.status, kStatusTimeoutEpilogue);
      tc_fence_after();
    }
    // sums to shared memory, [row of A][column of C], where the operands lay
    float* part = reinterpret_cast<float*>(smem);
#pragma unroll 1
    for (int c = 0; c < TN / 16 && m0 + 16 * c < g.M; ++c) {
      uint32_t r[16];
      if (kb1 > kb0 && ok) {
        tmem_ld_32x32b_x16(tmem + lanes + 16 * c, r);
        tmem_ld_wait();
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) r[j] = 0u;
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) part[(16 * c + j) * kBP + q * 32 + lane] = __uint_as_float(r[j]);
    }
    tc_fence_before();
  }
  if (splits > 1)
    cluster_sync_block();
  else
    __syncthreads();
  // rank r of the cluster adds and stores every splits-th row from r on, eight columns a thread
  for (int i = threadIdx.x; i < TN / splits * (kBP / 8); i += kThreads1) {
    const int j = rank + i / (kBP / 8) * splits, n = n0 + i % (kBP / 8) * 8;
    if (m0 + j >= g.M) break;
    if (n >= g.N) continue;
    const uint32_t at = smem_u32(smem) + (j * kBP + i % (kBP / 8) * 8) * 4;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < splits; ++s) {
      const float4 a = ld_cluster_f4(at, s), b = ld_cluster_f4(at + 16, s);
      v[0] += a.x;
      v[1] += a.y;
      v[2] += a.z;
      v[3] += a.w;
      v[4] += b.x;
      v[5] += b.y;
      v[6] += b.z;
      v[7] += b.w;
    }
    store_c8(g, m0 + j, n, v);
  }
  if (splits > 1) cluster_sync_block();   // nobody's sums go before they are read
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, F::kCols);
}

constexpr int kMaxDevices = 64;

template <int TN, int CAST>
int launch_block(const CUtensorMap& tmP, const CUtensorMap& tmQ, const BlockArgs& g, long long tiles,
                 int splits, cudaStream_t stream) {
  static bool configured[kMaxDevices] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return -10;
  if (!configured[dev]) {
    if (cudaFuncSetAttribute(gemm_block_kernel<TN, CAST>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             Cfg<TN, CAST>::kSmem) != cudaSuccess)
      return -10;
    configured[dev] = true;
  }
  return launch_pdl(gemm_block_kernel<TN, CAST>, dim3(unsigned(tiles * splits)), dim3(kThreads1), Cfg<TN, CAST>::kSmem,
                    stream, pdl_enabled(), splits, tmP, tmQ, g);
}

// What a launch takes apart from A.
int block_args(BlockArgs& g, CUtensorMap* tmP, int tn, int splits, const BlockMat& B, void* C, int M, int N, int K,
               long long ldc, int out_fp32, int accumulate, const void* bias, int* status, long long* tiles) {
  const int kb = (K + kScaleBlock - 1) / kScaleBlock;
  if (splits < 1 || splits > 8 || splits > kb) return -5;
  g.M = M;
  g.N = N;
  g.K = K;
  g.sb = B.scales;
  g.rows_sb = B.rows_s;
  g.C = C;
  g.ldc = ldc;
  g.out_fp32 = out_fp32;
  g.accumulate = accumulate;
  g.bias = static_cast<const __nv_bfloat16*>(bias);
  g.b_e5m2 = B.e5m2 ? 1 : 0;
  g.q_rows = M < tn ? M : tn;
  g.tiles_m = (M + tn - 1) / tn;
  g.vec = !(ldc & 7) && !(reinterpret_cast<uintptr_t>(C) & 15);
  g.status = status;
  *tiles = 1LL * g.tiles_m * ((N + kBP - 1) / kBP);
  if (*tiles * splits > 0x7fffffffLL) return -3;
  return make_tmap_2d(tmP, B.data, 1, (uint64_t)K, (uint64_t)N, (uint64_t)B.ld, 128, kBP, true);
}

}  // namespace

int block_gemm_1cta(int tn, int splits, const BlockMat& A, const BlockMat& B, void* C, int M, int N, int K,
                    long long ldc, int out_fp32, int accumulate, const void* bias, int* status,
                    cudaStream_t stream) {
  BlockArgs g{};
  CUtensorMap tmP, tmQ;
  long long tiles = 0;
  int rc = block_args(g, &tmP, tn, splits, B, C, M, N, K, ldc, out_fp32, accumulate, bias, status, &tiles);
  if (rc) return rc;
  g.sa = A.scales;
  g.rows_sa = A.rows_s;
  g.a_e5m2 = A.e5m2 ? 1 : 0;
  rc = make_tmap_2d(&tmQ, A.data, 1, (uint64_t)K, (uint64_t)M, (uint64_t)A.ld, 128, uint32_t(g.q_rows), true);
  if (rc) return rc;
  switch (tn) {
    case 16: return launch_block<16, 0>(tmP, tmQ, g, tiles, splits, stream);
    case 32: return launch_block<32, 0>(tmP, tmQ, g, tiles, splits, stream);
    case 64: return launch_block<64, 0>(tmP, tmQ, g, tiles, splits, stream);
    case 128: return launch_block<128, 0>(tmP, tmQ, g, tiles, splits, stream);
  }
  return -5;
}

// Up to 1280 deep: every CTA casts the rows to its own depth, 0.3 us a block beside what the weights take. Measured in
// one launch / two: 12 x 4096 x 2560 (640 deep a CTA) 8.1 / 11.0 us, 24 x 19456 x 2560 (2560 deep) 18.7 / 17.5.
bool block_casts_itself(const BlockPlan& p, int M, int K) {
  return M <= 32 && p.kernel == 0 && p.tn <= 32 && K <= 1280 * p.splits;
}

int block_gemm_cast(const BlockPlan& p, const void* x, long long ldx, const BlockMat& B, void* C, int M, int N, int K,
                    long long ldc, int out_fp32, const void* bias, int* status, cudaStream_t stream) {
  if (!block_casts_itself(p, M, K) || (K & 7) || (ldx & 7) || (reinterpret_cast<uintptr_t>(x) & 15)) return -3;
  BlockArgs g{};
  CUtensorMap tmP;
  long long tiles = 0;
  const int rc = block_args(g, &tmP, p.tn, p.splits, B, C, M, N, K, ldc, out_fp32, 0, bias, status, &tiles);
  if (rc) return rc;
  g.x = static_cast<const __nv_bfloat16*>(x);
  g.ldx = ldx;
  return p.tn == 16 ? launch_block<16, 1>(tmP, tmP, g, tiles, p.splits, stream)
                    : launch_block<32, 1>(tmP, tmP, g, tiles, p.splits, stream);
}

// Modelled time (us) of a product, beside 1431 runs of 173 sizes (rows 1 to 6144, columns 256 to 19456, depths 256 to
// 9728, every tile and split that fits, with what a launch costs in a CUDA graph): off by 13 % in the mean for the
// one-CTA kernel, by 8 % for the pairs; the variant it chooses takes 1.4 % longer than the best in the mean and 20 % at
// most, and 0.7 and 17 % where sums may be 1024 deep. Measured at what the choice turns on: 128 x 2304 x 768 5.0 us in
// tiles of 16, 6.2 on pairs; 128 x 19456 x 2560 17.8 in tiles of 128, 37.0 of 16, 20.0 on pairs; 12 x 2560 x 9728 10.1
// split four ways, 19.4 whole; 1000 x 4096 x 2560 13.6 on pairs, 16.3 in tiles of 128; 768 x 1152 x 8191 17.6 on pairs
// split four ways, 20.0 whole (in halves); 4097 x 16384 x 2048 100.5 on pairs, 106.2 as two sums.
static float cost_1cta(int M, int N, int K, int tn, int splits) {
  // launch, set-up and epilogue; 1000 deep of one CTA on an SM; of one of two
  constexpr float kSet[4] = {3.6f, 4.1f, 6.2f, 8.2f}, kOne[4] = {1.67f, 1.77f, 1.85f, 2.36f},
                  kTwo[4] = {1.29f, 1.56f, 1.47f, 2.14f};
  const int i = tn == 16 ? 0 : (tn == 32 ? 1 : (tn == 64 ? 2 : 3));
  const float ctas = 1.f * ((M + tn - 1) / tn) * ((N + kBP - 1) / kBP) * splits;
  const float depth = 1e-3f * K / splits, waves = ceilf(ctas / 296.f);
  const float body = fmaxf(kOne[i] * depth * waves, kTwo[i] * depth * ceilf(ctas / 148.f));
  const float t = kSet[i] * (0.5f + 0.5f * waves) + body + (splits > 1 ? 0.56f * splits : 0.f);
  return fmaxf(t, 4.8f + 0.2e-6f * N * float(K));   // what memory takes for the weights
}
// (The plan depends on the sizes alone, not on the device's count of pairs: storage is sized by it, and it fixes the
// order of sums.)
static float cost_2cta(int M, int N, int K, int splits, int deepest, bool halves) {
  constexpr float pairs = 74.f;
  const float tiles = 1.f * ((M + 255) / 256) * ((N + 255) / 256) * splits;
  const float each = 1e-3f * K / splits, full = floorf(tiles / pairs), rest = tiles - full * pairs;
  // `halves`: a last wave of few tiles runs in those
  const float waves = full + (rest == 0.f ? 0.f : (halves && splits == 1 && 2.f * rest <= pairs ? 0.55f : 1.f));
  // (the issuer waits for the end of a sum and the first of its columns before it starts the next: 0.6 to 0.8 us)
  const float joins = 0.6f * (block_2cta_sums(K, deepest) - 1);
  return 4.85f + waves * (1.83f + joins + 2.4f * each) +
         (splits > 1 ? 3.35f + 0.6e-6f * splits * M * float(N) : 0.f);
}

BlockPlan block_plan(int M, int N, int K, bool aligned, int deepest) {
  BlockPlan best{0, 128, 1, INFINITY, 0};
  const int kb = (K + kScaleBlock - 1) / kScaleBlock;
  if (deepest == 0 || K <= deepest) best.cost = cost_1cta(M, N, K, 128, 1);
  for (int tn = 16; tn <= 128; tn *= 2) {
    if (tn >= 32 && tn >= 2 * M) break;
    for (int s = 1; s <= 8 && s <= kb; s *= 2) {
      if (deepest > 0 && (kb + s - 1) / s * kScaleBlock > deepest) continue;
      const float c = cost_1cta(M, N, K, tn, s);
      if (c < best.cost) best = BlockPlan{0, tn, s, c, deepest};
    }
  }
  if (!aligned) return best;
  for (int s = 1; s <= 8; ++s) {
    if (!block_2cta_splits_ok(K, s) || (s > 1 && deepest > 0 && block_2cta_depth(K, s) > deepest)) continue;
    const float c = cost_2cta(M, N, K, s, s > 1 ? 0 : deepest, true);
    if (c < best.cost) best = BlockPlan{1, 0, s, c, deepest};
  }
  return best;
}

// The fused projection and activation on CTA pairs, or the products and a launch that activates and casts
// (the gated kernel runs no halves). Measured, SwiGLU, one or the other: 64 x 9728 x 2560 22.6 / 14.8 + 3.6 us, 500 x 4096 x
// 1024 10.3 / 10.1 + 5.7, 4097 x 8192 x 2048 100.6 / 100.5 + 41.7. The variant it chooses takes 0.4 % longer than the better
// one in the mean and 9 % at most (67 sizes, rows 12 to 4097). tanh-GELU (11.5 / 10.1 + 7.7 at the second size) adds as
// much to the one as to the other.
bool block_glu_fused(int T, int I, int K, int deepest) {
  return cost_2cta(T, 2 * I, K, 1, deepest, false) <
         block_plan(T, 2 * I, K, true, deepest).cost + 3.5f + 1.16e-6f * T * float(I);
}

size_t block_plan_bytes(const BlockPlan& p, int M, int N) {
  return p.kernel == 1 && p.splits > 1 ? size_t(p.splits) * M * N * 4 : 0;
}

int block_gemm(const BlockPlan& p, const BlockMat& A, const BlockMat& B, void* C, int M, int N, int K,
               long long ldc, int out_fp32, int accumulate, const void* bias, void* ws, int* status,
               cudaStream_t stream) {
  if (p.kernel == 0)
    return block_gemm_1cta(p.tn, p.splits, A, B, C, M, N, K, ldc, out_fp32, accumulate, bias, status, stream);
  if (p.splits == 1)
    return block_gemm_2cta(1, p.deepest, 0, A, B, C, M, N, K, ldc, out_fp32, accumulate, bias, status, stream);
  const long long stride = 1LL * M * N;
  const int rc = block_gemm_2cta(p.splits, 0, stride, A, B, ws, M, N, K, N, 1, 0, nullptr, status, stream);
  if (rc) return rc;
  return block_sum(static_cast<const float*>(ws), p.splits, stride, M, N, C, ldc, out_fp32, accumulate, bias,
                   stream);
}

}  // namespace lb

namespace {
bool aligned_for_pairs(const void* C, int N, long long ldc) {
  return !(N & 7) && !(ldc & 7) && !(reinterpret_cast<uintptr_t>(C) & 15);
}
}  // namespace

// Bytes of temporary storage that lb_gemm_block wants for this product (a 16-byte aligned C).
extern "C" long long lb_gemm_block_bytes(int M, int N, int K, long long ldc) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  return (long long)lb::block_plan_bytes(
      lb::block_plan(M, N, K, aligned_for_pairs(nullptr, N, ldc)), M, N);
}

// C [M, N] (bf16 or fp32, rows ldc elements apart) = A · Bᵀ + bias for A [M, K] and B [N, K] in 8 bits
// (bytes, rows lda / ldb apart, multiples of 16; e5m2 or e4m3) with scale words sa [ceil(K / 512)][rows_sa]
// and sb [..][rows_sb]. accumulate (fp32 only, no bias): C += A · Bᵀ. ws: lb_gemm_block_bytes, 16-byte aligned.
extern "C" int lb_gemm_block(const void* A, const void* B, void* C, int M, int N, int K, long long lda,
                             long long ldb, long long ldc, int a_e5m2, int b_e5m2, const void* sa,
                             long long rows_sa, const void* sb, long long rows_sb, int out_fp32, int accumulate,
                             const void* bias, void* ws, long long ws_bytes, int* status, void* stream_) {
  using namespace lb;
  if (M <= 0 || N <= 0) return 0;
  if (K <= 0) return -4;
  if ((lda & 15) || (ldb & 15) || lda < K || ldb < K || ldc < N || rows_sa < M || rows_sb < N) return -3;
  if (accumulate && (!out_fp32 || bias != nullptr)) return -5;
  const BlockMat a{(uint8_t*)A, lda, (uint32_t*)sa, rows_sa, a_e5m2};
  const BlockMat b{(uint8_t*)B, ldb, (uint32_t*)sb, rows_sb, b_e5m2};
  const BlockPlan p = block_plan(M, N, K, aligned_for_pairs(C, N, ldc));
  if (block_plan_bytes(p, M, N) > size_t(ws_bytes)) return -6;
  return block_gemm(p, a, b, C, M, N, K, ldc, out_fp32, accumulate, bias, ws, status,
                    reinterpret_cast<cudaStream_t>(stream_));
}
