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
#include <cuda_bf16.h>

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

template <int TN>
struct Cfg {
  static constexpr int kStages = TN <= 16 ? 6 : (TN <= 64 ? (TN <= 32 ? 5 : 4) : 3);
  static constexpr int kP = kBP * 128, kQ = TN * 128;    // bytes of a stage
  static constexpr int kAcc = TN < 32 ? 32 : TN;         // columns of the accumulator in TMEM
  static constexpr int kCols = TN <= 32 ? 64 : (TN <= 64 ? 128 : 256);
  static constexpr int kSmem = kStages * (kP + kQ) + 1024 + 256;
  static_assert(kAcc + 8 * kSlots <= kCols, "");
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
  int tiles_m;
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
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr, uint32_t rank) {
  uint32_t at;
  float v;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}

__device__ __forceinline__ void store_c(const BlockArgs& g, int m, int n, float v, float bias) {
  if (g.out_fp32) {
    float* p = static_cast<float*>(g.C) + m * g.ldc + n;
    *p = v + (g.accumulate ? *p : bias);
  } else {
    static_cast<__nv_bfloat16*>(g.C)[m * g.ldc + n] = __float2bfloat16(v + bias);
  }
}

template <int TN>
__global__ void __launch_bounds__(kThreads1, 2)
    gemm_block_kernel(const __grid_constant__ CUtensorMap tmP, const __grid_constant__ CUtensorMap tmQ,
                      BlockArgs g) {
  using F = Cfg<TN>;
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
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(&sfull[s], 4);
      mbar_init(&sempty[s], 1);
    }
    mbar_init(tfull, 1);
    mbar_fence_init();
    tma_prefetch_desc(&tmP);
    tma_prefetch_desc(&tmQ);
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
      const uint32_t bytes = F::kP + g.q_rows * 128;
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
        tma_load_2d(sp + F::kP, &tmQ, &full[stage], kb * kScaleBlock, m0);
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
        const uint32_t idesc = umma_idesc_block(kBP, TN, g.b_e5m2, g.a_e5m2, kb & 3);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          umma_block(tmem, umma_smem_desc(sp + 32 * k, 16, 1024), umma_smem_desc(sq + 32 * k, 16, 1024), idesc,
                     scales, scales + 4, kb > kb0 || k > 0);
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
          w[4 + c] = c * 32 < TN && m < g.M ? g.sa[(g0 + i) * g.rows_sa + m] : 0x7f7f7f7fu;
        }
      };
      fetch(0);
      for (int i = 0; i < groups; ++i) {
        const int slot = i % kSlots;
        // (all lanes take part in the store, and may see a bounded wait end differently)
        if (!__all_sync(0xffffffffu, mbar_wait(&sempty[slot], ((i / kSlots) & 1) ^ 1u))) {
          ok = false;
          break;
        }
        tmem_st_32x32b_x8(tmem + lanes + F::kAcc + 8 * slot, w);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sfull[slot]);
        if (i + 1 < groups) fetch(i + 1);
      }
      ok = ok && __all_sync(0xffffffffu, mbar_wait(tfull, 0));
      if (!ok) report_status(g.status, kStatusTimeoutEpilogue);
      tc_fence_after();
    }
    const int n = n0 + q * 32 + lane;
    const float bias = g.bias != nullptr && n < g.N ? __bfloat162float(g.bias[n]) : 0.f;
    float* part = reinterpret_cast<float*>(smem);
#pragma unroll 1
    for (int c = 0; c < TN / 16; ++c) {
      uint32_t r[16];
      if (kb1 > kb0 && ok) {
        tmem_ld_32x32b_x16(tmem + lanes + 16 * c, r);
        tmem_ld_wait();
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) r[j] = 0u;
      }
      if (splits > 1) {
#pragma unroll
        for (int j = 0; j < 16; ++j) part[(16 * c + j) * kBP + q * 32 + lane] = __uint_as_float(r[j]);
      } else if (n < g.N) {
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (m0 + 16 * c + j < g.M) store_c(g, m0 + 16 * c + j, n, __uint_as_float(r[j]), bias);
      }
    }
    tc_fence_before();
  }
  if (splits > 1) {
    cluster_sync_block();
    if (warp >= 2) {
      const int p = (warp & 3) * 32 + lane, n = n0 + p;
      if (n < g.N) {
        const float bias = g.bias != nullptr ? __bfloat162float(g.bias[n]) : 0.f;
        for (int j = rank; j < TN && m0 + j < g.M; j += splits) {
          const uint32_t at = smem_u32(smem) + (j * kBP + p) * 4;
          float v = 0.f;
          for (int s = 0; s < splits; ++s) v += ld_cluster_f32(at, s);
          store_c(g, m0 + j, n, v, bias);
        }
      }
    }
    cluster_sync_block();   // nobody's sums go before they are read
  }
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, F::kCols);
}

constexpr int kMaxDevices = 64;

template <int TN>
int launch_block(const CUtensorMap& tmP, const CUtensorMap& tmQ, const BlockArgs& g, long long tiles,
                 int splits, cudaStream_t stream) {
  static bool configured[kMaxDevices] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return -10;
  if (!configured[dev]) {
    if (cudaFuncSetAttribute(gemm_block_kernel<TN>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             Cfg<TN>::kSmem) != cudaSuccess)
      return -10;
    configured[dev] = true;
  }
  return launch_pdl(gemm_block_kernel<TN>, dim3(unsigned(tiles * splits)), dim3(kThreads1), Cfg<TN>::kSmem,
                    stream, pdl_enabled(), splits, tmP, tmQ, g);
}

}  // namespace

int block_gemm_1cta(int tn, int splits, const BlockMat& A, const BlockMat& B, void* C, int M, int N, int K,
                    long long ldc, int out_fp32, int accumulate, const void* bias, int* status,
                    cudaStream_t stream) {
  const int kb = (K + kScaleBlock - 1) / kScaleBlock;
  if (splits < 1 || splits > 8 || splits > kb) return -5;
  BlockArgs g{};
  g.M = M;
  g.N = N;
  g.K = K;
  g.sa = A.scales;
  g.sb = B.scales;
  g.rows_sa = A.rows_s;
  g.rows_sb = B.rows_s;
  g.C = C;
  g.ldc = ldc;
  g.out_fp32 = out_fp32;
  g.accumulate = accumulate;
  g.bias = static_cast<const __nv_bfloat16*>(bias);
  g.a_e5m2 = A.e5m2 ? 1 : 0;
  g.b_e5m2 = B.e5m2 ? 1 : 0;
  g.q_rows = M < tn ? M : tn;
  g.tiles_m = (M + tn - 1) / tn;
  g.status = status;
  const long long tiles = 1LL * g.tiles_m * ((N + kBP - 1) / kBP);
  if (tiles * splits > 0x7fffffffLL) return -3;
  CUtensorMap tmP, tmQ;
  int rc = make_tmap_2d(&tmP, B.data, 1, (uint64_t)K, (uint64_t)N, (uint64_t)B.ld, 128, kBP, true);
  if (rc) return rc;
  rc = make_tmap_2d(&tmQ, A.data, 1, (uint64_t)K, (uint64_t)M, (uint64_t)A.ld, 128, uint32_t(g.q_rows), true);
  if (rc) return rc;
  switch (tn) {
    case 16: return launch_block<16>(tmP, tmQ, g, tiles, splits, stream);
    case 32: return launch_block<32>(tmP, tmQ, g, tiles, splits, stream);
    case 64: return launch_block<64>(tmP, tmQ, g, tiles, splits, stream);
    case 128: return launch_block<128>(tmP, tmQ, g, tiles, splits, stream);
  }
  return -5;
}

BlockPlan block_plan(int M, int N, int K, int out_fp32, int accumulate, bool bias, bool aligned) {
  if (aligned && 1LL * ((M + 255) / 256) * ((N + 255) / 256) >= 40) return BlockPlan{1, 0, 1};
  const int tn = M <= 16 ? 16 : (M <= 32 ? 32 : (M <= 64 ? 64 : 128));
  const long long tiles = 1LL * ((M + tn - 1) / tn) * ((N + kBP - 1) / kBP);
  const int kb = (K + kScaleBlock - 1) / kScaleBlock;
  int splits = 1;
  while (splits < 8 && tiles * splits * 2 <= 2 * 148 && kb >= 4 * splits) splits *= 2;
  return BlockPlan{0, tn, splits};
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
    return block_gemm_2cta(1, 0, A, B, C, M, N, K, ldc, out_fp32, accumulate, bias, status, stream);
  const long long stride = 1LL * M * N;
  const int rc = block_gemm_2cta(p.splits, stride, A, B, ws, M, N, K, N, 1, 0, nullptr, status, stream);
  if (rc) return rc;
  return block_sum(static_cast<const float*>(ws), p.splits, stride, M, N, C, ldc, out_fp32, accumulate, stream);
}

}  // namespace lb

namespace {
bool aligned_for_pairs(const void* C, int N, long long ldc) {
  return !(N & 7) && !(ldc & 7) && !(reinterpret_cast<uintptr_t>(C) & 15);
}
}  // namespace

// Bytes of temporary storage that lb_gemm_block wants for this product (a 16-byte aligned C).
extern "C" long long lb_gemm_block_bytes(int M, int N, int K, long long ldc, int out_fp32, int accumulate,
                                         int bias) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  return (long long)lb::block_plan_bytes(
      lb::block_plan(M, N, K, out_fp32, accumulate, bias != 0, aligned_for_pairs(nullptr, N, ldc)), M, N);
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
  const BlockPlan p = block_plan(M, N, K, out_fp32, accumulate, bias != nullptr, aligned_for_pairs(C, N, ldc));
  if (block_plan_bytes(p, M, N) > size_t(ws_bytes)) return -6;
  return block_gemm(p, a, b, C, M, N, K, ldc, out_fp32, accumulate, bias, ws, status,
                    reinterpret_cast<cudaStream_t>(stream_));
}
