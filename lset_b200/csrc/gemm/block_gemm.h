// Block-scaled 8-bit products for callers within the library (gemm_block.cu, gemm_block_2cta.cu,
// block_cast.cu, block_layers.cu).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace lb {

// An 8-bit matrix [rows, cols]: bytes, rows ld apart, and scale words, `rows_s` of them a group of four
// blocks (block_scale.cuh).
struct BlockMat {
  uint8_t* data;
  long long ld;
  uint32_t* scales;
  long long rows_s;
  int e5m2;
};

// How a product runs: kernel 0 is the one-CTA kernel with tiles of 128 x tn and the contraction split over
// clusters of `splits`; kernel 1 the pair kernel, its contraction split into `splits` fp32 products that a
// second launch adds up.
struct BlockPlan {
  int kernel, tn, splits;
  float cost;   // modelled, us
  int deepest;
};
// How deep a sum in tensor memory may be (0: as deep as the product). The tensor cores cut a running sum to 24 bits after
// every 32 of depth instead of rounding it: errors of one sign, 1.4 x those of fp32 sums 768 deep, 2 x at 2048 and 5 x at
// 8192. A product whose values are rounded to bf16 and then to 8 bits passes them on as whole steps of those (2^-4
// of a value), so a training step's gate, up and dh are sums of parts this deep, added in fp32.
enum { kDeepestSum = 1024 };
// aligned: C may be written in pieces of 16 bytes, which the pair kernel does. deepest > 0: for a bf16 C, aligned, without
// bias.
BlockPlan block_plan(int M, int N, int K, bool aligned, int deepest = 0);
// Whether block_gemm_glu is the faster way to the gated projections of T rows.
bool block_glu_fused(int T, int I, int K, int deepest);
// Bytes of temporary storage of a plan.
size_t block_plan_bytes(const BlockPlan& p, int M, int N);

// C [M, N] = or += A · Bᵀ + bias; ws: block_plan_bytes.
int block_gemm(const BlockPlan& p, const BlockMat& A, const BlockMat& B, void* C, int M, int N, int K,
               long long ldc, int out_fp32, int accumulate, const void* bias, void* ws, int* status,
               cudaStream_t stream);

// The product of few rows whose A is bf16 still (rows ldx elements apart) and cast in the kernel, where
// block_casts_itself says so.
bool block_casts_itself(const BlockPlan& p, int M, int K);
int block_gemm_cast(const BlockPlan& p, const void* x, long long ldx, const BlockMat& B, void* C, int M, int N, int K,
                    long long ldc, int out_fp32, const void* bias, int* status, cudaStream_t stream);

int block_gemm_1cta(int tn, int splits, const BlockMat& A, const BlockMat& B, void* C, int M, int N, int K,
                    long long ldc, int out_fp32, int accumulate, const void* bias, int* status,
                    cudaStream_t stream);
int block_gemm_2cta(int splits, int deepest, long long split_stride, const BlockMat& A, const BlockMat& B, void* C, int M,
                    int N, int K, long long ldc, int out_fp32, int accumulate, const void* bias, int* status,
                    cudaStream_t stream);
// Whether `splits` divides the contraction into that many parts (whole groups of scale words each); their depth; how many
// sums a contraction is.
bool block_2cta_splits_ok(int K, int splits);
int block_2cta_depth(int K, int splits);
int block_2cta_sums(int K, int deepest);
// h = act(A · Wgᵀ) * (A · Wuᵀ), cast; Wu's rows follow Wg's scale words in one group. See gemm_block_2cta.cu.
int block_gemm_glu(int kind, int deepest, const BlockMat& A, const BlockMat& Wg, const BlockMat& Wu, int M, int I, int K,
                   void* gate, void* up, long long ld_gu, const BlockMat& h, int* status, cudaStream_t stream);

// block_cast.cu. Casts of x [R, C] as rows and / or transposed (data null: not wanted). colsum: fp32
// [ceil(R / 128)][C], the column sums of each 128 rows of x (null: not wanted).
int block_cast(const void* x, int R, int C, long long ldx, int tiled, int e5m2, const BlockMat& out,
               const BlockMat& out_t, int kb0_t, float* colsum, cudaStream_t stream);
// The same column sums of an fp32 matrix by themselves.
int block_colsum(const float* x, int R, int C, long long ldx, float* colsum, cudaStream_t stream);
// Up to kMaxCasts casts to e4m3 in one launch (where both layouts of all are wanted).
enum { kMaxCasts = 4 };
struct BlockCast {
  const void* x;
  int R, C;
  long long ldx;
  int tiled;
  BlockMat out, out_t;
  int kb0_t;
  bool fill_t;   // out_t's columns end here (not where another cast of the same launch writes on)
};
int block_casts(const BlockCast* jobs, int n, cudaStream_t stream);
int block_glu_fwd(int kind, const void* gate, const void* up, long long ld, int T, int I, const BlockMat& out,
                  cudaStream_t stream);
int block_glu_bwd(int kind, const void* dh, long long ld_dh, const void* gate, const void* up, long long ld,
                  int T, int I, const BlockMat& d, const BlockMat& d_t, const BlockMat& h_t,
                  cudaStream_t stream);
// out [rows, cols] (bf16 or fp32, rows ldo apart) = or += the sum of P matrices [rows, cols] of fp32, in order, + bias.
int block_sum(const float* part, int P, long long stride, int rows, int cols, void* out, long long ldo,
              int out_fp32, int accumulate, const void* bias, cudaStream_t stream);

}  // namespace lb
