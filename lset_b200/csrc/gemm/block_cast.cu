// Casts from bf16 to 8-bit floats in blocks of 128 with a power-of-two scale each (the format:
// block_scale.cuh), row-major and transposed in one pass.
//
// In place of the per-tensor and per-row casts of fp8_cast.cu where the scales are those of blocks: a block
// lies within a CTA's 128 x 128 tile, so the largest magnitude, the rounding and both layouts come from one
// read, and there is no pass for the maxima.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../common/pdl.h"
#include "../row/glu.cuh"
#include "block_gemm.h"
#include "block_scale.cuh"

namespace lb {
namespace {

using bf16 = __nv_bfloat16;

__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// The bytes of four words of a 4 x 4 block, transposed.
__device__ __forceinline__ void transpose4(uint32_t (&w)[4]) {
  const uint32_t ab0 = __byte_perm(w[0], w[1], 0x5140), ab1 = __byte_perm(w[0], w[1], 0x7362);
  const uint32_t cd0 = __byte_perm(w[2], w[3], 0x5140), cd1 = __byte_perm(w[2], w[3], 0x7362);
  w[0] = __byte_perm(ab0, cd0, 0x5410);
  w[1] = __byte_perm(ab0, cd0, 0x7632);
  w[2] = __byte_perm(ab1, cd1, 0x5410);
  w[3] = __byte_perm(ab1, cd1, 0x7632);
}

// One 8-bit matrix to write: bytes ld apart, scale words as block_scale.cuh lays them out (`rows` words a
// group of four blocks). kb0: block of a row that the first byte belongs to, where only part of the
// columns is written.
struct BlockOut {
  uint8_t* data;
  long long ld;
  uint32_t* scales;
  long long rows;
  int kb0;
};

// Scale byte e of block kb of row r; with the last block of a row, the rest of its word.
__device__ __forceinline__ void store_scale(const BlockOut& o, long long r, int kb, bool last, uint32_t e) {
  kb += o.kb0;
  uint8_t* p = reinterpret_cast<uint8_t*>(o.scales + (kb >> 2) * o.rows + r);
  p[kb & 3] = uint8_t(e);
  if (last)
    for (int k = (kb & 3) + 1; k < 4; ++k) p[k] = uint8_t(kScaleOne);
}

constexpr int kTile = 128;
struct CastSmem {
  uint32_t tile[kTile * kTile / 4];  // [column][four rows]
  uint32_t part[8][64];              // a warp's maxima of its 128 columns, two a word
  uint32_t all[8];
};

// The 128 x 128 tile at (r0, c0) of a matrix [R, C] that the CTA's 256 threads hold in registers: thread
// (rg, cg) = (threadIdx.x / 16, % 16) has rows rg * 4 + 64 u + i, columns cg * 8 .. cg * 8 + 7 in v[u][i]
// (zeros outside the matrix). TILED: one scale for the tile; else `out` has one for each row and `out_t`
// for each column. Either may be absent (data null).
//
// Magnitudes are compared as integers (bf16 bits without the sign), two at a time, which also lets NaN and
// infinities through to the top.
template <int TILED, int E5M2>
__device__ __forceinline__ void cast_tile(const uint4 (&v)[2][4], CastSmem& sm, int r0, int c0, int R, int C,
                                          const BlockOut& out, const BlockOut& out_t) {
  const int cg = threadIdx.x & 15, rq = threadIdx.x >> 4, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int c = c0 + cg * 8;
  constexpr uint32_t kAbs = 0x7fff7fffu;
  uint32_t col[4] = {0u, 0u, 0u, 0u};   // maxima of the thread's eight columns
  uint32_t row[4];                      // of its eight rows: rows i (low half) and i + 64
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t m[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const uint32_t w[4] = {v[u][i].x & kAbs, v[u][i].y & kAbs, v[u][i].z & kAbs, v[u][i].w & kAbs};
#pragma unroll
      for (int j = 0; j < 4; ++j) col[j] = __vmaxu2(col[j], w[j]);
      m[u] = __vmaxu2(__vmaxu2(w[0], w[1]), __vmaxu2(w[2], w[3]));
      m[u] = __vmaxu2(m[u], m[u] >> 16);
    }
    row[i] = __byte_perm(m[0], m[1], 0x5410);
  }
  uint32_t tile_max = 0u;
  if (TILED) {
    uint32_t m = __vmaxu2(__vmaxu2(col[0], col[1]), __vmaxu2(col[2], col[3]));
    m = max(m & 0xffffu, m >> 16);
    m = __reduce_max_sync(0xffffffffu, m);
    if (lane == 0) sm.all[warp] = m;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 8; ++k) tile_max = max(tile_max, sm.all[k]);
  } else {
    if (out.data != nullptr)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) row[i] = __vmaxu2(row[i], __shfl_xor_sync(0xffffffffu, row[i], o));
    if (out_t.data != nullptr) {
#pragma unroll
      for (int j = 0; j < 4; ++j) col[j] = __vmaxu2(col[j], __shfl_xor_sync(0xffffffffu, col[j], 16));
      if (lane < 16)
        *reinterpret_cast<uint4*>(&sm.part[warp][cg * 4]) = make_uint4(col[0], col[1], col[2], col[3]);
      __syncthreads();
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint4 p = *reinterpret_cast<const uint4*>(&sm.part[k][cg * 4]);
        col[0] = __vmaxu2(col[0], p.x);
        col[1] = __vmaxu2(col[1], p.y);
        col[2] = __vmaxu2(col[2], p.z);
        col[3] = __vmaxu2(col[3], p.w);
      }
    }
  }
  const uint32_t tile_e = block_scale_byte<E5M2>(tile_max);
  const float tile_inv = block_inverse(tile_e);
  const bool tile_ok = block_is_finite(tile_max);

  if (out.data != nullptr) {
    const int kb = c0 / kTile;
    const bool last = c0 + kTile >= C;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = r0 + rq * 4 + u * 64 + i;
        const uint32_t top = TILED ? tile_max : (row[i] >> (16 * u)) & 0xffffu;
        const uint32_t e = TILED ? tile_e : block_scale_byte<E5M2>(top);
        const bool ok = TILED ? tile_ok : block_is_finite(top);
        const float s = TILED ? tile_inv : block_inverse(e);
        if (r < R) {
          if (c < C) {
            const uint4& q = v[u][i];
            uint2 b = make_uint2(cast4<E5M2>(bf16_lo(q.x) * s, bf16_hi(q.x) * s, bf16_lo(q.y) * s, bf16_hi(q.y) * s),
                                 cast4<E5M2>(bf16_lo(q.z) * s, bf16_hi(q.z) * s, bf16_lo(q.w) * s, bf16_hi(q.w) * s));
            if (!ok) b = make_uint2(0x7f7f7f7fu, 0x7f7f7f7fu);
            *reinterpret_cast<uint2*>(out.data + (long long)r * out.ld + c) = b;
          }
          if (cg == 0) store_scale(out, r, kb, last, ok ? e : kScaleOne);
        }
      }
  }
  if (out_t.data == nullptr) return;
  uint32_t ce[8];
  float cs[8];
  bool cok[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t top = TILED ? tile_max : (col[j / 2] >> (16 * (j & 1))) & 0xffffu;
    ce[j] = TILED ? tile_e : block_scale_byte<E5M2>(top);
    cs[j] = TILED ? tile_inv : block_inverse(ce[j]);
    cok[j] = TILED ? tile_ok : block_is_finite(top);
  }
  if (rq == 0 && c < C) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      store_scale(out_t, c + j, r0 / kTile, r0 + kTile >= R, cok[j] ? ce[j] : kScaleOne);
  }
  // Word `rg` (four rows) of a column of group cg lies at rg ^ 2 cg: the words that a warp writes at a time
  // are in different banks, and four of a column stay together for the 16-byte reads.
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int rg = rq + u * 16;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      uint32_t q[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t a = k ? v[u][i].z : v[u][i].x, b = k ? v[u][i].w : v[u][i].y;
        q[i] = cast4<E5M2>(bf16_lo(a) * cs[4 * k], bf16_hi(a) * cs[4 * k + 1], bf16_lo(b) * cs[4 * k + 2],
                          bf16_hi(b) * cs[4 * k + 3]);
      }
      transpose4(q);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        sm.tile[(cg * 8 + k * 4 + j) * 32 + (rg ^ (2 * cg))] = cok[4 * k + j] ? q[j] : 0x7f7f7f7fu;
    }
  }
  __syncthreads();
  // row c of out_t holds column c of the tile: 16 rows of it a piece
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int tc = (threadIdx.x >> 3) + k * 32, m = threadIdx.x & 7, g = tc >> 3;
    uint4 w = *reinterpret_cast<const uint4*>(sm.tile + tc * 32 + 4 * (m ^ (g >> 1)));
    if (g & 1) w = make_uint4(w.z, w.w, w.x, w.y);
    if (c0 + tc < C && r0 + m * 16 < out_t.ld)
      *reinterpret_cast<uint4*>(out_t.data + (long long)(c0 + tc) * out_t.ld + r0 + m * 16) = w;
  }
}

__device__ __forceinline__ void load_tile(uint4 (&v)[2][4], const bf16* __restrict__ x, long long ldx, int r0,
                                          int c0, int R, int C) {
  const int c = c0 + (threadIdx.x & 15) * 8;
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = r0 + (threadIdx.x >> 4) * 4 + u * 64 + i;
      v[u][i] = r < R && c < C ? *reinterpret_cast<const uint4*>(x + r * ldx + c) : make_uint4(0u, 0u, 0u, 0u);
    }
}

// colsum (where it is wanted: the gradient of a bias): the tile's column sums to row r0 / 128 of a matrix
// [.., C], always added in the same order.
template <int TILED, int E5M2>
__global__ void __launch_bounds__(256)
    block_cast_kernel(const bf16* __restrict__ x, int R, int C, long long ldx, BlockOut out, BlockOut out_t,
                      float* __restrict__ colsum, int tiles_c) {
  __shared__ __align__(16) CastSmem sm;
  pdl_wait();
  pdl_trigger();
  const int rt = blockIdx.x / tiles_c;
  const int r0 = rt * kTile, c0 = (blockIdx.x - rt * tiles_c) * kTile;
  uint4 v[2][4];
  load_tile(v, x, ldx, r0, c0, R, C);
  if (!TILED && colsum != nullptr) {
    float s[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      s[j] = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint4& q = v[k / 4][k % 4];
        const uint32_t w = j / 2 == 0 ? q.x : (j / 2 == 1 ? q.y : (j / 2 == 2 ? q.z : q.w));
        s[j] += j & 1 ? bf16_hi(w) : bf16_lo(w);
      }
      s[j] += __shfl_xor_sync(0xffffffffu, s[j], 16);
    }
    float* part = reinterpret_cast<float*>(sm.tile);   // [8 warps][128 columns]
    const int warp = threadIdx.x >> 5, cg = threadIdx.x & 15;
    if ((threadIdx.x & 31) < 16) {
#pragma unroll
      for (int j = 0; j < 8; ++j) part[warp * kTile + cg * 8 + j] = s[j];
    }
    __syncthreads();
    if (threadIdx.x < kTile && c0 + threadIdx.x < C) {
      float t = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) t += part[k * kTile + threadIdx.x];
      colsum[(long long)rt * C + c0 + threadIdx.x] = t;
    }
    __syncthreads();
  }
  cast_tile<TILED, E5M2>(v, sm, r0, c0, R, C, out, out_t);
}

// h = act(gate) * up of [T, I] matrices (rows ld elements apart), rounded to bf16 as the separate activation
// rounds it, in blocks of a row.
template <int KIND>
__global__ void __launch_bounds__(256)
    block_glu_fwd_kernel(const bf16* __restrict__ gate, const bf16* __restrict__ up, long long ld, int T, int I,
                         BlockOut h, int tiles_c) {
  __shared__ __align__(16) CastSmem sm;
  pdl_wait();
  pdl_trigger();
  const int rt = blockIdx.x / tiles_c;
  const int r0 = rt * kTile, c0 = (blockIdx.x - rt * tiles_c) * kTile;
  uint4 g[2][4], u[2][4];
  load_tile(g, gate, ld, r0, c0, T, I);
  load_tile(u, up, ld, r0, c0, T, I);
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) g[k][i] = glu_fwd8<KIND>(g[k][i], u[k][i]);
  cast_tile<0, 0>(g, sm, r0, c0, T, I, h, BlockOut{});
}

// The way back: from dh, gate and up the gradients of gate and up (rounded to bf16) in blocks of a row (`d`
// [T, 2 I], gate columns first) and of 128 tokens (`d_t` [2 I, T]), and h once more, in blocks of 128 tokens
// (`h_t` [I, T]): the operands of the input gradient and of both weight gradients from one read. I is a
// multiple of 128, so that no block holds columns of both.
template <int KIND>
__global__ void __launch_bounds__(256, 2)
    block_glu_bwd_kernel(const bf16* __restrict__ dh, long long ld_dh, const bf16* __restrict__ gate,
                         const bf16* __restrict__ up, long long ld, int T, int I, BlockOut d, BlockOut d_t,
                         BlockOut h_t, int tiles_c) {
  __shared__ __align__(16) CastSmem sm;
  pdl_wait();
  pdl_trigger();
  const int rt = blockIdx.x / tiles_c;
  const int r0 = rt * kTile, c0 = (blockIdx.x - rt * tiles_c) * kTile;
  uint4 g[2][4], u[2][4], x[2][4];
  load_tile(g, gate, ld, r0, c0, T, I);
  load_tile(u, up, ld, r0, c0, T, I);
  load_tile(x, dh, ld_dh, r0, c0, T, I);
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint4 h = glu_fwd8<KIND>(g[k][i], u[k][i]);
      glu_bwd8<KIND>(g[k][i], u[k][i], x[k][i], g[k][i], u[k][i]);
      x[k][i] = h;
    }
  cast_tile<0, 0>(g, sm, r0, c0, T, 2 * I, d, d_t);
  __syncthreads();
  cast_tile<0, 0>(u, sm, r0, I + c0, T, 2 * I, d, d_t);
  if (h_t.data == nullptr) return;
  __syncthreads();
  cast_tile<0, 0>(x, sm, r0, c0, T, I, BlockOut{}, h_t);
}

// out [rows, cols] = (out +) sums of P matrices, part p at p * stride, each value in the order of p.
template <typename OutT>
__global__ void __launch_bounds__(256)
    block_sum_kernel(const float* __restrict__ part, int P, long long stride, int rows, int cols, OutT* out,
                     long long ldo, int accumulate) {
  pdl_wait();
  pdl_trigger();
  const int vecs = cols / 4;
  const long long n = 1LL * rows * vecs;
  for (long long i = 1LL * blockIdx.x * blockDim.x + threadIdx.x; i < n; i += 1LL * gridDim.x * blockDim.x) {
    const long long r = i / vecs;
    const int c = int(i - r * vecs) * 4;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int p = 0; p < P; ++p) {
      const float4 v = *reinterpret_cast<const float4*>(part + p * stride + 4 * i);
      s = make_float4(s.x + v.x, s.y + v.y, s.z + v.z, s.w + v.w);
    }
    OutT* o = out + r * ldo + c;
    if constexpr (sizeof(OutT) == 2) {
      *reinterpret_cast<uint2*>(o) = make_uint2(pack_bf16x2(s.x, s.y), pack_bf16x2(s.z, s.w));
    } else {
      float4* o4 = reinterpret_cast<float4*>(o);
      if (accumulate) {
        const float4 v = *o4;
        s = make_float4(v.x + s.x, v.y + s.y, v.z + s.z, v.w + s.w);
      }
      *o4 = s;
    }
  }
}

BlockOut block_out(const BlockMat& m, int kb0 = 0) { return BlockOut{m.data, m.ld, m.scales, m.rows_s, kb0}; }

// CTAs of the tiles of [R, C]; 0 where there are too many.
unsigned cast_grid(int R, int C) {
  const long long tiles = 1LL * ((C + kTile - 1) / kTile) * ((R + kTile - 1) / kTile);
  return tiles > 0x7fffffffLL ? 0u : unsigned(tiles);
}

bool fits(const BlockMat& m, long long rows, long long cols) {
  return m.data == nullptr || (!(m.ld & 15) && m.ld >= cols && m.rows_s >= rows && m.scales != nullptr);
}

}  // namespace

int block_cast(const void* x, int R, int C, long long ldx, int tiled, int e5m2, const BlockMat& out,
               const BlockMat& out_t, int kb0_t, float* colsum, cudaStream_t stream) {
  if (R <= 0 || C <= 0) return 0;
  if ((C & 7) || (ldx & 7) || (reinterpret_cast<uintptr_t>(x) & 15)) return -3;
  if (!fits(out, R, C) || !fits(out_t, C, R) || kb0_t < 0 || (kb0_t > 0 && (R % kTile))) return -3;
  if (colsum != nullptr && tiled) return -5;
  const unsigned grid = cast_grid(R, C);
  if (grid == 0) return -3;
  auto kern = tiled ? (e5m2 ? block_cast_kernel<1, 1> : block_cast_kernel<1, 0>)
                    : (e5m2 ? block_cast_kernel<0, 1> : block_cast_kernel<0, 0>);
  return launch_pdl(kern, dim3(grid), dim3(256), 0, stream, pdl_enabled(4LL * R * C), 1,
                    static_cast<const bf16*>(x), R, C, ldx, block_out(out), block_out(out_t, kb0_t), colsum,
                    (C + kTile - 1) / kTile);
}

// h = act(gate) * up of [T, I] (rows ld elements apart; I a multiple of 128) in blocks of a row. kind: 0 = SwiGLU,
// 1 = GeGLU (tanh).
int block_glu_fwd(int kind, const void* gate, const void* up, long long ld, int T, int I, const BlockMat& out,
                  cudaStream_t stream) {
  if (T <= 0 || I <= 0) return 0;
  if ((I % kTile) || (ld & 7) || !fits(out, T, I)) return -3;
  const unsigned grid = cast_grid(T, I);
  if (grid == 0) return -3;
  return launch_pdl(kind == kSwiglu ? block_glu_fwd_kernel<kSwiglu> : block_glu_fwd_kernel<kGeglu>, dim3(grid),
                    dim3(256), 0, stream, pdl_enabled(5LL * T * I), 1, static_cast<const bf16*>(gate),
                    static_cast<const bf16*>(up), ld, T, I, block_out(out), I / kTile);
}

// From dh [T, I], gate and up: `d` [T, 2 I] and `d_t` [2 I, T], the gradients of gate and up, and `h_t` [I, T].
int block_glu_bwd(int kind, const void* dh, long long ld_dh, const void* gate, const void* up, long long ld,
                  int T, int I, const BlockMat& d, const BlockMat& d_t, const BlockMat& h_t,
                  cudaStream_t stream) {
  if (T <= 0 || I <= 0) return 0;
  if ((I % kTile) || (ld & 7) || (ld_dh & 7)) return -3;
  if (!fits(d, T, 2LL * I) || !fits(d_t, 2LL * I, T) || !fits(h_t, I, T)) return -3;
  const unsigned grid = cast_grid(T, I);
  if (grid == 0) return -3;
  return launch_pdl(kind == kSwiglu ? block_glu_bwd_kernel<kSwiglu> : block_glu_bwd_kernel<kGeglu>, dim3(grid),
                    dim3(256), 0, stream, pdl_enabled(11LL * T * I), 1, static_cast<const bf16*>(dh), ld_dh,
                    static_cast<const bf16*>(gate), static_cast<const bf16*>(up), ld, T, I, block_out(d),
                    block_out(d_t), block_out(h_t), I / kTile);
}

// cols a multiple of 4; part, stride and out 16-byte aligned (out: 8 bytes in bf16).
int block_sum(const float* part, int P, long long stride, int rows, int cols, void* out, long long ldo,
              int out_fp32, int accumulate, cudaStream_t stream) {
  if (rows <= 0 || cols <= 0) return 0;
  if ((cols & 3) || (stride & 3) || (ldo & 3) || (accumulate && !out_fp32)) return -3;
  const long long n = 1LL * rows * (cols / 4);
  const unsigned grid = unsigned(n > 148LL * 8 * 256 ? 148 * 8 : (n + 255) / 256);
  const bool pdl = pdl_enabled(4LL * P * rows * cols);
  return out_fp32 ? launch_pdl(block_sum_kernel<float>, dim3(grid), dim3(256), 0, stream, pdl, 1, part, P, stride,
                               rows, cols, static_cast<float*>(out), ldo, accumulate)
                  : launch_pdl(block_sum_kernel<bf16>, dim3(grid), dim3(256), 0, stream, pdl, 1, part, P, stride,
                               rows, cols, static_cast<bf16*>(out), ldo, 0);
}

}  // namespace lb

// x [R, C] (bf16, rows ldx elements apart; C and ldx multiples of 8, x 16-byte aligned) in 8 bits: `out` [R, C]
// (rows ldo bytes apart, a multiple of 16) and / or `out_t` [C, R] (rows ldt bytes, a multiple of 16; zeros
// behind R up to the next 128th column). tiled: a scale for each 128 x 128 block; else `out` has one for each
// row and 128 columns and `out_t` for each column of x and 128 rows. scales / scales_t: words
// [ceil(C / 512)][rows_s] and [ceil(R / 512)][rows_st], rows_s >= R and rows_st >= C. kb0_t > 0: out_t points
// at column 128 kb0_t of a longer matrix, whose first scales are at scales_t (R a multiple of 128 then).
extern "C" int lb_block_cast(const void* x, int R, int C, long long ldx, int tiled, int e5m2, void* out,
                             long long ldo, void* scales, long long rows_s, void* out_t, long long ldt,
                             void* scales_t, long long rows_st, int kb0_t, void* stream_) {
  return lb::block_cast(x, R, C, ldx, tiled, e5m2,
                        lb::BlockMat{static_cast<uint8_t*>(out), ldo, static_cast<uint32_t*>(scales), rows_s, e5m2},
                        lb::BlockMat{static_cast<uint8_t*>(out_t), ldt, static_cast<uint32_t*>(scales_t), rows_st, e5m2},
                        kb0_t, nullptr, reinterpret_cast<cudaStream_t>(stream_));
}
