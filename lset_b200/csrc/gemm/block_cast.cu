// Casts from bf16 to 8-bit floats in blocks of 128 with a power-of-two scale each (the format:
// block_scale.cuh), row-major and transposed in one pass.
//
// In place of the per-tensor and per-row casts of fp8_cast.cu where the scales are those of blocks: a block
// lies within a CTA's 128 x 128 tile, so the largest magnitude, the rounding and both layouts come from one
// read, and there is no pass for the maxima.
// Measured: 16384 x 4096 in both layouts 46 us (5.8 TB/s, 0.89 of copy bandwidth; with a scale and an unpacking for each
// output, and every thread joining the warps' maxima, 62), the gated backward of 8192 x 4864 112 us (3.9 TB/s).
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../common/pdl.h"
#include "../common/row.cuh"
#include "block_gemm.h"
#include "block_glu.cuh"
#include "block_scale.cuh"

namespace lb {
namespace {

using bf16 = __nv_bfloat16;
constexpr int kMaxDevices = 64;

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
// columns is written; fill: the last block written is the row's last, and the rest of its word is filled.
struct BlockOut {
  uint8_t* data;
  long long ld;
  uint32_t* scales;
  long long rows;
  int kb0;
  bool fill;
};

// Scale byte e of block kb of row r; with the last block of a row, the rest of its word.
__device__ __forceinline__ void store_scale(const BlockOut& o, long long r, int kb, bool last, uint32_t e) {
  kb += o.kb0;
  uint8_t* p = reinterpret_cast<uint8_t*>(o.scales + (kb >> 2) * o.rows + r);
  p[kb & 3] = uint8_t(e);
  if (last && o.fill)
    for (int k = (kb & 3) + 1; k < 4; ++k) p[k] = uint8_t(kScaleOne);
}

constexpr int kTile = 128;
enum { kRows = 1, kCols = 2 };

// Shared memory of A tiles that are cast together.
template <int A>
struct CastSmem {
  uint32_t tile[A][kTile * kTile / 4];   // [column][four rows], bytes of the transposed copies
  uint32_t part[A][16][64];              // a warp's maxima of its 128 columns, two a word
  float2 cols[A][64];                    // what the columns are multiplied by
  uint32_t all[16];
};

// The 128 x 128 tile at (r0, c0) of a matrix [R, C] that the CTA's 512 / U threads hold in registers: thread
// (rq, cg) = (threadIdx.x / 16, % 16) has rows rq * 4 + 64 u + i, columns cg * 8 .. cg * 8 + 7 in v[u][i]
// (zeros outside the matrix). WANT kRows: to `out`, kCols: transposed to `out_t`. TILED: one scale for the
// tile; else `out` has one for each row and `out_t` for each column.
//
// Magnitudes are compared as integers (bf16 bits without the sign), two at a time, which also lets NaN and
// infinities through to the top. Bound by issued instructions before memory, so a value is unpacked once for both
// layouts and scaled two at a time, a lane stores one scale, and 64 threads join the warps' column maxima for all.
// The steps of a cast are apart, so that tiles cast together (the gated backward's three) share their barriers:
// maxima, barrier, join_cols, barrier, write, barrier, copy_cols.
template <int E5M2, int WANT, int U>
struct Cast {
  static constexpr int kWarps = 16 / U, kMine = 4 * U, kPairs = kMine / 2;   // a thread's rows; rows p, p + kPairs a word
  static constexpr uint32_t kAbs = 0x7fff7fffu;

  // rs: what the thread's rows are multiplied by (their scales are stored); the columns' maxima go to `part`.
  static __device__ __forceinline__ void maxima(const uint4 (&v)[U][4], uint32_t (&part)[16][64], float (&rs)[kMine],
                                                int r0, int c0, int R, int C, const BlockOut& out) {
    const int cg = threadIdx.x & 15, rq = threadIdx.x >> 4, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t col[4] = {0u, 0u, 0u, 0u}, m[kMine];
#pragma unroll
    for (int p = 0; p < kMine; ++p) {
      const uint4& q = v[p / 4][p % 4];
      const uint32_t w[4] = {q.x & kAbs, q.y & kAbs, q.z & kAbs, q.w & kAbs};
      if (WANT & kCols) {
#pragma unroll
        for (int j = 0; j < 4; ++j) col[j] = __vmaxu2(col[j], w[j]);
      }
      if (WANT & kRows) m[p] = __vmaxu2(__vmaxu2(w[0], w[1]), __vmaxu2(w[2], w[3]));
    }
    if (WANT & kCols) {
#pragma unroll
      for (int j = 0; j < 4; ++j) col[j] = __vmaxu2(col[j], __shfl_xor_sync(0xffffffffu, col[j], 16));
      if (lane < 16) *reinterpret_cast<uint4*>(&part[warp][cg * 4]) = make_uint4(col[0], col[1], col[2], col[3]);
    }
    if (WANT & kRows) {
      uint32_t mine = 0u;   // lane cg stores the scale of row cg of the thread's
#pragma unroll
      for (int p = 0; p < kPairs; ++p) {
        uint32_t w = __vmaxu2(__byte_perm(m[p], m[p + kPairs], 0x5410), __byte_perm(m[p], m[p + kPairs], 0x7632));
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) w = __vmaxu2(w, __shfl_xor_sync(0xffffffffu, w, o));
        block_inverse2<E5M2>(w, rs[p], rs[p + kPairs]);
        mine = cg % kPairs == p ? w : mine;
      }
      const int r = r0 + rq * 4 + (cg & 3) + (cg >> 2) * 64;
      if (cg < kMine && r < R)
        store_scale(out, r, c0 / kTile, c0 + kTile >= C,
                    block_scale_byte<E5M2>(cg >= kPairs ? mine >> 16 : mine & 0xffffu));
    }
  }

  // Word `word` of 64: columns 2 word and 2 word + 1.
  static __device__ __forceinline__ void join_cols(const uint32_t (&part)[16][64], float2 (&cols)[64], int word, int r0,
                                                   int c0, int R, int C, const BlockOut& out_t) {
    uint32_t m = 0u;
#pragma unroll
    for (int k = 0; k < kWarps; ++k) m = __vmaxu2(m, part[k][word]);
    block_inverse2<E5M2>(m, cols[word].x, cols[word].y);
    const int c = c0 + 2 * word;
    if (c < C) {   // (C is even)
      store_scale(out_t, c, r0 / kTile, r0 + kTile >= R, block_scale_byte<E5M2>(m & 0xffffu));
      store_scale(out_t, c + 1, r0 / kTile, r0 + kTile >= R, block_scale_byte<E5M2>(m >> 16));
    }
  }

  // ONE: every value is multiplied by rs[0].
  template <int ONE>
  static __device__ __forceinline__ void write(const uint4 (&v)[U][4], const float (&rs)[kMine], const float2 (&cols)[64],
                                               uint32_t* tile, int r0, int c0, int R, int C, const BlockOut& out) {
    const int cg = threadIdx.x & 15, rq = threadIdx.x >> 4, c = c0 + cg * 8;
    f2 cs[4];
    if (ONE) {
      cs[0] = cs[1] = cs[2] = cs[3] = f2_of(rs[0], rs[0]);
    } else if (WANT & kCols) {
      const float4 a = *reinterpret_cast<const float4*>(&cols[cg * 4]), b = *reinterpret_cast<const float4*>(&cols[cg * 4 + 2]);
      cs[0] = f2_of(a.x, a.y);
      cs[1] = f2_of(a.z, a.w);
      cs[2] = f2_of(b.x, b.y);
      cs[3] = f2_of(b.z, b.w);
    }
    // Word `rg` (four rows) of a column of group cg lies at rg ^ 2 cg: the words that a warp writes at a time
    // are in different banks, and four of a column stay together for the 16-byte reads.
    uint8_t* orow = WANT & kRows ? out.data + (long long)(r0 + rq * 4) * out.ld + c : nullptr;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      uint32_t b[4][2], q[2][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t w[4] = {v[u][i].x, v[u][i].y, v[u][i].z, v[u][i].w};
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const f2 lo = f2_bf16(w[2 * k]), hi = f2_bf16(w[2 * k + 1]);
          if (ONE || (WANT & kCols)) {
            const float2 x = f2_get(f2_mul(lo, cs[2 * k])), y = f2_get(f2_mul(hi, cs[2 * k + 1]));
            q[k][i] = cast4<E5M2>(x.x, x.y, y.x, y.y);
          }
          if (ONE) {
            b[i][k] = q[k][i];
          } else if (WANT & kRows) {
            const f2 s = f2_of(rs[4 * u + i], rs[4 * u + i]);
            const float2 x = f2_get(f2_mul(lo, s)), y = f2_get(f2_mul(hi, s));
            b[i][k] = cast4<E5M2>(x.x, x.y, y.x, y.y);
          }
        }
        if (WANT & kRows) {
          if (r0 + rq * 4 + u * 64 + i < R && c < C)
            *reinterpret_cast<uint2*>(orow + (u * 64 + i) * out.ld) = make_uint2(b[i][0], b[i][1]);
        }
      }
      if (WANT & kCols) {
        const int rg = rq + u * 16;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          transpose4(q[k]);
#pragma unroll
          for (int j = 0; j < 4; ++j) tile[(cg * 8 + k * 4 + j) * 32 + (rg ^ (2 * cg))] = q[k][j];
        }
      }
    }
  }

  // Row c of out_t holds column c of the tile: 16 rows of it a piece.
  static __device__ __forceinline__ void copy_cols(const uint32_t* tile, int r0, int c0, int C, const BlockOut& out_t) {
    const int m = threadIdx.x & 7, tc0 = threadIdx.x >> 3;
    uint8_t* ocol = out_t.data + (long long)(c0 + tc0) * out_t.ld + r0 + m * 16;
#pragma unroll
    for (int k = 0; k < 2 * U; ++k) {
      const int tc = tc0 + k * (64 / U), g = tc >> 3;
      uint4 w = *reinterpret_cast<const uint4*>(tile + tc * 32 + 4 * (m ^ (g >> 1)));
      if (g & 1) w = make_uint4(w.z, w.w, w.x, w.y);
      if (c0 + tc < C && r0 + m * 16 < out_t.ld) *reinterpret_cast<uint4*>(ocol + k * (64 / U) * out_t.ld) = w;
    }
  }
};

// One tile by itself.
template <int TILED, int E5M2, int WANT, int U>
__device__ __forceinline__ void cast_tile(const uint4 (&v)[U][4], CastSmem<1>& sm, int r0, int c0, int R, int C,
                                          const BlockOut& out, const BlockOut& out_t) {
  using K = Cast<E5M2, WANT, U>;
  float rs[K::kMine];
  if (TILED) {
    uint32_t m = 0u;
#pragma unroll
    for (int p = 0; p < K::kMine; ++p) {
      const uint4& q = v[p / 4][p % 4];
      m = __vmaxu2(m, __vmaxu2(__vmaxu2(q.x & K::kAbs, q.y & K::kAbs), __vmaxu2(q.z & K::kAbs, q.w & K::kAbs)));
    }
    m = __reduce_max_sync(0xffffffffu, max(m & 0xffffu, m >> 16));
    if ((threadIdx.x & 31) == 0) sm.all[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K::kWarps; ++k) m = max(m, sm.all[k]);
    rs[0] = block_inverse<E5M2>(m);
    if (threadIdx.x < kTile) {
      const uint32_t e = block_scale_byte<E5M2>(m);
      if ((WANT & kRows) && r0 + threadIdx.x < R) store_scale(out, r0 + threadIdx.x, c0 / kTile, c0 + kTile >= C, e);
      if ((WANT & kCols) && c0 + threadIdx.x < C) store_scale(out_t, c0 + threadIdx.x, r0 / kTile, r0 + kTile >= R, e);
    }
  } else {
    K::maxima(v, sm.part[0], rs, r0, c0, R, C, out);
    if (WANT & kCols) {
      __syncthreads();
      if (threadIdx.x < 64) K::join_cols(sm.part[0], sm.cols[0], threadIdx.x, r0, c0, R, C, out_t);
      __syncthreads();
    }
  }
  K::template write<TILED>(v, rs, sm.cols[0], sm.tile[0], r0, c0, R, C, out);
  if (WANT & kCols) {
    __syncthreads();
    K::copy_cols(sm.tile[0], r0, c0, C, out_t);
  }
}

template <int U>
__device__ __forceinline__ void load_tile(uint4 (&v)[U][4], const bf16* __restrict__ x, long long ldx, int r0,
                                          int c0, int R, int C) {
  const int c = c0 + (threadIdx.x & 15) * 8, r = r0 + (threadIdx.x >> 4) * 4;
  const bf16* p = x + r * ldx + c;
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v[u][i] = r + u * 64 + i < R && c < C ? *reinterpret_cast<const uint4*>(p + (u * 64 + i) * ldx)
                                            : make_uint4(0u, 0u, 0u, 0u);
}

// SUM (the gradient of a bias): the tile's column sums too, to row r0 / 128 of `colsum` [.., C], always added
// in the same order.
template <int TILED, int E5M2, int WANT, int SUM>
__global__ void __launch_bounds__(256, 4)
    block_cast_kernel(const bf16* __restrict__ x, int R, int C, long long ldx, BlockOut out, BlockOut out_t,
                      float* __restrict__ colsum, int tiles_c) {
  __shared__ __align__(16) CastSmem<1> sm;
  pdl_wait();
  pdl_trigger();
  const int rt = blockIdx.x / tiles_c;
  const int r0 = rt * kTile, c0 = (blockIdx.x - rt * tiles_c) * kTile;
  uint4 v[2][4];
  load_tile(v, x, ldx, r0, c0, R, C);
  if (SUM) {
    f2 s[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) s[j] = f2_of(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      f2 t[4];
      unpack8(v[k / 4][k % 4], t);
#pragma unroll
      for (int j = 0; j < 4; ++j) s[j] = f2_add(s[j], t[j]);
    }
    float* part = reinterpret_cast<float*>(sm.tile[0]);   // [16 thread rows][128 columns]
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 t = f2_get(s[j]);
      *reinterpret_cast<float2*>(part + (threadIdx.x >> 4) * kTile + (threadIdx.x & 15) * 8 + 2 * j) = t;
    }
    __syncthreads();
    if (threadIdx.x < kTile && c0 + threadIdx.x < C) {
      float t = 0.f;
#pragma unroll
      for (int k = 0; k < 16; ++k) t += part[k * kTile + threadIdx.x];
      colsum[(long long)rt * C + c0 + threadIdx.x] = t;
    }
    __syncthreads();
    // (the unpacked values are not to be kept for the cast: they would fill the registers of two CTAs)
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      uint4& q = v[k / 4][k % 4];
      asm volatile("" : "+r"(q.x), "+r"(q.y), "+r"(q.z), "+r"(q.w));
    }
  }
  if (WANT) cast_tile<TILED, E5M2, WANT, 2>(v, sm, r0, c0, R, C, out, out_t);
}

// Column sums of each 128 rows of x (fp32, rows ldx elements apart), always added in the same order: the gradient of a
// bias behind fp32 activations, whose dy is rounded for the products alone. Bound by memory.
__global__ void __launch_bounds__(2 * kTile)
    block_colsum_kernel(const float* __restrict__ x, int R, int C, long long ldx, float* __restrict__ colsum) {
  __shared__ float part[kTile];
  pdl_wait();
  pdl_trigger();
  const int tiles_c = (C + kTile - 1) / kTile, rt = blockIdx.x / tiles_c;
  const int r0 = rt * kTile, c = (blockIdx.x - rt * tiles_c) * kTile + threadIdx.x % kTile, odd = threadIdx.x / kTile;
  float t = 0.f;
  if (c < C) {
#pragma unroll 8
    for (int r = r0 + odd; r < min(r0 + kTile, R); r += 2) t += x[r * ldx + c];
  }
  if (odd) part[threadIdx.x % kTile] = t;
  __syncthreads();
  if (!odd && c < C) colsum[(long long)rt * C + c] = t + part[threadIdx.x];
}

// Several casts in one launch, both layouts of each: the activations and the weights of a layer, which do not wait for one
// another. Measured for x [257, 1024] and w [2048, 1024]: 3.9 + 3.3 us in launches of their own, with 1.6 between them;
// x [4097, 2048] with w [16384, 2048] and [2048, 8192]: 11.0 + 26.9 + 20.0 us, 38 together.
struct CastJob {
  const bf16* x;
  int R, C;
  long long ldx;
  int tiled, tiles_c;
  unsigned first;   // its first CTA
  BlockOut out, out_t;
};
struct CastJobs {
  CastJob job[kMaxCasts];
};
__global__ void __launch_bounds__(256, 4) block_casts_kernel(const __grid_constant__ CastJobs jobs) {
  __shared__ __align__(16) CastSmem<1> sm;
  pdl_wait();
  pdl_trigger();
  int j = 0;
#pragma unroll
  for (int k = 1; k < kMaxCasts; ++k)
    if (blockIdx.x >= jobs.job[k].first) j = k;
  const CastJob& g = jobs.job[j];
  const int at = int(blockIdx.x - g.first), rt = at / g.tiles_c;
  const int r0 = rt * kTile, c0 = (at - rt * g.tiles_c) * kTile;
  uint4 v[2][4];
  load_tile(v, g.x, g.ldx, r0, c0, g.R, g.C);
  if (g.tiled)
    cast_tile<1, 0, kRows | kCols, 2>(v, sm, r0, c0, g.R, g.C, g.out, g.out_t);
  else
    cast_tile<0, 0, kRows | kCols, 2>(v, sm, r0, c0, g.R, g.C, g.out, g.out_t);
}

// h = act(gate) * up of [T, I] matrices (rows ld elements apart), rounded to bf16, in blocks of a row.
template <int KIND>
__global__ void __launch_bounds__(512)
    block_glu_fwd_kernel(const bf16* __restrict__ gate, const bf16* __restrict__ up, long long ld, int T, int I,
                         BlockOut h, int tiles_c) {
  __shared__ __align__(16) CastSmem<1> sm;
  pdl_wait();
  pdl_trigger();
  const int rt = blockIdx.x / tiles_c;
  const int r0 = rt * kTile, c0 = (blockIdx.x - rt * tiles_c) * kTile;
  uint4 g[1][4], u[1][4];
  load_tile(g, gate, ld, r0, c0, T, I);
  load_tile(u, up, ld, r0, c0, T, I);
#pragma unroll
  for (int i = 0; i < 4; ++i) g[0][i] = block_glu8<KIND>(g[0][i], u[0][i]);
  cast_tile<0, 0, kRows, 1>(g, sm, r0, c0, T, I, h, BlockOut{});
}

// The way back: from dh, gate and up the gradients of gate and up (rounded to bf16) in blocks of a row (`d`
// [T, 2 I], gate columns first) and of 128 tokens (`d_t` [2 I, T]), and h once more, in blocks of 128 tokens
// (`h_t` [I, T]): the operands of the input gradient and of both weight gradients from one read. I is a
// multiple of 128, so that no block holds columns of both. WANT: of the gradients' layouts; H: h.
//
// 11 bytes and 51 instructions a value: bound by those (54 % of the issue slots) and by the loads that two CTAs of an SM
// leave uncovered. 16 warps of twice the values each (128 registers) took 128 us for the 112 of 8192 x 4864; a
// persistent form that loads the next tile ahead spilled 700 bytes a thread and took 177; a prefetch of a later tile
// into L2 109, with a quarter more read.
constexpr int kGluSmem = sizeof(CastSmem<3>);
template <int KIND, int WANT, int H>
__global__ void __launch_bounds__(512, 2)
    block_glu_bwd_kernel(const bf16* __restrict__ dh, long long ld_dh, const bf16* __restrict__ gate,
                         const bf16* __restrict__ up, long long ld, int T, int I, BlockOut d, BlockOut d_t,
                         BlockOut h_t, int tiles_c) {
  using K = Cast<0, WANT, 1>;
  using KH = Cast<0, kCols, 1>;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  CastSmem<3>& sm = *reinterpret_cast<CastSmem<3>*>(smem_raw);
  pdl_wait();
  pdl_trigger();
  const int rt = blockIdx.x / tiles_c;
  const int r0 = rt * kTile, c0 = (blockIdx.x - rt * tiles_c) * kTile;
  uint4 g[1][4], u[1][4], x[1][4];
  load_tile(g, gate, ld, r0, c0, T, I);
  load_tile(u, up, ld, r0, c0, T, I);
  load_tile(x, dh, ld_dh, r0, c0, T, I);
#pragma unroll
  for (int i = 0; i < 4; ++i) block_glu_grad8<KIND>(g[0][i], u[0][i], x[0][i]);
  float rg[K::kMine], ru[K::kMine], none[K::kMine];
  if (WANT) {
    K::maxima(g, sm.part[0], rg, r0, c0, T, 2 * I, d);
    K::maxima(u, sm.part[1], ru, r0, I + c0, T, 2 * I, d);
  }
  if (H) KH::maxima(x, sm.part[2], none, r0, c0, T, I, BlockOut{});
  constexpr bool kT = WANT & kCols;
  if (kT || H) {
    __syncthreads();
    const int a = threadIdx.x >> 6, word = threadIdx.x & 63;
    if (kT && a < 2) K::join_cols(sm.part[a], sm.cols[a], word, r0, a * I + c0, T, 2 * I, d_t);
    if (H && a == 2) KH::join_cols(sm.part[2], sm.cols[2], word, r0, c0, T, I, h_t);
    __syncthreads();
  }
  if (WANT) {
    K::template write<0>(g, rg, sm.cols[0], sm.tile[0], r0, c0, T, 2 * I, d);
    K::template write<0>(u, ru, sm.cols[1], sm.tile[1], r0, I + c0, T, 2 * I, d);
  }
  if (H) KH::template write<0>(x, none, sm.cols[2], sm.tile[2], r0, c0, T, I, BlockOut{});
  if (kT || H) {
    __syncthreads();
    if (kT) {
      K::copy_cols(sm.tile[0], r0, c0, 2 * I, d_t);
      K::copy_cols(sm.tile[1], r0, I + c0, 2 * I, d_t);
    }
    if (H) KH::copy_cols(sm.tile[2], r0, c0, I, h_t);
  }
}

// out [rows, cols] = (out +) sums of P matrices, part p at p * stride, each value in the order of p, and bias [cols] behind
// them (null: none).
template <typename OutT>
__global__ void __launch_bounds__(256)
    block_sum_kernel(const float* __restrict__ part, int P, long long stride, int rows, int cols, OutT* out,
                     long long ldo, int accumulate, const bf16* __restrict__ bias) {
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
    if (bias != nullptr) {   // (at any multiple of 2 bytes)
      s = make_float4(s.x + __bfloat162float(bias[c]), s.y + __bfloat162float(bias[c + 1]),
                      s.z + __bfloat162float(bias[c + 2]), s.w + __bfloat162float(bias[c + 3]));
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

BlockOut block_out(const BlockMat& m, int kb0 = 0, bool fill = true) {
  return BlockOut{m.data, m.ld, m.scales, m.rows_s, kb0, fill};
}

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
  const unsigned grid = cast_grid(R, C);
  if (grid == 0) return -3;
  const int want = (out.data != nullptr ? kRows : 0) | (out_t.data != nullptr ? kCols : 0);
  if (want == 0 && colsum == nullptr) return 0;
#define LB_CAST(TI, E, W, S) \
  if (tiled == TI && e5m2 == E && want == W && (colsum != nullptr) == S) kern = block_cast_kernel<TI, E, W, S>
  void (*kern)(const bf16*, int, int, long long, BlockOut, BlockOut, float*, int) = nullptr;
  tiled = tiled ? 1 : 0;
  e5m2 = e5m2 ? 1 : 0;
  LB_CAST(0, 0, 1, 0);
  LB_CAST(0, 0, 2, 0);
  LB_CAST(0, 0, 3, 0);
  LB_CAST(0, 1, 1, 0);
  LB_CAST(0, 1, 2, 0);
  LB_CAST(0, 1, 3, 0);
  LB_CAST(1, 0, 1, 0);
  LB_CAST(1, 0, 2, 0);
  LB_CAST(1, 0, 3, 0);
  LB_CAST(1, 1, 1, 0);
  LB_CAST(1, 1, 2, 0);
  LB_CAST(1, 1, 3, 0);
  LB_CAST(0, 0, 0, 1);
  LB_CAST(0, 0, 1, 1);
  LB_CAST(0, 0, 2, 1);
  LB_CAST(0, 0, 3, 1);
#undef LB_CAST
  if (kern == nullptr) return -5;
  return launch_pdl(kern, dim3(grid), dim3(256), 0, stream, pdl_enabled(4LL * R * C), 1,
                    static_cast<const bf16*>(x), R, C, ldx, block_out(out), block_out(out_t, kb0_t), colsum,
                    (C + kTile - 1) / kTile);
}

int block_colsum(const float* x, int R, int C, long long ldx, float* colsum, cudaStream_t stream) {
  const unsigned grid = cast_grid(R, C);
  if (R <= 0 || C <= 0 || grid == 0) return -3;
  return launch_pdl(block_colsum_kernel, dim3(grid), dim3(2 * kTile), 0, stream, pdl_enabled(4LL * R * C), 1, x, R, C, ldx,
                    colsum);
}

int block_casts(const BlockCast* jobs, int n, cudaStream_t stream) {
  if (n < 1 || n > kMaxCasts) return -3;
  CastJobs all{};
  long long tiles = 0, bytes = 0;
  bool both = n > 1;
  for (int i = 0; i < n; ++i) both = both && jobs[i].out.data != nullptr && jobs[i].out_t.data != nullptr;
  if (!both) {   // a layout that is not wanted: launches of their own
    for (int i = 0; i < n; ++i) {
      const BlockCast& j = jobs[i];
      PdlScope scope(i > 0 || pdl_enabled());
      // (one after the other: a part that fills a word of scales too far is followed by the part that has it)
      if (const int rc = block_cast(j.x, j.R, j.C, j.ldx, j.tiled, 0, j.out, j.out_t, j.kb0_t, nullptr, stream)) return rc;
    }
    return 0;
  }
  for (int i = 0; i < kMaxCasts; ++i) {
    all.job[i].first = 0xffffffffu;
    if (i >= n) continue;
    const BlockCast& j = jobs[i];
    if (j.R <= 0 || j.C <= 0 || (j.C & 7) || (j.ldx & 7) || (reinterpret_cast<uintptr_t>(j.x) & 15)) return -3;
    if (!fits(j.out, j.R, j.C) || !fits(j.out_t, j.C, j.R) || j.kb0_t < 0 || (j.kb0_t > 0 && (j.R % kTile))) return -3;
    all.job[i] = CastJob{static_cast<const bf16*>(j.x), j.R, j.C, j.ldx, j.tiled, (j.C + kTile - 1) / kTile,
                         unsigned(tiles), block_out(j.out), block_out(j.out_t, j.kb0_t, j.fill_t)};
    tiles += 1LL * all.job[i].tiles_c * ((j.R + kTile - 1) / kTile);
    bytes += 4LL * j.R * j.C;
    if (tiles > 0x7fffffffLL) return -3;
  }
  return launch_pdl(block_casts_kernel, dim3(unsigned(tiles)), dim3(256), 0, stream, pdl_enabled(bytes), 1, all);
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
                    dim3(512), 0, stream, pdl_enabled(5LL * T * I), 1, static_cast<const bf16*>(gate),
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
  const int want = (d.data != nullptr ? kRows : 0) | (d_t.data != nullptr ? kCols : 0), h = h_t.data != nullptr;
  if (want == 0 && h == 0) return 0;
#define LB_GLU(W, H) \
  if (want == W && h == H) kern = kind == kSwiglu ? block_glu_bwd_kernel<kSwiglu, W, H> : block_glu_bwd_kernel<kGeglu, W, H>
  void (*kern)(const bf16*, long long, const bf16*, const bf16*, long long, int, int, BlockOut, BlockOut, BlockOut,
               int) = nullptr;
  LB_GLU(0, 1);
  LB_GLU(1, 0);
  LB_GLU(1, 1);
  LB_GLU(2, 0);
  LB_GLU(2, 1);
  LB_GLU(3, 0);
  LB_GLU(3, 1);
#undef LB_GLU
  static bool configured[2][4][2][kMaxDevices] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return -10;
  bool& done = configured[kind == kSwiglu ? 0 : 1][want][h][dev];
  if (!done && cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kGluSmem) != cudaSuccess)
    return -10;
  done = true;
  return launch_pdl(kern, dim3(grid), dim3(512), kGluSmem, stream, pdl_enabled(11LL * T * I), 1, static_cast<const bf16*>(dh), ld_dh,
                    static_cast<const bf16*>(gate), static_cast<const bf16*>(up), ld, T, I, block_out(d),
                    block_out(d_t), block_out(h_t), I / kTile);
}

// cols a multiple of 4; part, stride and out 16-byte aligned (out: 8 bytes in bf16).
int block_sum(const float* part, int P, long long stride, int rows, int cols, void* out, long long ldo,
              int out_fp32, int accumulate, const void* bias, cudaStream_t stream) {
  if (rows <= 0 || cols <= 0) return 0;
  if ((cols & 3) || (stride & 3) || (ldo & 3) || (accumulate && !out_fp32)) return -3;
  const bf16* b = static_cast<const bf16*>(bias);
  const long long n = 1LL * rows * (cols / 4);
  const unsigned grid = unsigned(n > 148LL * 8 * 256 ? 148 * 8 : (n + 255) / 256);
  const bool pdl = pdl_enabled(4LL * P * rows * cols);
  return out_fp32 ? launch_pdl(block_sum_kernel<float>, dim3(grid), dim3(256), 0, stream, pdl, 1, part, P, stride,
                               rows, cols, static_cast<float*>(out), ldo, accumulate, b)
                  : launch_pdl(block_sum_kernel<bf16>, dim3(grid), dim3(256), 0, stream, pdl, 1, part, P, stride,
                               rows, cols, static_cast<bf16*>(out), ldo, 0, b);
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
