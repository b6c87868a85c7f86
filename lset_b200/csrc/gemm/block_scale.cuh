// 8-bit floats in blocks of 128 with one power-of-two scale each: the format, its rounding, and the
// tensor-core instruction that takes the scales.
//
// A block holds q in e4m3 (or e5m2) and a scale byte e (biased by 127): its values are q * 2^(e - 127).
// e is the smallest with which the block's largest magnitude is at most fmax = 448 (57344): both are
// 1.75 * 2^n, so e follows from the exponent of that magnitude, plus one where its mantissa is above 0.75.
// With powers of two scaling is exact in both directions, the one rounding of a value is that to its 3 (2)
// mantissa bits, and the tensor cores multiply by the scales themselves (kind::mxf8f6f4.block_scale), at
// their full 8-bit rate. Factors with a mantissa would have to be applied to every partial sum of 128 in
// registers; what they would buy is less than one bit of range at the lower end of a block.
//   * a block of zeros has the scale 1 (e = 127);
//   * e is kept in [1, 254], normal powers of two (magnitudes below 2^-118 lose range, not scale);
//   * a block with a NaN or an infinity is NaN throughout (q = 0x7f, e = 127): a product shows it, where
//     saturated values would hide it.
//
// Scales of a matrix [rows, K] lie as words [ceil(K / 512)][rows]: byte kb % 4 of word (kb / 4, row) is the
// scale of columns 128 kb .. 128 kb + 127 of that row. 128 x 128 blocks repeat theirs for every row. So a
// warp reads the words of 32 rows as one line, a word is what the tensor memory holds for a row and
// four blocks, and no row count needs padding.
#pragma once

#include "../common/ptx.cuh"

namespace lb {

constexpr int kScaleBlock = 128;
constexpr uint32_t kScaleOne = 127u;

// What the values of a block are multiplied by before they are rounded, 2^(127 - e) as float bits, for a block
// whose largest magnitude has the bf16 bits `a`; NaN where that is not finite (and then so is every product).
// (a + 31) / 128 is its exponent, plus one where the mantissa is above 0.75 = 96 / 128.
template <int E5M2>
__device__ __forceinline__ float block_inverse(uint32_t a) {
  const int x = min((E5M2 ? 269 : 262) - int((a + 31u) >> 7), 253);
  return __uint_as_float(a >= 0x7f80u ? 0x7fffffffu : uint32_t(x) << 23);
}
// The same for the two halves of a word: with n = 262 (269), 2^(127 - e) has the bits (n - x) << 23, and x << 23 is
// (a + 31) & 0xff80, 16 bits up.
template <int E5M2>
__device__ __forceinline__ void block_inverse2(uint32_t w, float& lo, float& hi) {
  constexpr uint32_t kTop = (E5M2 ? 269u : 262u) << 23, kMost = 253u << 23;
  const uint32_t x = (w + 0x001f001fu) & 0xff80ff80u;
  lo = __uint_as_float(min(kTop - (x << 16), kMost));
  hi = __uint_as_float(min(kTop - (x & 0xffff0000u), kMost));
  if (((w & 0xffffu) >= 0x7f80u) || w >= 0x7f800000u) {   // hardly ever
    lo = (w & 0xffffu) >= 0x7f80u ? __uint_as_float(0x7fffffffu) : lo;
    hi = w >= 0x7f800000u ? __uint_as_float(0x7fffffffu) : hi;
  }
}
// The scale byte that goes with it.
template <int E5M2>
__device__ __forceinline__ uint32_t block_scale_byte(uint32_t a) {
  const int x = min((E5M2 ? 269 : 262) - int((a + 31u) >> 7), 253);
  return a == 0u || a >= 0x7f80u ? kScaleOne : uint32_t(254 - x);
}

// Four values, scaled already, as bytes, to nearest even.
template <int E5M2>
__device__ __forceinline__ uint32_t cast4(float a, float b, float c, float d) {
  uint32_t o;
  if (E5M2)
    asm("{\n.reg .b16 lo, hi;\ncvt.rn.satfinite.e5m2x2.f32 lo, %2, %1;\ncvt.rn.satfinite.e5m2x2.f32 hi, %4, %3;\n"
        "mov.b32 %0, {lo, hi};\n}" : "=r"(o) : "f"(a), "f"(b), "f"(c), "f"(d));
  else
    asm("{\n.reg .b16 lo, hi;\ncvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\ncvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n"
        "mov.b32 %0, {lo, hi};\n}" : "=r"(o) : "f"(a), "f"(b), "f"(c), "f"(d));
  return o;
}

// D[tmem] (+)= (A[smem] * scales) * (B[smem] * scales), 8-bit floats, 32 elements of depth. The scale
// operands are tensor-memory addresses: row r's word lies in lane r % 32 (of every quarter of the lanes),
// column r / 32; the instruction descriptor says which of its bytes applies.
__device__ __forceinline__ void umma_block(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc,
                                           uint32_t idesc, uint32_t tmem_sa, uint32_t tmem_sb,
                                           uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %6, 0;\n"
      "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n"
      "}\n"
      :
      : "r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(tmem_sa), "r"(tmem_sb), "r"(accumulate)
      : "memory");
}

// Instruction descriptor of kind::mxf8f6f4: operand formats 0 = e4m3, 1 = e5m2, both K-major; scales are
// powers of two (bit 23), byte `sf` of their words.
__device__ __forceinline__ uint32_t umma_idesc_block(int M, int N, int a_e5m2, int b_e5m2, int sf) {
  return (uint32_t(sf) << 4)             // which byte of B's words
         | (uint32_t(a_e5m2) << 7)       // A format
         | (uint32_t(b_e5m2) << 10)      // B format
         | (uint32_t(N >> 3) << 17)      // N / 8
         | (1u << 23)                    // scale format: exponents
         | (uint32_t(M >> 7) << 27)      // M / 128
         | (uint32_t(sf) << 29);         // which byte of A's words
}

__device__ __forceinline__ void tmem_st_32x32b_x8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
      :
      : "r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
      : "memory");
}

__device__ __forceinline__ void tmem_st_32x32b_x4(uint32_t taddr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(taddr), "r"(a), "r"(b), "r"(c),
               "r"(d)
               : "memory");
}

}  // namespace lb
