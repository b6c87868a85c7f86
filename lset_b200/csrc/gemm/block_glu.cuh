// Gated activations of eight elements, on their way into block casts: in registers, two elements an
// instruction, from bf16 pairs to bf16 pairs.
//
// Both activations are g * sigmoid(z): SiLU with z = g, the tanh form of GELU with z = 2 sqrt(2 / pi) (g + k g^3), as
// (1 + tanh(y)) / 2 = sigmoid(2 y). So one exponential and one reciprocal do for value and derivative,
//   d/dg [g s(z)] = s + g z' s (1 - s).
// Both are the hardware's approximations (2 units in the last place of 32 bits); results are rounded to bf16, 2^-9,
// and then to 3 bits. The casts are bound by the instructions they issue: with a correctly rounded reciprocal
// and the sigmoid once for each direction the backward took 79 instructions an element.
#pragma once

#include "../common/row.cuh"

namespace lb {

enum { kSwiglu = 0, kGeglu = 1 };

__device__ __forceinline__ float sigmoid_approx(float minus_z_log2e) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(minus_z_log2e));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
  return r;
}

// s = sigmoid(z(g)) of two gates and, where DERIV, dz = z'(g).
template <int KIND, bool DERIV>
__device__ __forceinline__ void glu_sigmoid2(f2 g, f2& s, f2& dz) {
  constexpr float kLog2e = 1.4426950408889634f, k0 = 2.f * 0.7978845608028654f, k1 = 0.044715f;
  f2 t;
  if (KIND == kSwiglu) {
    t = f2_mul(g, f2_of(-kLog2e, -kLog2e));
  } else {
    const f2 g2 = f2_mul(g, g);
    constexpr float a = -kLog2e * k0;
    t = f2_mul(g, f2_fma(g2, f2_of(a * k1, a * k1), f2_of(a, a)));
    if (DERIV) dz = f2_fma(g2, f2_of(3.f * k0 * k1, 3.f * k0 * k1), f2_of(k0, k0));
  }
  const float2 x = f2_get(t);
  s = f2_of(sigmoid_approx(x.x), sigmoid_approx(x.y));
}

// act(gate) * up
template <int KIND>
__device__ __forceinline__ uint4 block_glu8(const uint4& gq, const uint4& uq) {
  f2 g[4], u[4], s, dz;
  unpack8(gq, g);
  unpack8(uq, u);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    glu_sigmoid2<KIND, false>(g[j], s, dz);
    g[j] = f2_mul(f2_mul(g[j], s), u[j]);
  }
  return pack8(g);
}

// In place: gate, up and the gradient d of h = act(gate) * up become the gradient of gate, that of up, and h.
template <int KIND>
__device__ __forceinline__ void block_glu_grad8(uint4& gq, uint4& uq, uint4& dq) {
  f2 g[4], u[4], d[4], s, dz;
  const f2 one = f2_of(1.f, 1.f), minus_one = f2_of(-1.f, -1.f);
  unpack8(gq, g);
  unpack8(uq, u);
  unpack8(dq, d);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    glu_sigmoid2<KIND, true>(g[j], s, dz);
    const f2 act = f2_mul(g[j], s), rest = f2_fma(s, minus_one, one);
    const f2 gz = KIND == kSwiglu ? g[j] : f2_mul(g[j], dz);
    const f2 dact = f2_mul(s, f2_fma(gz, rest, one));
    g[j] = f2_mul(f2_mul(d[j], u[j]), dact);
    const f2 h = f2_mul(act, u[j]);
    u[j] = f2_mul(d[j], act);
    d[j] = h;
  }
  gq = pack8(g);
  uq = pack8(u);
  dq = pack8(d);
}

}  // namespace lb
