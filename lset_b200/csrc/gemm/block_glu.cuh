// Gated activations of eight elements, on their way into block casts: in registers, two elements an
// instruction, from bf16 pairs to bf16 pairs.
//
// SiLU: g s with s = sigmoid(g), and its derivative s (1 + g (1 - s)), from one exponential and one reciprocal, the
// hardware's approximations. s is off by |g| 2^-24 of itself (-g log2(e) is rounded to 24 bits before it is an exponent)
// and 2^-22 more, and is 0 below g = -87.3, where 1 + exp(-g) passes 2^126; results are rounded to bf16, 2^-8, and then to
// 3 bits. With expf and a correctly rounded reciprocal as many of those fall to another side than 64 bits put them (4.4e-6
// of the gradients at 4097 x 2048 x 8192 either way: the sums in front decide), and the epilogue that activates
// is bound by them: the gate and up product of that size takes 187 us for 140, the gated backward 108 for 103.
// The tanh form of GELU as it is written, with CUDA's tanhf: g sigmoid(2 y) in place of g (1 + tanh(y)) / 2 would be
// cheaper and closer to 64 bits where 1 + tanh cancels, but other than the layers one by one, by more than a step of
// bf16 for one value in 100 there.
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

// act(g) of two gates and, where DERIV, its derivative.
template <int KIND, bool DERIV>
__device__ __forceinline__ void act2(f2 g, f2& act, f2& dact) {
  if (KIND == kSwiglu) {
    constexpr float kLog2e = 1.4426950408889634f;
    const float2 x = f2_get(f2_mul(g, f2_of(-kLog2e, -kLog2e)));
    const f2 s = f2_of(sigmoid_approx(x.x), sigmoid_approx(x.y)), one = f2_of(1.f, 1.f);
    act = f2_mul(g, s);
    if (DERIV) dact = f2_mul(s, f2_fma(g, f2_fma(s, f2_of(-1.f, -1.f), one), one));
  } else {
    const float2 x = f2_get(g);
    float a[2], d[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      constexpr float c = 0.7978845608028654f, k = 0.044715f;
      const float v = i ? x.y : x.x;
      const float t = tanhf(__fmul_rn(c, __fadd_rn(v, __fmul_rn(__fmul_rn(__fmul_rn(k, v), v), v))));
      const float half = __fmul_rn(0.5f, v), up = __fadd_rn(1.f, t);
      a[i] = __fmul_rn(half, up);
      if (DERIV) {
        const float slope = __fmul_rn(__fmul_rn(half, __fadd_rn(1.f, -__fmul_rn(t, t))), c);
        d[i] = __fadd_rn(__fmul_rn(0.5f, up),
                         __fmul_rn(slope, __fadd_rn(1.f, __fmul_rn(__fmul_rn(3.f * k, v), v))));
      }
    }
    act = f2_of(a[0], a[1]);
    if (DERIV) dact = f2_of(d[0], d[1]);
  }
}

// act(gate) * up
template <int KIND>
__device__ __forceinline__ uint4 block_glu8(const uint4& gq, const uint4& uq) {
  f2 g[4], u[4], a, none;
  unpack8(gq, g);
  unpack8(uq, u);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    act2<KIND, false>(g[j], a, none);
    g[j] = f2_mul(a, u[j]);
  }
  return pack8(g);
}

// In place: gate, up and the gradient d of h = act(gate) * up become the gradient of gate, that of up, and h.
template <int KIND>
__device__ __forceinline__ void block_glu_grad8(uint4& gq, uint4& uq, uint4& dq) {
  f2 g[4], u[4], d[4], act, dact;
  unpack8(gq, g);
  unpack8(uq, u);
  unpack8(dq, d);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    act2<KIND, true>(g[j], act, dact);
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
