// The gated activations of eight elements, for the kernels that run them on rows in memory (act.cu) and on
// tiles that are cast at once (gemm/block_cast.cu): the same instructions, the same bits.
#pragma once

#include "../common/row.cuh"

namespace lb {

enum { kSwiglu = 0, kGeglu = 1 };

__device__ __forceinline__ float sigmoidf_(float x) { return __frcp_rn(1.f + __expf(-x)); }

__device__ __forceinline__ float gelu_tanh_(float x) {
  const float k0 = 0.7978845608028654f, k1 = 0.044715f;
  return 0.5f * x * (1.f + tanhf(k0 * (x + k1 * x * x * x)));
}
__device__ __forceinline__ float gelu_tanh_grad_(float x) {
  const float k0 = 0.7978845608028654f, k1 = 0.044715f;
  const float t = tanhf(k0 * (x + k1 * x * x * x));
  return 0.5f * (1.f + t) + 0.5f * x * (1.f - t * t) * k0 * (1.f + 3.f * k1 * x * x);
}

template <int KIND>
__device__ __forceinline__ uint4 glu_fwd8(const uint4& gq, const uint4& uq) {
  f2 g[4], u[4], o[4];
  unpack8(gq, g);
  unpack8(uq, u);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 x = f2_get(g[j]);
    const f2 a = KIND == kSwiglu ? f2_mul(g[j], f2_of(sigmoidf_(x.x), sigmoidf_(x.y)))
                                 : f2_of(gelu_tanh_(x.x), gelu_tanh_(x.y));
    o[j] = f2_mul(a, u[j]);
  }
  return pack8(o);
}

// d_gate and d_up of eight elements from the gradient of act(gate) * up.
template <int KIND>
__device__ __forceinline__ void glu_bwd8(const uint4& gq, const uint4& uq, const uint4& dq, uint4& dgq, uint4& duq) {
  const f2 one = f2_of(1.f, 1.f), minus_one = f2_of(-1.f, -1.f);
  f2 g[4], u[4], d[4], dg[4], du[4];
  unpack8(gq, g);
  unpack8(uq, u);
  unpack8(dq, d);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 x = f2_get(g[j]);
    f2 act, dact;
    if (KIND == kSwiglu) {
      const f2 s = f2_of(sigmoidf_(x.x), sigmoidf_(x.y));
      act = f2_mul(g[j], s);
      dact = f2_mul(s, f2_fma(g[j], f2_fma(s, minus_one, one), one));
    } else {
      act = f2_of(gelu_tanh_(x.x), gelu_tanh_(x.y));
      dact = f2_of(gelu_tanh_grad_(x.x), gelu_tanh_grad_(x.y));
    }
    du[j] = f2_mul(d[j], act);
    dg[j] = f2_mul(f2_mul(d[j], u[j]), dact);
  }
  dgq = pack8(dg);
  duq = pack8(du);
}

}  // namespace lb
