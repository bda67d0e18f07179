// silu(g) = g / (1 + e^-g) and sigmoid(g), shared by the kernels that fuse SwiGLU.
#pragma once

#include "fm_common.h"

namespace fm {

// e^-g to about an ulp: 2^(-g log2 e) with the product split into a rounded
// part and its exact remainder (the remainder's share of the exponent would
// otherwise cost |g| 2^-24 ln 2 relative), the hardware 2^x on the fraction
// of the rounded part plus the remainder (|x| <= 0.5 + 2^-24), and the integer
// part as an exponent.  Overflow (g < -88.7) gives +inf, which the callers
// treat as IEEE division would.  Beyond +-1000 the result is that of +-1000,
// infinity or 0: from 2^31 on the remainder alone would pass the exponents'
// range.  (A NaN counts as a bound; the callers' other operand is g itself.)
__device__ __forceinline__ float exp_neg(float g) {
#pragma clang fp contract(off)   // ph must be rounded: pl is its exact remainder
  constexpr float kL = 1.44269502162933349609375f;   // RN(log2 e)
  constexpr float kLlo = 1.925963033500011e-08f;     // log2 e - kL
  g = __builtin_amdgcn_fmed3f(g, -1000.f, 1000.f);
  const float ph = -g * kL;
  const float pl = fmaf(-g, kLlo, fmaf(-g, kL, -ph));
  const float n = __builtin_rintf(ph);   // 2^x on x in [-0.5, 0.5], then the exponent
  return __builtin_amdgcn_ldexpf(__builtin_amdgcn_exp2f((ph - n) + pl), int(n));
}

// silu(g) = g / d and sigmoid(g) = 1 / d, d = 1 + e^-g: the expressions of
// the reference's torch silu and its backward (x / (1 + exp(-x)), sigmoid =
// 1 / (1 + exp(-x))).  Quotients from the hardware reciprocal with a
// residual correction (within an ulp of the rounded quotient).  d infinite
// (g < -88.7): sigmoid 0 and silu -0, as IEEE division gives; g infinite: silu
// infinite, where the residual is infinity less infinity (and a NaN is itself).
__device__ __forceinline__ float silu_quotient(float g, float d, float r) {
#pragma clang fp contract(off)
  const float q0 = g * r;
  const float q = fmaf(fmaf(-d, q0, g), r, q0);
  return d <= 3.40282347e38f ? (g <= 3.40282347e38f ? q : g) : g * 0.f;
}
__device__ __forceinline__ float silu_only(float g) {
  const float d = 1.f + exp_neg(g);
  return silu_quotient(g, d, __builtin_amdgcn_rcpf(d));
}

struct SigSilu {
  float s, silu;
};
__device__ __forceinline__ SigSilu sig_silu(float g) {
#pragma clang fp contract(off)
  const float d = 1.f + exp_neg(g);
  float r = __builtin_amdgcn_rcpf(d);
  r = fmaf(fmaf(-d, r, 1.f), r, r);
  return SigSilu{d <= 3.40282347e38f ? r : 0.f, silu_quotient(g, d, r)};
}

// SwiGLU of eight values and its backward, every product and sum rounded (the same values in every kernel that inlines them):
// h = silu(g) u; torch autograd of it: dg = (dh u) s (1 + g (1 - s)), du = dh silu(g), each operation rounded in this order (an
// infinite g gives a NaN dg there and here).
__device__ __forceinline__ void swiglu8(const float (&g)[8], const float (&u)[8], float (&h)[8]) {
#pragma clang fp contract(off)
#pragma unroll
  for (int i = 0; i < 8; ++i) h[i] = silu_only(g[i]) * u[i];
}
__device__ __forceinline__ void swiglu8_backward(const float (&g)[8], const float (&u)[8], const float (&dh)[8], float (&dg)[8],
                                                 float (&du)[8]) {
#pragma clang fp contract(off)
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const SigSilu s = sig_silu(g[i]);
    dg[i] = ((dh[i] * u[i]) * s.s) * (1.f + g[i] * (1.f - s.s));
    du[i] = dh[i] * s.silu;
  }
}

}  // namespace fm
