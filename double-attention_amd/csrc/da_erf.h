// erf of the GELU in the GEMM epilogues and the 8-bit activation kernels.
#pragma once

#include "da_common.h"

namespace da {

constexpr float kSqrtHalf = 0.70710678118654752f;     // 1 / sqrt(2)
constexpr float kInvSqrt2Pi = 0.39894228040143268f;   // 1 / sqrt(2 pi)

// erf for the 16-bit GEMM's GELU epilogue: Abramowitz & Stegun, Handbook of
// Mathematical Functions, formula 7.1.26, erf(x) = 1 - (a1 t + ... + a5 t^5)
// e^(-x^2) with t = 1 / (1 + p x) for x >= 0 (odd extension), absolute error
// <= 1.5e-7, far below one rounding of the 16-bit outputs.  Branch-free: a
// reciprocal, an exponential and five FMAs, where the library erff takes
// several times the VALU work (the epilogue of a 4096 x 1536 GEMM runs it 6.3
// million times).
__device__ __forceinline__ float erf_fast(float x) {
  const float ax = fabsf(x);
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3275911f, ax, 1.f));
  float poly = __builtin_fmaf(t, 1.061405429f, -1.453152027f);
  poly = __builtin_fmaf(t, poly, 1.421413741f);
  poly = __builtin_fmaf(t, poly, -0.284496736f);
  poly = __builtin_fmaf(t, poly, 0.254829592f);
  poly *= t;
  const float y = 1.f - poly * __builtin_amdgcn_exp2f(-ax * ax * kLog2e);
  return copysignf(y, x);
}

// The normal distribution's Phi(v), and e^(-v^2 / 2), which the same formula
// forms on the way: with x = |v| / sqrt(2), Phi(-|v|) = (1 - erf(x)) / 2 =
// (a1 t + ... + a5 t^5) / 2 e^(-x^2), at most 7.5e-8 off.  The factors 1 / 2
// and 1 / sqrt(2) sit in the constants: GELU is v Phi(v), and its slope
// Phi(v) + v e^(-v^2 / 2) / sqrt(2 pi).  No contraction beyond the FMAs that are
// written, so that every kernel rounds alike.
__device__ __forceinline__ float normal_cdf(float v, float& density) {
#pragma clang fp contract(off)
  const float a = fabsf(v);
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3275911f * kSqrtHalf, a, 1.f));
  float poly = __builtin_fmaf(t, 0.5f * 1.061405429f, 0.5f * -1.453152027f);
  poly = __builtin_fmaf(t, poly, 0.5f * 1.421413741f);
  poly = __builtin_fmaf(t, poly, 0.5f * -0.284496736f);
  poly = __builtin_fmaf(t, poly, 0.5f * 0.254829592f);
  const float r = v * 0.84932180028801904f;   // sqrt(log2(e) / 2)
  density = __builtin_amdgcn_exp2f(-(r * r));
  const float tail = poly * t * density;      // Phi(-|v|)
  return v < 0.f ? tail : 1.f - tail;
}
__device__ __forceinline__ float gelu(float v) {
#pragma clang fp contract(off)
  float density;
  return v * normal_cdf(v, density);
}

}  // namespace da
