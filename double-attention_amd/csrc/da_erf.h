// erf of the GELU in the GEMM epilogues and the 8-bit activation kernels.
#pragma once

#include "da_common.h"

namespace da {

constexpr float kSqrtHalf = 0.70710678118654752f;     // 1 / sqrt(2)
constexpr float kInvSqrt2Pi = 0.39894228040143268f;   // 1 / sqrt(2 pi)

// erf(x), and e^(-x^2), which the formula forms on the way: Abramowitz &
// Stegun, Handbook of Mathematical Functions, formula 7.1.26, erf(x) =
// 1 - (a1 t + ... + a5 t^5) e^(-x^2) with t = 1 / (1 + p x) for x >= 0 (odd
// extension), absolute error <= 1.5e-7, far below one rounding of the 16-bit
// outputs.  Branch-free: a reciprocal, an
// exponential and five FMAs, where the library erff takes several times the
// VALU work (the epilogue of a 4096 x 1536 GEMM runs it 6.3 million times).
__device__ __forceinline__ float erf_density(float x, float& density) {
  const float ax = fabsf(x);
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3275911f, ax, 1.f));
  float poly = __builtin_fmaf(t, 1.061405429f, -1.453152027f);
  poly = __builtin_fmaf(t, poly, 1.421413741f);
  poly = __builtin_fmaf(t, poly, -0.284496736f);
  poly = __builtin_fmaf(t, poly, 0.254829592f);
  poly *= t;
  density = __builtin_amdgcn_exp2f(-ax * ax * kLog2e);
  const float y = 1.f - poly * density;
  return copysignf(y, x);
}

__device__ __forceinline__ float erf_fast(float x) {
  float density;
  return erf_density(x, density);
}

}  // namespace da
