// Activations of the group-norm and matrix-product kernels, with their slopes (MIS_ACT_* of misamd.h).
//   relu  max(u, 0)                      slope [u > 0]
//   silu  u s,  s = 1 / (1 + e^-u)       slope s (1 + u (1 - s))
//   gelu  u Phi(u), Phi the normal distribution function;  slope Phi + u e^(-u^2/2) / sqrt(2 pi)
// Phi(-|u|) = P(t) t e^(-u^2/2) / 2, t = 1 / (1 + p |u| / sqrt 2), with the five coefficients of Abramowitz &
// Stegun 7.1.26 (absolute error 1.5e-7 on erf): one exponential serves the value and the slope, and the small side
// is formed without a cancellation.  e^x goes through the hardware's 2^x (relative error about |x| 2^-24).
#pragma once
#include "common.h"

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float fast_rcp(float x) { return __builtin_amdgcn_rcpf(x); }

// the two halves of gelu: Phi(u) and e^(-u^2/2)
__device__ __forceinline__ void gelu_parts(float u, float& phi, float& e) {
  const float z = fabsf(u);
  const float t = fast_rcp(fmaf(0.3275911f * 0.70710678f, z, 1.f));
  e = fast_exp2(-0.72134752f * u * u);
  float p = fmaf(t, 1.061405429f, -1.453152027f);
  p = fmaf(t, p, 1.421413741f);
  p = fmaf(t, p, -0.284496736f);
  p = fmaf(t, p, 0.254829592f);
  const float q = 0.5f * p * t * e;
  phi = u >= 0.f ? 1.f - q : q;
}

template <int ACT>
__device__ __forceinline__ float act_value(float u) {
  if constexpr (ACT == MIS_ACT_RELU) {
    return u < 0.f ? 0.f : u;                    // (NaN stays NaN)
  } else if constexpr (ACT == MIS_ACT_SILU) {
    return u * fast_rcp(1.f + fast_exp2(-1.44269504f * u));
  } else if constexpr (ACT == MIS_ACT_GELU) {
    float phi, e;
    gelu_parts(u, phi, e);
    return u * phi;
  } else {
    return u;
  }
}

template <int ACT>
__device__ __forceinline__ float act_slope(float u) {
  if constexpr (ACT == MIS_ACT_RELU) {
    return u > 0.f ? 1.f : 0.f;
  } else if constexpr (ACT == MIS_ACT_SILU) {
    const float s = fast_rcp(1.f + fast_exp2(-1.44269504f * u));
    return s * fmaf(u, 1.f - s, 1.f);
  } else if constexpr (ACT == MIS_ACT_GELU) {
    float phi, e;
    gelu_parts(u, phi, e);
    return fmaf(0.39894228f * u, e, phi);
  } else {
    return 1.f;
  }
}
