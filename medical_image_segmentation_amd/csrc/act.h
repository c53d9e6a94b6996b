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

// the two parts of gelu: q = Phi(-|u|) and e = e^(-u^2/2); the coefficients carry erfc's factor 1/2
__device__ __forceinline__ void gelu_parts(float u, float& q, float& e) {
  const float t = fast_rcp(fmaf(0.3275911f * 0.70710678f, fabsf(u), 1.f));
  e = fast_exp2(-0.72134752f * u * u);
  float p = fmaf(t, 0.5f * 1.061405429f, 0.5f * -1.453152027f);
  p = fmaf(t, p, 0.5f * 1.421413741f);
  p = fmaf(t, p, 0.5f * -0.284496736f);
  p = fmaf(t, p, 0.5f * 0.254829592f);
  q = p * (t * e);
}

template <int ACT>
__device__ __forceinline__ float act_value(float u) {
  if constexpr (ACT == MIS_ACT_RELU) {
    return u < 0.f ? 0.f : u;                    // (NaN stays NaN)
  } else if constexpr (ACT == MIS_ACT_SILU) {
    return u * fast_rcp(1.f + fast_exp2(-1.44269504f * u));
  } else if constexpr (ACT == MIS_ACT_GELU) {
    float q, e;                                  // u Phi(u) = max(u, 0) - |u| Phi(-|u|)
    gelu_parts(u, q, e);
    return fmaf(-fabsf(fminf(u, 64.f)), q, fmaxf(u, 0.f));       // (q is 0 from 64 on, also at infinity; NaN for NaN)
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
    float q, e;
    gelu_parts(u, q, e);
    return fmaf(0.39894228f * u, e, u < 0.f ? q : 1.f - q);
  } else {
    return 1.f;
  }
}
