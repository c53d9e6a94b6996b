// Activations of the group-norm and matrix-product kernels, with their slopes (MIS_ACT_* of misamd.h).
//   relu  max(u, 0)                      slope [u > 0]
//   silu  u s,  s = 1 / (1 + e^-u)       slope s (1 + u (1 - s))
//   gelu  u Phi(u), Phi the normal distribution function;  slope Phi + u e^(-u^2/2) / sqrt(2 pi)
// Phi(-|u|) = t P(t) e^(-u^2/2), t = 1 / (1 + 0.3 |u|), P the polynomial of degree 7 with the least largest relative error
// over |u| <= 14, 1.5e-7 (found by reweighted least squares on 4000 Chebyshev nodes in t; with degree 5 it would be 8e-6, 8
// 3e-8, which the float32 evaluation does not show): one exponential serves the value and the slope, and the small side is formed
// without a cancellation.  e^x goes through the hardware's 2^x, with a relative error of about |x| 2^-24 from its argument: Phi
// is right to 5e-7 of itself at -1, 9e-7 at -3, 2e-6 at -5.
#pragma once
#include "common.h"

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float fast_rcp(float x) { return __builtin_amdgcn_rcpf(x); }

// the two parts of gelu: q = Phi(-|u|) and e = e^(-u^2/2)
__device__ __forceinline__ void gelu_parts(float u, float& q, float& e) {
  const float t = fast_rcp(fmaf(0.3f, fabsf(u), 1.f));
  e = fast_exp2(-0.72134752f * u * u);
  float p = fmaf(t, 0.0356747732f, -0.157203078f);
  p = fmaf(t, p, 0.2063535f);
  p = fmaf(t, p, -0.0536836423f);
  p = fmaf(t, p, 0.128561631f);
  p = fmaf(t, p, 0.0999134928f);
  p = fmaf(t, p, 0.120753959f);
  p = fmaf(t, p, 0.119629301f);
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
