// The activations of the decoder operators and their derivatives.
#pragma once

#include "decoder_common.cuh"

#include <type_traits>

enum { ACT_SILU = 0, ACT_GELU = 1, ACT_RELU = 2 };

// act(g) and its derivative.  Exponentials are 2^(g log2 e) on the hardware unit: a relative
// error of |g| 2^-24, which the factor s (1 - s) |g| <= 0.28 |g| of silu and the decay of
// the others keep under 2^-23 of |g| in the result.
//
// gelu takes Phi(-|g|) as a polynomial times exp(-g^2 / 2), an exponential that its derivative
// shares.  16-bit tensors: the five coefficients of Abramowitz and Stegun 7.1.26 in
// 1 / (1 + c |g|), off by 7e-8.  float32: six and a constant of 1/2 in v = |g| / (1 + 0.264 |g|),
// fitted to the smallest largest error, 1e-9; in v the reciprocal's rounding fades towards
// zero, and gelu of normal g is as far from 64 bits as 0.5 g (1 + erf) in 32 (with the five, 2.3
// times as far).  They cost 16-bit tensors 17 us of 167 (1M rows 64-256-48, forward), for nothing
// that these would show, float32 8 of 387 (300k rows 59-128-3, both directions).
template <int ACT, typename T>
__device__ __forceinline__ float2 activation(float g) {
  if constexpr (ACT == ACT_RELU) {
    return make_float2(g < 0.f ? 0.f : g, g > 0.f ? 1.f : 0.f);  // (NaN stays, -inf gives 0)
  } else if constexpr (ACT == ACT_SILU) {
    const float s = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(g * -1.44269504f));
    const float a = g * s;
    return make_float2(a, fmaf(a, 1.f - s, s));
  } else {
    const float e = __builtin_amdgcn_exp2f(g * g * -0.72134752f);  // exp(-g^2 / 2)
    float q;
    if constexpr (std::is_same<T, float>::value) {
      const float m = fminf(fabsf(g), 64.f);  // (e is 0 long before; an infinity would make v NaN)
      const float v = m * __builtin_amdgcn_rcpf(fmaf(m, 0.264f, 1.f));
      q = fmaf(v, -5.17113608e-05f, 0.000272698357f);
      q = fmaf(v, q, 0.0021007601f);
      q = fmaf(v, q, -0.0287824044f);
      q = fmaf(v, q, 0.144678869f);
      q = fmaf(v, q, -0.398942273f);
      q = fmaf(v, q, 0.5f) * e;
    } else {
      const float t = __builtin_amdgcn_rcpf(fmaf(fabsf(g), 0.3275911f * 0.70710678f, 1.f));
      q = fmaf(t, 0.5f * 1.061405429f, 0.5f * -1.453152027f);
      q = fmaf(t, q, 0.5f * 1.421413741f);
      q = fmaf(t, q, 0.5f * -0.284496736f);
      q = fmaf(t, q, 0.5f * 0.254829592f);
      q = q * t * e;
    }
    const float phi = g >= 0.f ? 1.f - q : q;
    return make_float2(g * phi, fmaf(g * 0.39894228f, e, phi));
  }
}
