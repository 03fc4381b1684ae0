// What the gated feed-forward block's kernels share: the gate's arithmetic, and the
// interface of the kernels for narrow rows.
#pragma once

#include "matrix.cuh"

enum { ACT_SILU = 0, ACT_GELU = 1, ACT_RELU = 2 };

// act(g) and its derivative.  Exponentials are 2^(g log2 e) on the hardware unit: a relative
// error of |g| 2^-24, which the factor s (1 - s) |g| <= 0.28 |g| of silu and the decay of
// the others keep under 2^-23 of |g| in the result.  gelu of 16-bit tensors takes
// erfc from Abramowitz and Stegun 7.1.26 (off by 1.5e-7 at most, a 2^-13th of a
// bfloat16's spacing at 1), which shares its exponential with the derivative.
template <typename T, int ACT>
__device__ __forceinline__ float2 activation(float g) {
  if constexpr (ACT == ACT_RELU) {
    return g > 0.f ? make_float2(g, 1.f) : make_float2(0.f * g, 0.f);
  } else if constexpr (ACT == ACT_SILU) {
    const float s = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(g * -1.44269504f));
    const float a = g * s;
    return make_float2(a, fmaf(a, 1.f - s, s));
  } else {
    const float e = __builtin_amdgcn_exp2f(g * g * -0.72134752f);  // exp(-g^2 / 2)
    float phi;
    if constexpr (sizeof(T) == 4) {
      phi = 0.5f * (1.f + erff(g * 0.70710678f));
    } else {
      const float t = __builtin_amdgcn_rcpf(fmaf(fabsf(g), 0.3275911f * 0.70710678f, 1.f));
      float q = fmaf(t, 0.5f * 1.061405429f, 0.5f * -1.453152027f);
      q = fmaf(t, q, 0.5f * 1.421413741f);
      q = fmaf(t, q, 0.5f * -0.284496736f);
      q = fmaf(t, q, 0.5f * 0.254829592f);
      q = q * t * e;
      phi = g >= 0.f ? 1.f - q : q;
    }
    return make_float2(g * phi, fmaf(g * 0.39894228f, e, phi));
  }
}

// Calls f with the activation as a constant (the branch is the same for all lanes).
template <typename F>
__device__ __forceinline__ void with_activation(int act, F&& f) {
  if (act == ACT_SILU)
    f(std::integral_constant<int, ACT_SILU>());
  else if (act == ACT_GELU)
    f(std::integral_constant<int, ACT_GELU>());
  else
    f(std::integral_constant<int, ACT_RELU>());
}

// The block's sizes and tensors, as the entry points get them.
struct FfnCall {
  int64_t rows;
  int32_t width, hidden, out, act;
  int64_t x_pitch, dy_pitch;
  const void *x, *wg, *wu, *wd, *bg, *bu, *bd, *dy;
  void *y, *dx, *dwg, *dwu, *dwd, *dbg, *dbu, *dbd;
};

// Narrow rows (gated_ffn_rows.cuh): whether a call's sizes are theirs, the workspace they
// take and their launches.
template <typename T>
struct RowKernels {
  static bool takes(int64_t rows, int32_t width, int32_t hidden, int32_t out);
  static uint64_t workspace(int32_t width, int32_t hidden, int32_t out);
  static void forward(const FfnCall& c, void* workspace, hipStream_t stream);
};
