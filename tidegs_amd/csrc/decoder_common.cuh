// Element types of the decoder operators (layer norm, dropout, gated
// feed-forward): 32-bit floats, bfloat16 and IEEE half.  Every kernel computes in
// 32 bits and rounds once, to nearest even, where a value is stored.
#pragma once

#include "tgs_common.cuh"

#include <algorithm>

enum { TGS_F32 = 0, TGS_BF16 = 1, TGS_F16 = 2 };

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

template <typename T>
__device__ __forceinline__ float to_f32(T v) {
  return (float)v;
}
template <typename T>
__device__ __forceinline__ T from_f32(float v) {
  return (T)v;
}

// 16 bytes of consecutive values: the widest load of a lane.
template <typename T>
struct alignas(16) Vec16 {
  static constexpr int N = 16 / sizeof(T);
  T v[N];
};

template <typename T>
static inline bool aligned16(const T* p, int64_t pitch) {
  return ((uintptr_t)p % 16 == 0) && (pitch * (int64_t)sizeof(T) % 16 == 0);
}

// Calls f with a value of the element type of `dtype`; an error code otherwise.
template <typename F>
static inline int with_dtype(int32_t dtype, const char* name, F&& f) {
  switch (dtype) {
    case TGS_F32: return f(float{});
    case TGS_BF16: return f(bf16_t{});
    case TGS_F16: return f(f16_t{});
  }
  tgs_set_error("%s: dtype must be 0 (float32), 1 (bfloat16) or 2 (float16), got %d", name, dtype);
  return TGS_ERR_ARG;
}
