// Loads and stores of consecutive values on their elements' alignment alone: the memory
// system takes 16-byte accesses at any address, so views cut out of a buffer anywhere, or
// rows at an odd pitch, are read as wide as aligned ones.
#pragma once

#include "decoder_common.cuh"

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef u32x4 u32x4_at1 __attribute__((aligned(1)));
typedef u32x2 u32x2_at1 __attribute__((aligned(1)));
typedef uint32_t u32_at1 __attribute__((aligned(1)));

// BYTES (2, 4, 8, or a multiple of 16) from p to w or back.
template <int BYTES>
__device__ __forceinline__ void load_bytes(void* w, const void* p) {
  if constexpr (BYTES % 16 == 0) {
#pragma unroll
    for (int k = 0; k < BYTES / 16; ++k) ((u32x4*)w)[k] = ((const u32x4_at1*)p)[k];
  } else if constexpr (BYTES == 8) {
    *(u32x2*)w = *(const u32x2_at1*)p;
  } else if constexpr (BYTES == 4) {
    *(uint32_t*)w = *(const u32_at1*)p;
  } else {
    *(uint16_t*)w = *(const uint16_t*)p;
  }
}
template <int BYTES>
__device__ __forceinline__ void store_bytes(void* p, const void* w) {
  if constexpr (BYTES % 16 == 0) {
#pragma unroll
    for (int k = 0; k < BYTES / 16; ++k) ((u32x4_at1*)p)[k] = ((const u32x4*)w)[k];
  } else if constexpr (BYTES == 8) {
    *(u32x2_at1*)p = *(const u32x2*)w;
  } else if constexpr (BYTES == 4) {
    *(u32_at1*)p = *(const uint32_t*)w;
  } else {
    *(uint16_t*)p = *(const uint16_t*)w;
  }
}
// The same, for values that nothing reads soon: they do not displace what the caches hold.
template <int BYTES>
__device__ __forceinline__ void store_bytes_once(void* p, const void* w) {
  // (of two stores in an if and its else the compiler would make one, a plain one)
  asm volatile("");
  if constexpr (BYTES % 16 == 0) {
#pragma unroll
    for (int k = 0; k < BYTES / 16; ++k)
      __builtin_nontemporal_store(((const u32x4*)w)[k], (u32x4_at1*)p + k);
  } else if constexpr (BYTES == 8) {
    __builtin_nontemporal_store(*(const u32x2*)w, (u32x2_at1*)p);
  } else {
    store_bytes<BYTES>(p, w);
  }
  asm volatile("");
}

// N values of T in registers.
template <typename T, int N>
struct alignas(N * sizeof(T) >= 16 ? 16 : N * sizeof(T)) Run {
  T v[N];
  __device__ __forceinline__ void load(const T* p) { load_bytes<N * sizeof(T)>(v, p); }
  __device__ __forceinline__ void store(T* p) const { store_bytes<N * sizeof(T)>(p, v); }
  __device__ __forceinline__ void store_once(T* p) const {
    store_bytes_once<N * sizeof(T)>(p, v);
  }
  // Makes the compiler take the values for new ones: what was computed from them is computed
  // again rather than kept in registers.
  __device__ __forceinline__ void forget() {
    if constexpr (sizeof(v) % 4 == 0) {
#pragma unroll
      for (int k = 0; k < (int)sizeof(v) / 4; ++k) asm volatile("" : "+v"(((uint32_t*)v)[k]));
    } else {
      asm volatile("" : "+v"(*(uint16_t*)v));
    }
  }
};
