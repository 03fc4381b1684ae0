// Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3",
// 2011): four random words of a counter and a key, ten rounds of two wide products.
#pragma once

#include "tgs_common.cuh"

__device__ __forceinline__ void philox4x32_10(uint32_t c[4], uint32_t k0, uint32_t k1) {
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = (uint64_t)c[0] * 0xD2511F53u, b = (uint64_t)c[2] * 0xCD9E8D57u;
    c[0] = (uint32_t)(b >> 32) ^ c[1] ^ k0;
    c[2] = (uint32_t)(a >> 32) ^ c[3] ^ k1;
    c[1] = (uint32_t)b;
    c[3] = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
}

// Draw k of a block's eight: 16 bits of word k >> 1, low half first.
__device__ __forceinline__ uint32_t philox_draw16(const uint32_t c[4], int k) {
  return k & 1 ? c[k >> 1] >> 16 : c[k >> 1] & 0xFFFFu;
}
