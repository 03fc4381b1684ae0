// Dropout from a counter-based generator: the mask is a function of (seed, offset,
// element index), so the backward computes it again and it is never stored.
//
//   t = round(65536 p), scale = 65536 / (65536 - t)
//   y_i = (draw_i >= t ? x_i scale : 0) + residual_i
//
// draw_i is 16 bits of Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random
// numbers: as easy as 1, 2, 3", 2011): block i >> 3 of the 64-bit stream `offset`
// under the key `seed`, word (i & 7) >> 1, low half first.  The share dropped is
// exactly t / 65536 and the scale is that share's own, so the expectation is exact
// whatever p rounds to; 32-bit draws would halve what a block of the generator
// yields (20 wide multiplications) for a resolution of p that no user sets.
// A dropped value is not read into the result: infinities and NaN there give 0.
//
// Memory bound: x is read and y written once, 16 bytes a lane where the pointers allow,
// and a thread's eight values are one block of the generator, so no draw is thrown away
// and the generator's arithmetic runs under the loads.  4M rows of 64 bfloat16 with a
// residual (1.54 GB) take 264 us, 5.8 TB/s; 300k of 59 float32 (142 MB) 26 us, 5.5 TB/s.
#include "decoder_common.cuh"
#include "philox.cuh"

// One thread per block of eight values.  VEC: every pointer is 16-byte aligned.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) dropout_kernel(uint64_t n, const T* __restrict__ x,
                                                      const T* __restrict__ residual,
                                                      T* __restrict__ y, uint32_t threshold,
                                                      float scale, uint64_t seed,
                                                      uint64_t offset) {
  using V = Vec16<T>;
  const uint64_t groups = (n + 7) / 8, stride = (uint64_t)gridDim.x * blockDim.x;
  for (uint64_t g = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; g < groups; g += stride) {
    uint32_t c[4] = {(uint32_t)g, (uint32_t)(g >> 32), (uint32_t)offset, (uint32_t)(offset >> 32)};
    const uint64_t i0 = g * 8;
    const bool whole = i0 + 8 <= n;
    T in[8], res[8];
    if (VEC && whole) {
#pragma unroll
      for (int k = 0; k < 8 / V::N; ++k) {
        *(V*)(in + k * V::N) = ((const V*)(x + i0))[k];
        if (residual) *(V*)(res + k * V::N) = ((const V*)(residual + i0))[k];
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const bool ok = i0 + k < n;
        in[k] = ok ? x[i0 + k] : (T)0.f;
        res[k] = residual && ok ? residual[i0 + k] : (T)0.f;
      }
    }
    philox4x32_10(c, (uint32_t)seed, (uint32_t)(seed >> 32));
    T out[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t draw = philox_draw16(c, k);
      float v = draw >= threshold ? to_f32(in[k]) * scale : 0.f;
      if (residual) v += to_f32(res[k]);
      out[k] = from_f32<T>(v);
    }
    if (VEC && whole) {
#pragma unroll
      for (int k = 0; k < 8 / V::N; ++k) ((V*)(y + i0))[k] = *(V*)(out + k * V::N);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (i0 + k < n) y[i0 + k] = out[k];
    }
  }
}

extern "C" int tgs_dropout(uint64_t n, int32_t dtype, const void* x, const void* residual, void* y,
                           uint32_t threshold, uint64_t seed, uint64_t offset,
                           hipStream_t stream) {
  return with_dtype(dtype, "tgs_dropout", [&](auto tag) -> int {
    using T = decltype(tag);
    TGS_CHECK_ARG(threshold <= 65536, "tgs_dropout: threshold %u is above 65536", threshold);
    if (n == 0) return TGS_OK;
    TGS_CHECK_ARG(x && y, "tgs_dropout: null pointer");
    const float scale = threshold < 65536 ? (float)(65536.0 / (65536 - threshold)) : 0.f;
    const uint64_t blocks = std::min<uint64_t>((n + 2047) / 2048, 1 << 20);
    const bool vec = aligned16((const T*)x, 0) && aligned16((const T*)y, 0) &&
                     aligned16((const T*)residual, 0);
    const auto launch = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), 0, stream, n, (const T*)x,
                         (const T*)residual, (T*)y, threshold, scale, seed, offset);
    };
    if (vec)
      launch(dropout_kernel<T, true>);
    else
      launch(dropout_kernel<T, false>);
    TGS_RETURN_LAUNCH("tgs_dropout");
  });
}
