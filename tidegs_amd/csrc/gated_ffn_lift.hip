// The powers of two that half precision's h, dg and du are multiplied by in the backward
// (gated_ffn.cuh): every tensor's largest finite magnitude, then bounds from these.
//
// Bound by memory: x, dy and the weights are read once more, 16 bytes a lane; x and dy of 1M
// rows of 64 (256 MB) take 48 us, 5.3 TB/s, and the powers 5, of 610 for the block 64-256-64, both ways.
#include "gated_ffn.cuh"

#define LIFT_TENSORS 7

struct PeakJob {
  const f16_t* p;
  int64_t rows, pitch, end;  // end: one past the last value
  int32_t cols, wide;        // wide: rows start on 16 bytes
  uint32_t blocks;           // of the launch, up to and with this job's
};
struct PeakJobs {
  PeakJob job[LIFT_TENSORS];
};

typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));

// Finite halves without their signs, less infinity's bits, are 0x8400 .. 0xFFFF in the order of
// their magnitudes; what is not finite is below them.
#define HALF_INFINITY 0x7C00u
#define HALF_FINITE 0x8400u

__global__ void __launch_bounds__(256) ffn_peak_kernel(PeakJobs jobs, float* __restrict__ peaks) {
  constexpr int U = 4;  // rows that a thread has in flight
  __shared__ uint32_t s[4];
  int k = 0;
  uint32_t first = 0;
  while (blockIdx.x >= jobs.job[k].blocks) first = jobs.job[k++].blocks;
  const PeakJob& job = jobs.job[k];
  const int32_t chunks = (job.cols + 7) / 8;
  int32_t lanes = 1;  // of a row
  while (lanes < chunks && lanes < 256) lanes *= 2;
  const int64_t per = 256 / lanes, step = per * (job.blocks - first);
  u16x8 most = 0;
  for (int64_t r0 = (int64_t)(blockIdx.x - first) * per + threadIdx.x / lanes; r0 < job.rows;
       r0 += step * U) {
    for (int32_t c = (threadIdx.x % lanes) * 8; c < job.cols; c += lanes * 8) {
      u16x8 v[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int64_t at = (r0 + i * step < job.rows ? r0 + i * step : r0) * job.pitch + c;
        const uint16_t* p = (const uint16_t*)job.p + at;
        if (job.wide && at + 8 <= job.end) {  // (with what lies between two rows)
          v[i] = *(const u16x8*)p;
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[i][e] = c + e < job.cols && at + e < job.end ? p[e] : 0;
        }
      }
      if (c + 8 > job.cols)
#pragma unroll
        for (int i = 0; i < U; ++i)
#pragma unroll
          for (int e = 0; e < 8; ++e) v[i][e] = c + e < job.cols ? v[i][e] : 0;
#pragma unroll
      for (int i = 0; i < U; ++i)
        most = __builtin_elementwise_max(most, (u16x8)((v[i] & (uint16_t)0x7FFF) - (uint16_t)HALF_INFINITY));
    }
  }
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) m = max(m, (uint32_t)most[e]);
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) m = max(m, (uint32_t)__shfl_xor((int)m, off, 64));
  if (threadIdx.x % 64 == 0) s[threadIdx.x / 64] = m;
  __syncthreads();
  if (threadIdx.x == 0) {
    m = max(max(s[0], s[1]), max(s[2], s[3]));
    union {
      uint16_t bits;
      f16_t h;
    } u;
    u.bits = m >= HALF_FINITE ? (uint16_t)(m + HALF_INFINITY) : 0;
    peaks[blockIdx.x] = (float)u.h;
  }
}

// The largest power of two, from 1 on, that keeps what `bound` bounds below 2^15 (half ends at
// 65504).
__device__ static inline int lift_exponent(float bound) {
  const int e = (int)(__float_as_uint(bound) >> 23) - 127;  // bound < 2^(e + 1)
  return min(max(14 - e, 0), 60);
}

// A wavefront per tensor, in the order x, dy, Wg, Wu, Wd, bg, bu.
__global__ void __launch_bounds__(64 * LIFT_TENSORS) ffn_lift_kernel(PeakJobs jobs,
                                                                    const float* __restrict__ peaks,
                                                                    float width, float out, Lift* lift) {
  __shared__ float s[LIFT_TENSORS];
  const uint32_t k = threadIdx.x / 64;
  float m = 0.f;
  for (uint32_t b = (k ? jobs.job[k - 1].blocks : 0) + threadIdx.x % 64; b < jobs.job[k].blocks; b += 64)
    m = fmaxf(m, peaks[b]);
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
  if (threadIdx.x % 64 == 0) s[k] = m;
  __syncthreads();
  if (threadIdx.x) return;
  // |g| and |u|; |act(g)| <= |g|, |act'(g)| <= 1.13
  const float gu = width * s[0] * fmaxf(s[2], s[3]) + fmaxf(s[5], s[6]);
  const int h = lift_exponent(gu * gu), d = lift_exponent(1.13f * out * s[1] * s[4] * gu);
  *lift = {ldexpf(1.f, h), ldexpf(1.f, -h), ldexpf(1.f, d), ldexpf(1.f, -d)};
}

void ffn_lift(const FfnCall& c, Lift* lift, float* peaks, hipStream_t stream) {
  PeakJobs jobs;
  int n = 0;
  uint32_t blocks = 0;
  const auto add = [&](const void* p, int64_t rows, int64_t cols, int64_t pitch) {
    const int64_t end = p ? (rows - 1) * pitch + cols : 0;
    if (pitch == cols) {  // dense: rows of any length
      pitch = cols = 2048;
      rows = tiles(end, cols);
    }
    // (none shorter than 16 values a thread)
    blocks += (uint32_t)std::min<int64_t>(tiles(end, 4096), LIFT_BLOCKS);
    jobs.job[n++] = PeakJob{(const f16_t*)p, p ? rows : 0, pitch, end, (int32_t)cols,
                            aligned16((const f16_t*)p, pitch), blocks};
  };
  add(c.x, c.rows, c.width, c.x_pitch);
  add(c.dy, c.rows, c.out, c.dy_pitch);
  add(c.wg, c.hidden, c.width, c.width);
  add(c.wu, c.hidden, c.width, c.width);
  add(c.wd, c.out, c.hidden, c.hidden);
  add(c.bg, 1, c.hidden, c.hidden);
  add(c.bu, 1, c.hidden, c.hidden);
  hipLaunchKernelGGL(ffn_peak_kernel, dim3(blocks), dim3(256), 0, stream, jobs, peaks);
  hipLaunchKernelGGL(ffn_lift_kernel, dim3(1), dim3(64 * LIFT_TENSORS), 0, stream, jobs, peaks,
                     (float)c.width, (float)c.out, lift);
}
