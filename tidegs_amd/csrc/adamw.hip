// AdamW over many tensors at once, and the common norm of many gradients.
//
//   g' = g min(1, max_norm / (norm + 1e-6))       (where a norm is given)
//   m' = b1 m + (1 - b1) g',  v' = b2 v + (1 - b2) g'^2
//   p' = p (1 - lr wd) - lr / (1 - b1^t) m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
//
// Memory bound: p, m and v are read and written once and g is read once, 28 bytes a value in
// 32 bits.  The tables of 4M Gaussians (236M values, 6.6 GB) take 1215 us, 5.4 TB/s; 256M values
// of bfloat16 with states of 8 bits (2.6 GB, 51 instructions a value) 460 us, 5.6 TB/s.  A launch
// takes up to 56 tensors, described in its arguments (no table in memory: nothing to upload,
// nothing that a captured graph would have to keep), cut into chunks of 2048 values; a lane has
// eight values next to each other of each buffer.
//
// States of 8 bits: blocks of 128 values (16 lanes) with a scale each.  m is kept in e4m3, to
// nearest; v in e5m2, stochastically: v moves by a thousandth a step, far below half a step of
// any 8-bit float, and rounded to nearest it would stay where it is for good, while this way
// its expectation is the moving average itself.  (m moves by a tenth, nearest rounding does
// not hold it.)  Scales are powers of two, so that a new scale moves no value off its grid,
// and put a block's largest value right below the type's (BORDER).  A positive v never
// becomes 0: what it divides would explode.
// 16-bit parameters are rounded stochastically as well: a step is mostly below half of their
// last bit.  The draws are 16 bits a value of Philox4x32-10 with key `seed` and counter
// (index >> 3, step, tensor's number): the same call gives the same bits.  A value's one draw
// serves both its v and its parameter: each is unbiased, and nothing multiplies their errors.
#include "decoder_common.cuh"
#include "philox.cuh"
#include "vector_io.cuh"

#include <math.h>

#include "../../include/tidegs_amd.h"

#define ADAMW_TENSORS 56  // of a launch, in 4 KB of arguments
#define ADAMW_GROUPS 4
#define ADAMW_CHUNK 2048  // values of a workgroup at once
#define ADAMW_BLOCK 128   // values that share a scale
#define M_TOP 8           // scales bring a block's largest value to BORDER / 2 .. BORDER times
#define V_TOP 15          // 2^TOP; the types end at 1.75 times that

// 1.7320508's mantissa.  Not 1.75 and not 1: moments of few bits, averaged with decimal
// shares, often lie exactly there, and an average's last bit would decide the scale.
#define BORDER_BITS 0x5DB3D7u

struct AdamwGroup {
  float decay, step_size, root;  // 1 - lr wd, lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
  float beta1, one_m_beta1, beta2, one_m_beta2, eps;
  uint32_t step;
  const float4* live;  // {decay, step_size, root, step} on the device, or null
};

struct AdamwTensor {
  void* p;
  const void* g;
  void* m;
  void* v;
  float* m_scale;
  float* v_scale;
  uint64_t n;
  uint32_t number, group;
};

struct AdamwBatch {
  uint32_t count;
  uint32_t first[ADAMW_TENSORS + 1];  // each tensor's first chunk; the number of chunks
  AdamwTensor t[ADAMW_TENSORS];
  AdamwGroup group[ADAMW_GROUPS];
};
static_assert(sizeof(AdamwBatch) <= 4096 - 64, "arguments of a launch");

// The tensor whose chunk this is: the last that begins at or before it.
template <typename Batch>
__device__ __forceinline__ uint32_t tensor_of(const Batch& b, uint32_t chunk) {
  static_assert(sizeof(b.t) / sizeof(b.t[0]) <= 64, "a lane each");
  const uint32_t lane = threadIdx.x & 63;
  const bool at = lane < b.count && b.first[lane < b.count ? lane : 0] <= chunk;
  return __builtin_amdgcn_readfirstlane(__popcll(tgs_ballot(at)) - 1);
}

// Eight consecutive values (tensors may be cut out of a flat buffer anywhere); past the end of
// the tensor zeros, and nothing stored.
template <typename T>
struct Eight {
  union {
    uint32_t w[8 * sizeof(T) / 4];
    T v[8];
  };
  template <bool FULL>
  __device__ __forceinline__ void load(const T* p, uint64_t i, uint64_t n) {
    if (FULL || i + 8 <= n) {
      load_bytes<8 * sizeof(T)>(w, p + i);
    } else {
#pragma unroll
      for (int k = 0; k < (int)(8 * sizeof(T) / 4); ++k) w[k] = 0;
      if (i < n) {  // (one lane of a tensor)
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (i + k < n) v[k] = p[i + k];
      }
    }
  }
  template <bool FULL>
  __device__ __forceinline__ void store(T* p, uint64_t i, uint64_t n) const {
    if (FULL || i + 8 <= n) {
      store_bytes<8 * sizeof(T)>(p + i, w);
    } else if (i < n) {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (i + k < n) p[i + k] = v[k];
    }
  }
};

// The largest finite magnitude of a block's 16 lanes, as bits (NaN never is the larger one;
// infinities are looked for only where there is one).
__device__ __forceinline__ uint32_t block_most(const float (&x)[8]) {
  const auto over_block = [](uint32_t most) {
    most = max(most, tgs_dpp_u32<0xB1>(most));   // quad_perm [1,0,3,2]
    most = max(most, tgs_dpp_u32<0x4E>(most));   // quad_perm [2,3,0,1]
    most = max(most, tgs_dpp_u32<0x141>(most));  // row_half_mirror
    return max(most, tgs_dpp_u32<0x140>(most));  // row_mirror
  };
  float most = 0.f;
#pragma unroll
  for (int k = 0; k < 8; k += 2) most = fmaxf(most, fmaxf(fabsf(x[k]), fabsf(x[k + 1])));
  if (__builtin_expect(tgs_ballot(most == INFINITY) != 0, 0)) {  // (uniform: all lanes go on)
    most = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) most = fmaxf(most, fabsf(x[k]) == INFINITY ? 0.f : fabsf(x[k]));
  }
  return over_block(__float_as_uint(most));
}

// The power of two of a block's scale; 2^-120 where all is zero.
__device__ __forceinline__ int scale_exponent(uint32_t most, int top) {
  const int e = (int)((most + (0x800000u - BORDER_BITS)) >> 23) - 127 - top;
  return most ? min(max(e, -120), 120) : -120;
}

__device__ __forceinline__ float power_of_two(int e) {
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

template <int FORMAT>  // 0: e4m3, 1: e5m2
__device__ __forceinline__ void decode8(const uint32_t (&w)[2], float scale, float (&x)[8]) {
#pragma unroll
  for (int k = 0; k < 8; k += 2) {
    const int word = (int)w[k >> 2];
    const auto two = FORMAT ? (k & 2 ? __builtin_amdgcn_cvt_pk_f32_bf8(word, true)
                                     : __builtin_amdgcn_cvt_pk_f32_bf8(word, false))
                            : (k & 2 ? __builtin_amdgcn_cvt_pk_f32_fp8(word, true)
                                     : __builtin_amdgcn_cvt_pk_f32_fp8(word, false));
    x[k] = two[0] * scale;
    x[k + 1] = two[1] * scale;
  }
}

// e4m3 to nearest even; infinities (which it has none of) become NaN.
__device__ __forceinline__ void encode_m(const float (&x)[8], float inverse, uint32_t (&w)[2]) {
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const float* y = x + 4 * k;
    const int low = __builtin_amdgcn_cvt_pk_fp8_f32(y[0] * inverse, y[1] * inverse, 0, false);
    w[k] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2] * inverse, y[3] * inverse, low, true);
  }
}

// Stochastic rounding by the hardware's conversions: what lies below the last bit is rounded
// away from zero where it and the upper bits of a random word, both as parts of one, reach one
// (21 bits of it for e5m2, 16 for bfloat16, 13 for half; all values of e5m2 and bfloat16 and
// half's normal ones agreed with that rule in integer arithmetic).  The draw stands in the
// upper half of the word.
__device__ __forceinline__ uint32_t draw_word(const uint32_t c[4], int k) {
  return k & 1 ? c[k >> 1] & 0xFFFF0000u : c[k >> 1] << 16;
}

// e5m2; the word's next bit centres the draw.  A positive value becomes 2^-16 at least.
__device__ __forceinline__ void encode_v(const float (&v)[8], float inverse, const uint32_t c[4],
                                         uint32_t (&w)[2]) {
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    int word = 0;
    float x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float y = v[4 * k + e] * inverse;
      x[e] = y > 0.f ? fmaxf(y, 0x1p-16f) : y;  // (NaN stays)
    }
    word = __builtin_amdgcn_cvt_sr_bf8_f32(x[0], draw_word(c, 4 * k) | 0x8000u, word, 0);
    word = __builtin_amdgcn_cvt_sr_bf8_f32(x[1], draw_word(c, 4 * k + 1) | 0x8000u, word, 1);
    word = __builtin_amdgcn_cvt_sr_bf8_f32(x[2], draw_word(c, 4 * k + 2) | 0x8000u, word, 2);
    word = __builtin_amdgcn_cvt_sr_bf8_f32(x[3], draw_word(c, 4 * k + 3) | 0x8000u, word, 3);
    w[k] = (uint32_t)word;
  }
}

// Eight parameters in their type.
__device__ __forceinline__ void encode_p(const float (&p)[8], const uint32_t*, Eight<float>& out) {
#pragma unroll
  for (int k = 0; k < 8; ++k) out.v[k] = p[k];
}
typedef bf16_t bf16x2 __attribute__((ext_vector_type(2)));
typedef f16_t f16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void encode_p(const float (&p)[8], const uint32_t* c,
                                         Eight<bf16_t>& out) {
#pragma unroll
  for (int k = 0; k < 8; k += 2) {
    bf16x2 two = {(bf16_t)0.f, (bf16_t)0.f};
    two = __builtin_amdgcn_cvt_sr_bf16_f32(two, p[k], draw_word(c, k), false);
    two = __builtin_amdgcn_cvt_sr_bf16_f32(two, p[k + 1], draw_word(c, k + 1), true);
    out.w[k / 2] = __builtin_bit_cast(uint32_t, two);
  }
}
__device__ __forceinline__ void encode_p(const float (&p)[8], const uint32_t* c,
                                         Eight<f16_t>& out) {
#pragma unroll
  for (int k = 0; k < 8; k += 2) {
    f16x2 two = {(f16_t)0.f, (f16_t)0.f};
    two = __builtin_amdgcn_cvt_sr_f16_f32(two, p[k], draw_word(c, k), false);
    two = __builtin_amdgcn_cvt_sr_f16_f32(two, p[k + 1], draw_word(c, k + 1), true);
    out.w[k / 2] = __builtin_bit_cast(uint32_t, two);
  }
}

template <typename T, int BITS, bool FULL>
__device__ __forceinline__ void adamw_eight(const AdamwTensor& t, const AdamwGroup& h, uint64_t i,
                                            float clip, float decay, float step_size, float root,
                                            uint32_t step, uint64_t seed) {
#pragma clang fp contract(off)
  constexpr bool EIGHT = BITS == 8;
  using S = typename std::conditional<EIGHT, uint8_t, float>::type;
  Eight<T> p8, g8;
  Eight<S> m8, v8;
  p8.template load<FULL>((const T*)t.p, i, t.n);
  g8.template load<FULL>((const T*)t.g, i, t.n);
  m8.template load<FULL>((const S*)t.m, i, t.n);
  v8.template load<FULL>((const S*)t.v, i, t.n);
  float m[8], v[8];
  const bool in = FULL || i < t.n;
  if constexpr (EIGHT) {
    decode8<0>(m8.w, in ? t.m_scale[i / ADAMW_BLOCK] : 0.f, m);
    decode8<1>(v8.w, in ? t.v_scale[i / ADAMW_BLOCK] : 0.f, v);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) m[k] = m8.v[k], v[k] = v8.v[k];
  }
  uint32_t c[4] = {(uint32_t)(i >> 3), (uint32_t)(i >> 35), step, t.number};
  if constexpr (EIGHT || sizeof(T) == 2) philox4x32_10(c, (uint32_t)seed, (uint32_t)(seed >> 32));
  float p[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float g = to_f32(g8.v[k]) * clip;
    m[k] = h.beta1 * m[k] + h.one_m_beta1 * g;
    v[k] = h.beta2 * v[k] + h.one_m_beta2 * g * g;
    p[k] = to_f32(p8.v[k]) * decay;
  }
  // The hardware's root and reciprocal are off by one unit, and take what is below 2^-126 for
  // zero: 2^-63 root at most, 2^-25 of this eps.  (With the exact forms, and conversions and maxima
  // in integer arithmetic, 256M values of bfloat16 with states of 8 bits took 586 us.)
  if (h.eps >= root * 0x1p-38f) {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      p[k] -= m[k] * __builtin_amdgcn_rcpf(__builtin_amdgcn_sqrtf(v[k]) * root + h.eps) * step_size;
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) p[k] -= m[k] / (sqrtf(v[k]) * root + h.eps) * step_size;
  }
  encode_p(p, c, p8);
  p8.template store<FULL>((T*)t.p, i, t.n);
  if constexpr (EIGHT) {
    const int me = scale_exponent(block_most(m), M_TOP), ve = scale_exponent(block_most(v), V_TOP);
    encode_m(m, power_of_two(-me), m8.w);
    encode_v(v, power_of_two(-ve), c, v8.w);
    if (in && threadIdx.x % 16 == 0) {
      t.m_scale[i / ADAMW_BLOCK] = power_of_two(me);
      t.v_scale[i / ADAMW_BLOCK] = power_of_two(ve);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) m8.v[k] = m[k], v8.v[k] = v[k];
  }
  m8.template store<FULL>((S*)t.m, i, t.n);
  v8.template store<FULL>((S*)t.v, i, t.n);
}

template <typename T, int BITS>
__global__ void __launch_bounds__(256) adamw_kernel(AdamwBatch b, uint64_t seed,
                                                    const float* __restrict__ norm,
                                                    float max_norm) {
  float clip = 1.f;
  if (norm) {
    const double share = (double)max_norm / ((double)*norm + 1e-6);
    clip = share >= 1.0 ? 1.f : (float)share;  // (NaN stays)
  }
  for (uint32_t chunk = blockIdx.x; chunk < b.first[b.count]; chunk += gridDim.x) {
    const uint32_t k = tensor_of(b, chunk);
    const AdamwTensor& t = b.t[k];
    const AdamwGroup& h = b.group[t.group];
    float decay = h.decay, step_size = h.step_size, root = h.root;
    uint32_t step = h.step;
    if (h.live) {
      const float4 live = *h.live;
      decay = live.x, step_size = live.y, root = live.z, step = __float_as_uint(live.w);
    }
    const uint64_t base = (uint64_t)(chunk - b.first[k]) * ADAMW_CHUNK;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const uint64_t i = base + threadIdx.x * 8;
    if (base + (wave + 1) * 512 <= t.n)
      adamw_eight<T, BITS, true>(t, h, i, clip, decay, step_size, root, step, seed);
    else if (base + wave * 512 < t.n)  // (a block's lanes are in one wavefront: all or none)
      adamw_eight<T, BITS, false>(t, h, i, clip, decay, step_size, root, step, seed);
  }
}

// Steps counted on the device (a captured graph's): one thread a group.
struct AdamwSchedules {
  tgs_adamw_group g[32];
};

__global__ void __launch_bounds__(64) adamw_begin_kernel(uint32_t count, AdamwSchedules s,
                                                         float4* __restrict__ live) {
  const uint32_t k = threadIdx.x;
  if (k >= count) return;
  const tgs_adamw_group& g = s.g[k];
  const int64_t t = ++*g.step_device;
  const double lr = g.lr_device ? (double)*g.lr_device : g.lr;
  live[k] = make_float4((float)(1.0 - lr * g.weight_decay),
                        (float)(lr / (1.0 - pow(g.beta1, (double)t))),
                        (float)(1.0 / sqrt(1.0 - pow(g.beta2, (double)t))),
                        __uint_as_float((uint32_t)t));
}

static AdamwGroup prepared(const tgs_adamw_group& g, const float4* live) {
  const double t = (double)g.step;
  AdamwGroup h;
  h.decay = (float)(1.0 - g.lr * g.weight_decay);
  h.step_size = live ? 0.f : (float)(g.lr / (1.0 - pow(g.beta1, t)));
  h.root = live ? 0.f : (float)(1.0 / sqrt(1.0 - pow(g.beta2, t)));
  h.beta1 = (float)g.beta1;
  h.one_m_beta1 = (float)(1.0 - g.beta1);
  h.beta2 = (float)g.beta2;
  h.one_m_beta2 = (float)(1.0 - g.beta2);
  h.eps = (float)g.eps;
  h.step = (uint32_t)g.step;
  h.live = live;
  return h;
}

static uint64_t chunks_of(uint64_t n) { return (n + ADAMW_CHUNK - 1) / ADAMW_CHUNK; }

extern "C" uint64_t tgs_adamw_workspace_size(uint32_t n_groups) {
  return (uint64_t)n_groups * sizeof(float4);
}

// Launches over the tensors of one type: batches of as many tensors and groups as a launch's
// arguments hold.
template <typename T>
static void adamw_launches(uint32_t n_tensors, const tgs_adamw_tensor* tensors,
                           const tgs_adamw_group* groups, int32_t dtype, int32_t state_bits,
                           uint64_t seed, const float* grad_norm, float max_norm,
                           const float4* lives, hipStream_t stream) {
  AdamwBatch b = {};
  uint32_t used = 0, of[ADAMW_GROUPS];  // the batch's groups, as the caller numbers them
  uint64_t chunks = 0;
  const auto flush = [&] {
    if (b.count) {
      b.first[b.count] = (uint32_t)chunks;
      const dim3 grid((uint32_t)std::min<uint64_t>(chunks, 1u << 20));
      if (state_bits == 8)
        hipLaunchKernelGGL((adamw_kernel<T, 8>), grid, dim3(256), 0, stream, b, seed, grad_norm,
                           max_norm);
      else
        hipLaunchKernelGGL((adamw_kernel<T, 32>), grid, dim3(256), 0, stream, b, seed, grad_norm,
                           max_norm);
    }
    b.count = used = 0;
    chunks = 0;
  };
  for (uint32_t k = 0; k < n_tensors; ++k) {
    const tgs_adamw_tensor& t = tensors[k];
    if (t.n == 0 || t.dtype != dtype) continue;
    uint32_t h = std::find(of, of + used, t.group) - of;
    if (b.count == ADAMW_TENSORS || (h == used && used == ADAMW_GROUPS) ||
        chunks + chunks_of(t.n) > 0x7FFFFFFFull) {
      flush();
      h = 0;
    }
    if (h == used) {
      of[used] = t.group;
      b.group[used++] = prepared(groups[t.group], lives ? lives + t.group : nullptr);
    }
    b.first[b.count] = (uint32_t)chunks;
    b.t[b.count++] = {t.param, t.grad, t.exp_avg, t.exp_avg_sq, t.exp_avg_scale,
                      t.exp_avg_sq_scale, t.n, t.number, h};
    chunks += chunks_of(t.n);
  }
  flush();
}

extern "C" int tgs_adamw(uint32_t n_tensors, const tgs_adamw_tensor* tensors, uint32_t n_groups,
                         const tgs_adamw_group* groups, int32_t state_bits, uint64_t seed,
                         const float* grad_norm, float max_norm, void* workspace,
                         uint64_t workspace_bytes, hipStream_t stream) {
  TGS_CHECK_ARG(state_bits == 32 || state_bits == 8, "tgs_adamw: states of %d bits", state_bits);
  if (n_tensors == 0) return TGS_OK;
  TGS_CHECK_ARG(tensors && groups && n_groups, "tgs_adamw: null pointer");
  TGS_CHECK_ARG(!grad_norm || max_norm > 0.f, "tgs_adamw: max_norm must be positive");
  const bool live = groups[0].step_device != nullptr;
  for (uint32_t k = 0; k < n_groups; ++k) {
    const tgs_adamw_group& g = groups[k];
    TGS_CHECK_ARG((g.step_device != nullptr) == live && (live || !g.lr_device),
                  "tgs_adamw: steps of all groups are counted on the device, or of none");
    TGS_CHECK_ARG(live || (g.step >= 1 && g.step < (1ull << 32)), "tgs_adamw: step %llu",
                  (unsigned long long)g.step);
    TGS_CHECK_ARG(g.beta1 >= 0 && g.beta1 < 1 && g.beta2 >= 0 && g.beta2 < 1 && g.eps >= 0,
                  "tgs_adamw: betas lie in [0, 1), eps is not negative");
  }
  bool any = live;  // (counts advance even if every tensor is empty)
  for (uint32_t k = 0; k < n_tensors; ++k) {
    const tgs_adamw_tensor& t = tensors[k];
    any |= t.n > 0;
    TGS_CHECK_ARG(t.dtype >= TGS_F32 && t.dtype <= TGS_F16,
                  "tgs_adamw: dtype must be 0 (float32), 1 (bfloat16) or 2 (float16), got %d",
                  t.dtype);
    TGS_CHECK_ARG(t.group < n_groups, "tgs_adamw: group %u of %u", t.group, n_groups);
    TGS_CHECK_ARG(t.n < (1ull << 41), "tgs_adamw: %llu values", (unsigned long long)t.n);
    TGS_CHECK_ARG(t.n == 0 || (t.param && t.grad && t.exp_avg && t.exp_avg_sq &&
                               (state_bits == 32 || (t.exp_avg_scale && t.exp_avg_sq_scale))),
                  "tgs_adamw: null pointer in tensor %u", k);
  }
  if (!any) return TGS_OK;
  float4* lives = live ? (float4*)workspace : nullptr;
  if (live) {
    if (workspace_bytes < tgs_adamw_workspace_size(n_groups)) {
      tgs_set_error("tgs_adamw: workspace too small");
      return TGS_ERR_WORKSPACE;
    }
    TGS_CHECK_ARG(workspace && (uintptr_t)workspace % 16 == 0,
                  "tgs_adamw: the workspace starts on 16 bytes");
    for (uint32_t k = 0; k < n_groups; k += 32) {
      AdamwSchedules s = {};
      const uint32_t count = std::min(n_groups - k, 32u);
      std::copy(groups + k, groups + k + count, s.g);
      hipLaunchKernelGGL(adamw_begin_kernel, dim3(1), dim3(64), 0, stream, count, s, lives + k);
    }
  }
  for (int32_t dtype = TGS_F32; dtype <= TGS_F16; ++dtype)
    with_dtype(dtype, "tgs_adamw", [&](auto tag) {
      adamw_launches<decltype(tag)>(n_tensors, tensors, groups, dtype, state_bits, seed, grad_norm,
                                    max_norm, lives, stream);
      return TGS_OK;
    });
  TGS_RETURN_LAUNCH("tgs_adamw");
}

// ---------------------------------------------------------------------------
// The common norm: sqrt(sum over all tensors of g^2), in 64 bits (the square of a 32-bit value
// may leave their range, and a sum of a hundred million keeps what 32 would lose), joined in a
// fixed order.  12.6M floats: 10 us (5.2 TB/s) and 2 for the join.
// ---------------------------------------------------------------------------

#define NORM_TENSORS 64
#define NORM_CHUNK 8192
#define NORM_PARTS 2048  // workgroups of a launch
// Chunks that one workgroup sums alone: up to there as fast as two launches (19 to 21 us a call
// that is waited for), and 2.5 us less of the host's time.
#define NORM_SINGLE 8

struct NormBatch {
  uint32_t count;
  uint32_t first[NORM_TENSORS + 1];
  struct {
    const void* p;
    uint64_t n;
  } t[NORM_TENSORS];
};

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int off = 32; off; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

template <int WAVES>
__device__ __forceinline__ double group_sum64(double v) {
  __shared__ double s[WAVES];
  v = wave_sum64(v);
  if (threadIdx.x % 64 == 0) s[threadIdx.x / 64] = v;
  __syncthreads();
  double sum = 0;
#pragma unroll
  for (int k = 0; k < WAVES; ++k) sum += s[k];
  return sum;
}

// One workgroup writes the norm itself.
template <typename T>
__global__ void __launch_bounds__(256) norm_kernel(NormBatch b, double* __restrict__ parts,
                                                   float* __restrict__ norm) {
  double sum = 0;
  for (uint32_t chunk = blockIdx.x; chunk < b.first[b.count]; chunk += gridDim.x) {
    const uint32_t k = tensor_of(b, chunk);
    const uint64_t n = b.t[k].n, base = (uint64_t)(chunk - b.first[k]) * NORM_CHUNK;
    const T* p = (const T*)b.t[k].p;
    Eight<T> x[NORM_CHUNK / 2048];
    if (base + NORM_CHUNK <= n) {
#pragma unroll
      for (int j = 0; j < NORM_CHUNK / 2048; ++j)
        x[j].template load<true>(p, base + j * 2048 + threadIdx.x * 8, n);
    } else {
#pragma unroll
      for (int j = 0; j < NORM_CHUNK / 2048; ++j)
        x[j].template load<false>(p, base + j * 2048 + threadIdx.x * 8, n);
    }
#pragma unroll
    for (int j = 0; j < NORM_CHUNK / 2048; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const double v = (double)to_f32(x[j].v[e]);
        sum = fma(v, v, sum);
      }
  }
  sum = group_sum64<4>(sum);
  if (threadIdx.x != 0) return;
  if (norm)
    *norm = (float)sqrt(sum);
  else
    parts[blockIdx.x] = sum;
}

__global__ void __launch_bounds__(1024) norm_join_kernel(uint32_t count,
                                                         const double* __restrict__ parts,
                                                         float* __restrict__ norm) {
  double sum = 0;
  for (uint32_t k = threadIdx.x; k < count; k += 1024) sum += parts[k];
  sum = group_sum64<16>(sum);
  if (threadIdx.x == 0) *norm = (float)sqrt(sum);
}

// Launches over the tensors of one type; returns the number of workgroups.
template <typename T>
static uint32_t norm_launches(uint32_t n_tensors, const tgs_span* tensors, int32_t dtype,
                              double* parts, float* norm, hipStream_t stream) {
  uint32_t groups = 0;
  NormBatch b = {};
  uint64_t chunks = 0;
  const auto flush = [&] {
    if (!b.count) return;
    b.first[b.count] = (uint32_t)chunks;
    const uint32_t grid = norm ? 1 : (uint32_t)std::min<uint64_t>(chunks, NORM_PARTS);
    hipLaunchKernelGGL(norm_kernel<T>, dim3(grid), dim3(256), 0, stream, b, parts + groups, norm);
    groups += grid;
    b.count = 0;
    chunks = 0;
  };
  for (uint32_t k = 0; k < n_tensors; ++k) {
    if (tensors[k].n == 0 || tensors[k].dtype != dtype) continue;
    b.first[b.count] = (uint32_t)chunks;
    b.t[b.count].p = tensors[k].data;
    b.t[b.count++].n = tensors[k].n;
    chunks += (tensors[k].n + NORM_CHUNK - 1) / NORM_CHUNK;  // (64 of at most 2^25)
    if (b.count == NORM_TENSORS) flush();
  }
  flush();
  return groups;
}

// (a launch for every 64 tensors and one more of each type)
extern "C" uint64_t tgs_grad_norm_workspace_size(uint32_t n_tensors) {
  return ((uint64_t)n_tensors / NORM_TENSORS + 3) * NORM_PARTS * sizeof(double);
}

extern "C" int tgs_grad_norm(uint32_t n_tensors, const tgs_span* tensors, float* norm,
                             void* workspace, uint64_t workspace_bytes, hipStream_t stream) {
  TGS_CHECK_ARG(norm && (tensors || !n_tensors), "tgs_grad_norm: null pointer");
  for (uint32_t k = 0; k < n_tensors; ++k) {
    TGS_CHECK_ARG(tensors[k].dtype >= TGS_F32 && tensors[k].dtype <= TGS_F16,
                  "tgs_grad_norm: dtype must be 0 (float32), 1 (bfloat16) or 2 (float16), got %d",
                  tensors[k].dtype);
    TGS_CHECK_ARG(tensors[k].data || !tensors[k].n, "tgs_grad_norm: null pointer in tensor %u", k);
    TGS_CHECK_ARG(tensors[k].n <= (1ull << 38), "tgs_grad_norm: %llu values",
                  (unsigned long long)tensors[k].n);
  }
  if (workspace_bytes < tgs_grad_norm_workspace_size(n_tensors)) {
    tgs_set_error("tgs_grad_norm: workspace too small");
    return TGS_ERR_WORKSPACE;
  }
  TGS_CHECK_ARG(workspace && (uintptr_t)workspace % 8 == 0,
                "tgs_grad_norm: the workspace starts on 8 bytes");
  double* parts = (double*)workspace;
  // A few values of one type: one workgroup, one launch.
  uint64_t total = 0;
  bool single = n_tensors > 0 && n_tensors <= NORM_TENSORS;
  for (uint32_t k = 0; k < n_tensors; ++k) {
    total += (tensors[k].n + NORM_CHUNK - 1) / NORM_CHUNK;
    single &= tensors[k].dtype == tensors[0].dtype;
  }
  single &= total > 0 && total <= NORM_SINGLE;
  uint32_t count = 0;
  for (int32_t dtype = TGS_F32; dtype <= TGS_F16; ++dtype)
    with_dtype(dtype, "tgs_grad_norm", [&](auto tag) {
      count += norm_launches<decltype(tag)>(n_tensors, tensors, dtype, parts + count,
                                            single ? norm : nullptr, stream);
      return TGS_OK;
    });
  if (single) TGS_RETURN_LAUNCH("tgs_grad_norm");
  hipLaunchKernelGGL(norm_join_kernel, dim3(1), dim3(1024), 0, stream, count, parts, norm);
  TGS_RETURN_LAUNCH("tgs_grad_norm");
}
