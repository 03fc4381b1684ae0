// The gated feed-forward block for up to 32 rows: every weight is read once, straight into the
// registers of the wavefront that multiplies it, and the sums over k are split over the
// wavefronts of a workgroup and joined in LDS.
//
// A workgroup takes 16 hidden columns (then 16 outputs) and all rows, which are the second
// operand of its products, 16 a tile: the same four matrix instructions a weight whether one
// row or sixteen are there, and the loads are what counts.  Two launches, the hidden
// values of a call (32 rows of 4096: 256 KB) between them in L2.  One row of 1024-4096-1024
// bfloat16 takes 6.0 + 6.9 us: 2.8 and 1.2 TB/s of weights, of float32 11.3 + 9.8 (3.0 and
// 1.7), 20 of bfloat16 8.9 + 16.  The matrix cores idle meanwhile,
// so a hidden value of 16 bits is multiplied with what its rounding left as a second plane:
// y is off by its own rounding alone.
#include "gated_ffn.cuh"

// Sixteen bytes at a byte offset of a buffer; zeros past its end.
__device__ __forceinline__ i32x4 load16(rsrc_t r, uint32_t off) {
  return __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0);
}

// Eight values of a buffer of T from value `at` on, as planes (`live`: else zeros).
template <typename T>
__device__ __forceinline__ void load_planes(rsrc_t r, uint32_t at, bool live,
                                            frag_t<typename Planes<T>::E> (&out)[Planes<T>::N]) {
  const uint32_t off = live ? at * (uint32_t)sizeof(T) : MX_OUTSIDE;
  union {
    i32x4 w[sizeof(T) / 2];
    T v[8];
  } u;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) u.w[i] = load16(r, off + i * 16);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    typename Planes<T>::E p[Planes<T>::N];
    split<T>(to_f32(u.v[e]), p);
#pragma unroll
    for (int s = 0; s < Planes<T>::N; ++s) out[s][e] = p[s];
  }
}

// Planes of a hidden value.
template <typename T>
constexpr int HIDDEN_PLANES = Planes<T>::N == 1 ? 2 : 3;

template <typename T>
struct FewArgs {
  using E = typename Planes<T>::E;
  const T *x, *wg, *wu, *wd, *bg, *bu, *bd;
  E* h;  // [HIDDEN_PLANES, rows, hidden8]
  T* y;
  int64_t x_pitch;
  int32_t rows, width, hidden, hidden8, out;
  int32_t each;  // outputs of a workgroup: 16, or 8 where 16 would leave half the CUs idle
  int32_t wide_x, wide_w, wide_d;  // rows of x, of Wg and Wu, of Wd are read 16 bytes at a time
};

#define FEW_HIDDEN_WAVES 8
#define FEW_OUT_WAVES 16

template <typename T, int RT, int ACT>
__global__ void __launch_bounds__(64 * FEW_HIDDEN_WAVES) ffn_few_hidden_kernel(FewArgs<T> a) {
  using E = typename Planes<T>::E;
  constexpr int P = Planes<T>::N, W = FEW_HIDDEN_WAVES;
  __shared__ f32x4 s[W][RT][2][64];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int f0 = blockIdx.x * 16, row = lane & 15, col = (lane >> 4) * 8;
  const int live = min(16, a.hidden - f0);  // weight rows
  const int64_t from = (int64_t)f0 * a.width;
  const rsrc_t rg = buffer_of(a.wg + from, (uint32_t)(live * a.width * sizeof(T)));
  const rsrc_t ru = buffer_of(a.wu + from, (uint32_t)(live * a.width * sizeof(T)));
  f32x4 g[RT] = {}, u[RT] = {};
  const int steps = (a.width + 31) / 32;
#pragma unroll 4
  for (int k = wave; k < steps; k += W) {
    const int c = k * 32 + col;
    frag_t<E> wg[P], wu[P];
    if (a.wide_w) {
      const bool in = row < live && c < a.width;
      load_planes<T>(rg, row * a.width + c, in, wg);
      load_planes<T>(ru, row * a.width + c, in, wu);
    } else {
      load_fragment<T>(a.wg + from + (int64_t)row * a.width, c, a.width, row < live, false, wg);
      load_fragment<T>(a.wu + from + (int64_t)row * a.width, c, a.width, row < live, false, wu);
    }
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      frag_t<E> x[P];
      const int m = i * 16 + row;
      load_fragment<T>(a.x + m * a.x_pitch, c, a.width, m < a.rows, a.wide_x, x);
      g[i] = mfma_planes<T>(wg, x, g[i]);
      u[i] = mfma_planes<T>(wu, x, u[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < RT; ++i) s[wave][i][0][lane] = g[i], s[wave][i][1][lane] = u[i];
  __syncthreads();
  if (wave >= RT) return;
  const int m = wave * 16 + row, f = f0 + (lane >> 4) * 4;
  f32x4 gs = s[0][wave][0][lane], us = s[0][wave][1][lane];
#pragma unroll
  for (int w = 1; w < W; ++w) gs += s[w][wave][0][lane], us += s[w][wave][1][lane];
  if (m >= a.rows || f >= a.hidden8) return;
  float v[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const bool in = f + r < a.hidden;
    const float gv = gs[r] + (a.bg && in ? to_f32(a.bg[f + r]) : 0.f);
    const float uv = us[r] + (a.bu && in ? to_f32(a.bu[f + r]) : 0.f);
    v[r] = in ? activation<ACT, T>(gv).x * uv : 0.f;
  }
  constexpr int HP = HIDDEN_PLANES<T>;
  four_t<E> h[HP];
  if constexpr (P == 1) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      h[0][r] = (E)v[r];
      const float rest = v[r] - (float)h[0][r];  // not finite: nothing
      h[1][r] = (E)(__builtin_fabsf(rest) < __builtin_inff() ? rest : 0.f);
    }
  } else {
    split4<T>(v, h);
  }
#pragma unroll
  for (int q = 0; q < HP; ++q)
    *(four_t<E>*)(a.h + ((int64_t)q * a.rows + m) * a.hidden8 + f) = h[q];
}

template <typename T, int RT>
__global__ void __launch_bounds__(64 * FEW_OUT_WAVES) ffn_few_out_kernel(FewArgs<T> a) {
  using E = typename Planes<T>::E;
  constexpr int P = Planes<T>::N, HP = HIDDEN_PLANES<T>, W = FEW_OUT_WAVES;
  __shared__ f32x4 s[W][RT][64];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int o0 = blockIdx.x * a.each, row = lane & 15, col = (lane >> 4) * 8;
  const int live = min(a.each, a.out - o0);
  const int64_t from = (int64_t)o0 * a.hidden;
  const rsrc_t rd = buffer_of(a.wd + from, (uint32_t)(live * a.hidden * sizeof(T)));
  const rsrc_t rh = buffer_of(a.h, (uint32_t)(HP * a.rows * a.hidden8 * 2));
  f32x4 y[RT] = {};
  const int steps = (a.hidden + 31) / 32;
#pragma unroll 4
  for (int k = wave; k < steps; k += W) {
    const int c = k * 32 + col;
    frag_t<E> w[P];
    if (a.wide_d)
      load_planes<T>(rd, row * a.hidden + c, row < live && c < a.hidden, w);
    else
      load_fragment<T>(a.wd + from + (int64_t)row * a.hidden, c, a.hidden, row < live, false, w);
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const int m = i * 16 + row;
      frag_t<E> h[HP];
#pragma unroll
      for (int q = 0; q < HP; ++q) {
        union {
          i32x4 w;
          frag_t<E> f;
        } v;
        v.w = load16(rh, m < a.rows && c < a.hidden8
                             ? (uint32_t)((q * a.rows + m) * a.hidden8 + c) * 2 : MX_OUTSIDE);
        h[q] = v.f;
      }
      if constexpr (P == 1)
        y[i] = mfma32(w[0], h[0], mfma32(w[0], h[1], y[i]));
      else
        y[i] = mfma_planes<T>(w, h, y[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < RT; ++i) s[wave][i][lane] = y[i];
  __syncthreads();
  if (wave >= RT) return;
  const int m = wave * 16 + row, o = o0 + (lane >> 4) * 4;
  f32x4 v = s[0][wave][lane];
#pragma unroll
  for (int w = 1; w < W; ++w) v += s[w][wave][lane];
  if (m >= a.rows) return;
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (o + r < o0 + live)
      a.y[(int64_t)m * a.out + o + r] = from_f32<T>(v[r] + (a.bd ? to_f32(a.bd[o + r]) : 0.f));
}

template <typename T>
uint64_t FewKernels<T>::workspace(int64_t rows, int32_t hidden) {
  return HIDDEN_PLANES<T> * rows * round8(hidden) * 2;
}

template <typename T>
void FewKernels<T>::forward(const FfnCall& c, void* workspace, hipStream_t stream) {
  using E = typename Planes<T>::E;
  const auto wide = [](const void* p, int64_t cols, int64_t pitch) {
    return cols % 8 == 0 && aligned16((const T*)p, pitch);
  };
  const FewArgs<T> a{(const T*)c.x, (const T*)c.wg, (const T*)c.wu, (const T*)c.wd,
                     (const T*)c.bg, (const T*)c.bu, (const T*)c.bd, (E*)workspace, (T*)c.y,
                     c.x_pitch, (int32_t)c.rows, c.width, c.hidden, (int32_t)round8(c.hidden), c.out,
                     c.out < 16 * 128 ? 8 : 16,
                     wide(c.x, c.width, c.x_pitch),
                     wide(c.wg, c.width, c.width) && wide(c.wu, c.width, c.width),
                     wide(c.wd, c.hidden, c.hidden)};
  const auto launch = [&](auto rt) {
    with_activation(c.act, [&](auto act) {
      hipLaunchKernelGGL((ffn_few_hidden_kernel<T, rt.value, act.value>),
                         dim3((unsigned)tiles(c.hidden, 16)), dim3(64 * FEW_HIDDEN_WAVES), 0, stream, a);
    });
    hipLaunchKernelGGL((ffn_few_out_kernel<T, rt.value>), dim3((unsigned)tiles(c.out, a.each)),
                       dim3(64 * FEW_OUT_WAVES), 0, stream, a);
  };
  if (c.rows <= 16)
    launch(std::integral_constant<int, 1>());
  else
    launch(std::integral_constant<int, 2>());
}

template struct FewKernels<float>;
template struct FewKernels<bf16_t>;
template struct FewKernels<f16_t>;
