// Layer norm over the last dimension, forward and backward.
//
//   mean = sum x / n, rstd = 1 / sqrt(sum (x - mean)^2 / n + eps), xhat = (x - mean) rstd
//   y = xhat w + b
//   with g = dy w:  dx = rstd (g - mean(g) - xhat mean(g xhat)),
//                   dw = sum_rows dy xhat, db = sum_rows dy
//
// Memory bound.  A row is read once: 8 to 64 lanes hold it in registers (the variance
// is the second pass over them, not a difference of moments) and the backward computes
// mean and rstd again from the x it reads anyway, so nothing is kept between the two.
// The weight's gradient is a sum over rows: every lane adds up its columns over the
// rows of its wavefront, the workgroup joins its wavefronts through LDS into one
// partial row, and a second launch adds the partial rows, all in a fixed order.
//
// 4M rows of 64 bfloat16: forward 179 us (5.7 TB/s), backward 309 (5.0 TB/s) and 7 for the
// join; 300k rows of 59 float32 at a pitch of 64, read value by value: 24, 44 and 5 us (6.0
// and 4.8 TB/s); 8191 rows of 1024 halves: 9, 14 and 4 us.  Rows that a workgroup reads again for
// each sum: 4000 of 5000 bfloat16 52, 432 and 9 us (its partial row is read and written for
// every row), 4000 of 2501 float32 26, 195 and 6.
#include "decoder_common.cuh"

// How LANES lanes hold a row of up to LANES * E values.  VEC: lane l has runs of 16
// bytes, the runs of one load next to each other (every row 16-byte aligned and a
// whole number of runs); otherwise values l, l + LANES, ...
template <typename T, int LANES, int E, bool VEC>
struct RowMap {
  static constexpr int R = VEC ? Vec16<T>::N : 1;  // values of a run
  static_assert(E % R == 0, "whole runs");
  __device__ static __forceinline__ int column(int lane, int e) {
    return (e / R * LANES + lane) * R + e % R;
  }
  // A row as it lies in memory: the loads of several rows are on their way before the first
  // is converted.  Lanes past the end load the row's first values and keep zeros.
  struct Raw {
    Vec16<T> run[VEC ? E / R : 1];
    T one[VEC ? 1 : E];
  };
  __device__ static __forceinline__ void load(const T* row, int lane, uint32_t n, Raw& v) {
#pragma unroll
    for (int e = 0; e < E; e += R) {
      const uint32_t c = column(lane, e);
      if constexpr (VEC)
        v.run[e / R] = *(const Vec16<T>*)(row + (c < n ? c : 0));
      else
        v.one[e] = row[c < n ? c : 0];
    }
  }
  __device__ static __forceinline__ void convert(const Raw& raw, int lane, uint32_t n,
                                                 float (&v)[E]) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const bool in = (uint32_t)column(lane, e / R * R) < n;
      if constexpr (VEC)
        v[e] = in ? to_f32(raw.run[e / R].v[e % R]) : 0.f;
      else
        v[e] = in ? to_f32(raw.one[e]) : 0.f;
    }
  }
  __device__ static __forceinline__ void store(T* row, int lane, uint32_t n, const float (&v)[E]) {
#pragma unroll
    for (int e = 0; e < E; e += R) {
      const uint32_t c = column(lane, e);
      if (c >= n) continue;
      if constexpr (VEC) {
        Vec16<T> t;
#pragma unroll
        for (int k = 0; k < R; ++k) t.v[k] = from_f32<T>(v[e + k]);
        *(Vec16<T>*)(row + c) = t;
      } else {
        row[c] = from_f32<T>(v[e]);
      }
    }
  }
};

// Sum over the LANES lanes of a row, the same in each of them: DPP within 16 lanes (every
// step adds a group of lanes that all hold one sum to another), shuffles beyond.
template <int LANES>
__device__ __forceinline__ float group_sum(float v) {
  v += tgs_dpp<0xB1>(v);   // quad_perm [1,0,3,2]
  v += tgs_dpp<0x4E>(v);   // quad_perm [2,3,0,1]
  v += tgs_dpp<0x141>(v);  // row_half_mirror
  if constexpr (LANES >= 16) v += tgs_dpp<0x140>(v);  // row_mirror
  if constexpr (LANES >= 32) v += __shfl_xor(v, 16, 64);
  if constexpr (LANES >= 64) v += __shfl_xor(v, 32, 64);
  return v;
}

// Below this variance (which eps has to be below, too) squares of 32 bits start to fall out of
// the range and the hardware's reciprocal root takes its argument for zero: the differences are
// squared again TINY_SCALE times as large, the variance comes out TINY_SCALE^2 as large.
#define TINY_VARIANCE 0x1p-100f
#define TINY_SCALE 0x1p100f

__device__ __forceinline__ float tiny_variance(float squares_over_n, float eps) {
  return squares_over_n + eps * TINY_SCALE * TINY_SCALE;
}

// x becomes xhat; returns rstd.  Lanes past the row's end hold zeros, and keep them: the
// mean that is taken from them is zero.
template <typename Map, int LANES, int E>
__device__ __forceinline__ float normalise(float (&x)[E], int lane, uint32_t n, float inv_n,
                                           float eps) {
  float s = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) s += x[e];
  const float mean = group_sum<LANES>(s) * inv_n;
  float q = 0.f;
#pragma unroll
  for (int e = 0; e < E; e += Map::R) {
    const float m = (uint32_t)Map::column(lane, e) < n ? mean : 0.f;
#pragma unroll
    for (int k = 0; k < Map::R; ++k) {
      x[e + k] -= m;
      q = fmaf(x[e + k], x[e + k], q);
    }
  }
  float var = fmaf(group_sum<LANES>(q), inv_n, eps), scale = 1.f;
  if (var < TINY_VARIANCE) {  // (the same for all lanes of a row)
    scale = TINY_SCALE;
    q = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      x[e] *= scale;
      q = fmaf(x[e], x[e], q);
    }
    var = tiny_variance(group_sum<LANES>(q) * inv_n, eps);
  }
  const float rstd = __builtin_amdgcn_rsqf(var);
#pragma unroll
  for (int e = 0; e < E; ++e) x[e] *= rstd;
  return rstd * scale;
}

// The weight's or bias's values of this lane's columns; `other` where there are none.
template <typename Map, bool VEC, typename W, int E>
__device__ __forceinline__ void load_columns(const W* w, int lane, uint32_t n, float other,
                                             float (&v)[E]) {
  constexpr int R = VEC ? Vec16<W>::N : 1;
#pragma unroll
  for (int e = 0; e < E; e += R) {
    const uint32_t c = Map::column(lane, e);
    if (w && c < n) {
      if constexpr (VEC) {
        const Vec16<W> t = *(const Vec16<W>*)(w + c);
#pragma unroll
        for (int k = 0; k < R; ++k) v[e + k] = to_f32(t.v[k]);
      } else {
        v[e] = to_f32(w[c]);
      }
    } else {
#pragma unroll
      for (int k = 0; k < R; ++k) v[e + k] = other;
    }
  }
}

// Rows that a lane has in flight at once.
template <int E>
constexpr int rows_at_once() {
  return E <= 4 ? 4 : E <= 16 ? 2 : 1;
}

template <typename T, typename W, int LANES, int E, bool VEC>
__global__ void __launch_bounds__(256) layer_norm_fwd_kernel(
    uint64_t rows, uint32_t n, const T* __restrict__ x, int64_t pitch, const W* __restrict__ weight,
    const W* __restrict__ bias, float eps, T* __restrict__ y) {
  using Map = RowMap<T, LANES, E, VEC>;
  constexpr int PER = 256 / LANES, U = rows_at_once<E>();  // rows of a workgroup at once
  const int lane = threadIdx.x % LANES;
  const float inv_n = 1.f / (float)n;
  float w[E], b[E];
  load_columns<Map, VEC>(weight, lane, n, 1.f, w);
  load_columns<Map, VEC>(bias, lane, n, 0.f, b);
  // (a row's sums stay inside its own lanes, so lanes without a row need no barrier)
  for (uint64_t r0 = (uint64_t)blockIdx.x * PER * U + threadIdx.x / LANES; r0 < rows;
       r0 += (uint64_t)gridDim.x * PER * U) {
    typename Map::Raw raw[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const uint64_t r = min(r0 + k * PER, rows - 1);  // (the last row again: not stored)
      Map::load(x + (int64_t)r * pitch, lane, n, raw[k]);
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      float v[E];
      Map::convert(raw[k], lane, n, v);
      normalise<Map, LANES, E>(v, lane, n, inv_n, eps);
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = fmaf(v[e], w[e], b[e]);
      const uint64_t r = r0 + k * PER;
      if (r < rows) Map::store(y + r * n, lane, n, v);
    }
  }
}

template <typename T, typename W, int LANES, int E, bool VEC>
__global__ void __launch_bounds__(256) layer_norm_bwd_kernel(
    uint64_t rows, uint32_t n, const T* __restrict__ x, int64_t pitch, const T* __restrict__ dy,
    int64_t dy_pitch, const W* __restrict__ weight, float eps, T* __restrict__ dx,
    float* __restrict__ partial, W* __restrict__ dweight, W* __restrict__ dbias) {
  using Map = RowMap<T, LANES, E, VEC>;
  constexpr int PER = 256 / LANES, U = rows_at_once<E>();
  __shared__ float s_part[2][LANES * E];
  const int lane = threadIdx.x % LANES;
  const float inv_n = 1.f / (float)n;
  float w[E], dw[E] = {}, db[E] = {};
  load_columns<Map, VEC>(weight, lane, n, 1.f, w);
  for (uint64_t r0 = (uint64_t)blockIdx.x * PER * U + threadIdx.x / LANES; r0 < rows;
       r0 += (uint64_t)gridDim.x * PER * U) {
    typename Map::Raw raw_x[U], raw_dy[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const uint64_t r = min(r0 + k * PER, rows - 1);
      Map::load(x + (int64_t)r * pitch, lane, n, raw_x[k]);
      Map::load(dy + (int64_t)r * dy_pitch, lane, n, raw_dy[k]);
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const uint64_t r = r0 + k * PER;
      if (r >= rows) break;
      float v[E], g[E];
      Map::convert(raw_x[k], lane, n, v);
      Map::convert(raw_dy[k], lane, n, g);
      const float rstd = normalise<Map, LANES, E>(v, lane, n, inv_n, eps);
      float s = 0.f, q = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        dw[e] = fmaf(g[e], v[e], dw[e]);
        db[e] += g[e];
        g[e] *= w[e];
        s += g[e];
        q = fmaf(g[e], v[e], q);
      }
      if (dx) {
        s = group_sum<LANES>(s) * inv_n;
        q = group_sum<LANES>(q) * inv_n;
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = rstd * (g[e] - s - v[e] * q);
        Map::store(dx + r * n, lane, n, v);
      }
    }
  }
  if (!partial) return;
#pragma unroll
  for (int e = 0; e < E; ++e)
#pragma unroll
    for (int off = LANES; off < 64; off <<= 1) {
      dw[e] += __shfl_xor(dw[e], off, 64);
      db[e] += __shfl_xor(db[e], off, 64);
    }
  for (uint32_t wave = 0; wave < 4; ++wave) {
    if (threadIdx.x / 64 == wave && threadIdx.x % 64 < LANES) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int c = Map::column(lane, e);
        s_part[0][c] = wave ? s_part[0][c] + dw[e] : dw[e];
        s_part[1][c] = wave ? s_part[1][c] + db[e] : db[e];
      }
    }
    __syncthreads();
  }
  for (uint32_t i = threadIdx.x; i < 2 * n; i += 256) {
    const float v = i < n ? s_part[0][i] : s_part[1][i - n];
    W* out = i < n ? dweight : dbias;
    if (gridDim.x > 1)
      partial[(uint64_t)blockIdx.x * 2 * n + i] = v;
    else if (out)  // nothing to join
      out[i < n ? i : i - n] = from_f32<W>(v);
  }
}

// A row of any width, one workgroup per row, read again for each of its sums (rows
// that 64 lanes do not hold in registers).
__device__ __forceinline__ float block_sum(float v, float* s) {
  v = tgs_wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
  __syncthreads();
  return (s[0] + s[1]) + (s[2] + s[3]);
}

// xhat is (x - mean) scale root, dx has the factor scale root as well.
struct RowStats {
  float mean, scale, root;
  __device__ __forceinline__ float xhat(float x) const { return (x - mean) * scale * root; }
};

template <typename T>
__device__ __forceinline__ RowStats row_stats(const T* x, uint32_t n, float eps, float* s) {
  float a = 0.f;
  for (uint32_t c = threadIdx.x; c < n; c += 256) a += to_f32(x[c]);
  const float mean = block_sum(a, s) / (float)n;
  const auto squares = [&](float scale) {
    float q = 0.f;
    for (uint32_t c = threadIdx.x; c < n; c += 256) {
      const float d = (to_f32(x[c]) - mean) * scale;
      q = fmaf(d, d, q);
    }
    return block_sum(q, s) / (float)n;
  };
  const float var = squares(1.f) + eps;
  if (var < TINY_VARIANCE)  // (the same for all threads)
    return {mean, TINY_SCALE, 1.f / sqrtf(tiny_variance(squares(TINY_SCALE), eps))};
  return {mean, 1.f, 1.f / sqrtf(var)};
}

template <typename T, typename W>
__global__ void __launch_bounds__(256) layer_norm_fwd_wide_kernel(
    uint64_t rows, uint32_t n, const T* __restrict__ x, int64_t pitch, const W* __restrict__ weight,
    const W* __restrict__ bias, float eps, T* __restrict__ y) {
  __shared__ float s[4];
  for (uint64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* row = x + (int64_t)r * pitch;
    const RowStats stats = row_stats(row, n, eps, s);
    for (uint32_t c = threadIdx.x; c < n; c += 256)
      y[r * n + c] = from_f32<T>(fmaf(stats.xhat(to_f32(row[c])),
                                      weight ? to_f32(weight[c]) : 1.f,
                                      bias ? to_f32(bias[c]) : 0.f));
  }
}

// The workgroup's partial row is its own in memory: thread t adds to columns t, t + 256, ...
template <typename T, typename W>
__global__ void __launch_bounds__(256) layer_norm_bwd_wide_kernel(
    uint64_t rows, uint32_t n, const T* __restrict__ x, int64_t pitch, const T* __restrict__ dy,
    int64_t dy_pitch, const W* __restrict__ weight, float eps, T* __restrict__ dx,
    float* __restrict__ partial, W*, W*) {
  __shared__ float s[4];
  float* dw = partial ? partial + (uint64_t)blockIdx.x * 2 * n : nullptr;
  if (dw)
    for (uint32_t c = threadIdx.x; c < n; c += 256) dw[c] = dw[n + c] = 0.f;
  for (uint64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* row = x + (int64_t)r * pitch;
    const T* grad = dy + (int64_t)r * dy_pitch;
    const RowStats stats = row_stats(row, n, eps, s);
    float a = 0.f, q = 0.f;
    for (uint32_t c = threadIdx.x; c < n; c += 256) {
      const float d = to_f32(grad[c]), xh = stats.xhat(to_f32(row[c]));
      if (dw) {
        dw[c] = fmaf(d, xh, dw[c]);
        dw[n + c] += d;
      }
      const float g = d * (weight ? to_f32(weight[c]) : 1.f);
      a += g;
      q = fmaf(g, xh, q);
    }
    a = block_sum(a, s) / (float)n;
    q = block_sum(q, s) / (float)n;
    if (!dx) continue;
    for (uint32_t c = threadIdx.x; c < n; c += 256) {
      const float g = to_f32(grad[c]) * (weight ? to_f32(weight[c]) : 1.f);
      dx[r * n + c] =
          from_f32<T>(stats.root * stats.scale * (g - a - stats.xhat(to_f32(row[c])) * q));
    }
  }
}

// dw and db: the partial rows' sums, 8 columns by 128 interleaved runs of rows a workgroup
// (32 by 32 left the few columns of narrow rows to four workgroups: 20 us for 2048 partial
// rows of 59, now 5).
template <typename W>
__global__ void __launch_bounds__(1024) layer_norm_join_kernel(uint32_t parts, uint32_t n,
                                                               const float* __restrict__ partial,
                                                               W* __restrict__ dweight,
                                                               W* __restrict__ dbias) {
  __shared__ float s[1024];
  const uint32_t c = blockIdx.x * 8 + threadIdx.x % 8, k = threadIdx.x / 8;
  float a = 0.f;
  if (c < 2 * n) {
#pragma unroll 8
    for (uint32_t p = k; p < parts; p += 128) a += partial[(uint64_t)p * 2 * n + c];
  }
  s[threadIdx.x] = a;
  for (uint32_t h = 64; h > 0; h >>= 1) {
    __syncthreads();
    if (k < h) s[threadIdx.x] += s[threadIdx.x + 8 * h];
  }
  if (k == 0 && c < 2 * n) {
    W* out = c < n ? dweight : dbias;
    if (out) out[c < n ? c : c - n] = from_f32<W>(s[threadIdx.x]);
  }
}

// Values of a row that 64 lanes hold in registers; half as many one by one, whose backward
// would spill.
static uint32_t most_held(bool vec) { return vec ? 4096 : 2048; }

// Workgroups of a backward launch: each leaves a partial row of both sums, so none for fewer
// than 16 rows once the CUs have one each (8191 rows of 1024: 2048 workgroups' partial rows
// were as many bytes as x).
static uint32_t norm_groups(uint64_t rows) {
  return (uint32_t)std::min<uint64_t>(std::max<uint64_t>(rows / 16, std::min<uint64_t>(rows, 256)),
                                      2048);
}

// Calls f(LANES, E) as constants: the fewest lanes that hold n values.
template <typename T, bool VEC, typename F>
static void with_row_map(uint32_t n, F&& f) {
  constexpr int R = VEC ? Vec16<T>::N : 1;
#define LN_MAP(LANES, E) \
  if (n <= (LANES) * (E)) return f(std::integral_constant<int, LANES>(), std::integral_constant<int, E>())
  if constexpr (R > 1) {
    LN_MAP(8, R);
    LN_MAP(16, R);
    LN_MAP(32, R);
  }
  if constexpr (R < 2) {
    LN_MAP(16, 1);
    LN_MAP(16, 2);
    LN_MAP(16, 4);
    LN_MAP(64, 2);
  }
  if constexpr (R < 8) LN_MAP(64, 4);
  LN_MAP(64, 8);
  LN_MAP(64, 16);
  LN_MAP(64, 32);
  if constexpr (R > 1) LN_MAP(64, 64);
#undef LN_MAP
}

extern "C" int tgs_layer_norm_fwd(uint64_t rows, uint32_t width, int32_t dtype, const void* x,
                                  int64_t x_pitch, const void* weight, const void* bias,
                                  int32_t weight_dtype, float eps, void* y, hipStream_t stream) {
  return with_dtype(dtype, "tgs_layer_norm_fwd", [&](auto tag) -> int {
    using T = decltype(tag);
    TGS_CHECK_ARG(width > 0 && width <= (1u << 30), "tgs_layer_norm_fwd: width %u", width);
    TGS_CHECK_ARG(weight_dtype == dtype || weight_dtype == TGS_F32,
                  "tgs_layer_norm_fwd: the weights have x's type or float32");
    if (rows == 0) return TGS_OK;
    TGS_CHECK_ARG(x && y, "tgs_layer_norm_fwd: null pointer");
    TGS_CHECK_ARG(x_pitch >= (int64_t)width || rows == 1, "tgs_layer_norm_fwd: pitch below width");
    const auto typed = [&](auto wtag) {
      using W = decltype(wtag);
      const auto launch = [&](auto kernel, uint64_t groups) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)groups), dim3(256), 0, stream, rows, width,
                           (const T*)x, x_pitch, (const W*)weight, (const W*)bias, eps, (T*)y);
      };
      const auto held = [&](auto vec) {
        with_row_map<T, vec.value>(width, [&](auto lanes, auto e) {
          const uint64_t per = 256 / lanes.value * rows_at_once<e.value>();
          launch(layer_norm_fwd_kernel<T, W, lanes.value, e.value, vec.value>,
                 std::min<uint64_t>((rows + per - 1) / per, 4096));
        });
      };
      const bool vec = width % Vec16<T>::N == 0 && aligned16((const T*)x, x_pitch) &&
                       aligned16((const T*)y, width) && aligned16((const W*)weight, 0) &&
                       aligned16((const W*)bias, 0);
      if (width > most_held(vec))
        launch(layer_norm_fwd_wide_kernel<T, W>, std::min<uint64_t>(rows, 4096));
      else if (vec)
        held(std::true_type());
      else
        held(std::false_type());
    };
    if (weight_dtype == dtype)
      typed(T{});
    else
      typed(float{});
    TGS_RETURN_LAUNCH("tgs_layer_norm_fwd");
  });
}

extern "C" uint64_t tgs_layer_norm_bwd_workspace_size(uint64_t rows, uint32_t width) {
  return (uint64_t)norm_groups(rows) * 2 * width * sizeof(float);
}

extern "C" int tgs_layer_norm_bwd(uint64_t rows, uint32_t width, int32_t dtype, const void* x,
                                  int64_t x_pitch, const void* dy, int64_t dy_pitch,
                                  const void* weight, int32_t weight_dtype, float eps, void* dx,
                                  void* dweight, void* dbias, void* workspace,
                                  uint64_t workspace_bytes, hipStream_t stream) {
  return with_dtype(dtype, "tgs_layer_norm_bwd", [&](auto tag) -> int {
    using T = decltype(tag);
    TGS_CHECK_ARG(width > 0 && width <= (1u << 30), "tgs_layer_norm_bwd: width %u", width);
    TGS_CHECK_ARG(weight_dtype == dtype || weight_dtype == TGS_F32,
                  "tgs_layer_norm_bwd: the weights have x's type or float32");
    const bool sums = dweight || dbias;
    TGS_CHECK_ARG(rows == 0 || (x && dy), "tgs_layer_norm_bwd: null pointer");
    TGS_CHECK_ARG((x_pitch >= (int64_t)width && dy_pitch >= (int64_t)width) || rows <= 1,
                  "tgs_layer_norm_bwd: pitch below width");
    const uint32_t groups = rows ? norm_groups(rows) : 0;
    if (sums && workspace_bytes < tgs_layer_norm_bwd_workspace_size(rows, width)) {
      tgs_set_error("tgs_layer_norm_bwd: workspace too small");
      return TGS_ERR_WORKSPACE;
    }
    TGS_CHECK_ARG(!sums || rows == 0 || workspace, "tgs_layer_norm_bwd: null workspace");
    if (!sums && (!dx || rows == 0)) return TGS_OK;
    float* partial = sums ? (float*)workspace : nullptr;
    const auto typed = [&](auto wtag) {
      using W = decltype(wtag);
      const auto launch = [&](auto kernel, uint32_t g) {
        hipLaunchKernelGGL(kernel, dim3(g), dim3(256), 0, stream, rows, width, (const T*)x,
                           x_pitch, (const T*)dy, dy_pitch, (const W*)weight, eps, (T*)dx, partial,
                           (W*)dweight, (W*)dbias);
      };
      const bool vec = width % Vec16<T>::N == 0 && aligned16((const T*)x, x_pitch) &&
                       aligned16((const T*)dy, dy_pitch) && (!dx || aligned16((const T*)dx, width)) &&
                       aligned16((const W*)weight, 0);
      uint32_t parts = groups;
      const auto held = [&](auto vec) {
        with_row_map<T, vec.value>(width, [&](auto lanes, auto e) {
          const uint64_t per = 256 / lanes.value * rows_at_once<e.value>();
          parts = (uint32_t)std::min<uint64_t>((rows + per - 1) / per, groups);
          launch(layer_norm_bwd_kernel<T, W, lanes.value, e.value, vec.value>, parts);
        });
      };
      if (rows) {
        if (width > most_held(vec))
          launch(layer_norm_bwd_wide_kernel<T, W>, groups);
        else if (vec)
          held(std::true_type());
        else
          held(std::false_type());
      }
      if (sums && (parts != 1 || width > most_held(vec)))
        hipLaunchKernelGGL(layer_norm_join_kernel<W>, dim3((2 * width + 7) / 8), dim3(1024), 0,
                           stream, parts, width, partial, (W*)dweight, (W*)dbias);
    };
    if (weight_dtype == dtype)
      typed(T{});
    else
      typed(float{});
    TGS_RETURN_LAUNCH("tgs_layer_norm_bwd");
  });
}
