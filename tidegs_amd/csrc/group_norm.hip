// Group norm with an activation over channels-last tensors, forward and backward.
//
// x [samples, pixels, width]; a sample's group is `each` = width / groups neighbouring channels
// of all its pixels, m = pixels * each values:
//
//   mean = sum x / m, rstd = 1 / sqrt(sum (x - mean)^2 / m + eps), xhat = (x - mean) rstd
//   z = xhat w + b, y = act(z)
//   with dz = dy act'(z), g = dz w:  dx = rstd (g - sum(g) / m - xhat sum(g xhat) / m),
//                                    dw = sum dz xhat, db = sum dz  over samples and pixels
//
// Memory bound.  Two ways, by the size of a group:
//
// Held (up to 64 lanes by 8 runs of values): a team of lanes keeps a group in registers, so x
// is read once and a launch does all.  The backward computes mean and rstd again.
//
// Streamed: workgroups take runs of pixels by up to 64 vectors of channels and leave each channel's
// mean and sum of squared differences (of dz and dz xhat in the backward), a second launch
// joins them by group, a third reads x again and writes.  The forward keeps mean and rstd for
// the backward.
//
// Sums of squares are of differences from a value near by (a thread's first one, a mean), and
// partial ones are joined by their means, so no large mean cancels.  All joins are in a fixed
// order.
#include "activation.cuh"
#include "vector_io.cuh"

#define ACT_NONE 3
#define HELD_RUNS 8     // runs of a lane at most
#define TILE_VECTORS 64  // vectors of channels of a streaming workgroup

struct GnCall {
  uint64_t samples, pixels;
  uint32_t width, groups, each;
  int32_t act, wide_weights;  // wide_weights: float32 whatever x is
  const void* x;
  const void* dy;
  int64_t x_sample, x_pitch, dy_sample, dy_pitch;  // distances of samples and pixels, in values
  const void* weight;
  const void* bias;
  float eps;
  void* y;   // (dx in the backward)
  float2* stats;  // mean and rstd of each sample's group
};

template <typename F>
__device__ __forceinline__ void with_act(int act, F&& f) {
  if (act == ACT_SILU)
    f(std::integral_constant<int, ACT_SILU>());
  else if (act == ACT_GELU)
    f(std::integral_constant<int, ACT_GELU>());
  else if (act == ACT_RELU)
    f(std::integral_constant<int, ACT_RELU>());
  else
    f(std::integral_constant<int, ACT_NONE>());
}

template <int ACT, typename T>
__device__ __forceinline__ float act_value(float z) {
  if constexpr (ACT == ACT_NONE)
    return z;
  else
    return activation<ACT, T>(z).x;
}
template <int ACT, typename T>
__device__ __forceinline__ float act_slope(float z) {
  if constexpr (ACT == ACT_NONE)
    return 1.f;
  else
    return activation<ACT, T>(z).y;
}

// Channel c's weight or bias.
template <typename T>
__device__ __forceinline__ float column(const void* w, int wide, uint32_t c, float other) {
  return !w ? other : wide ? ((const float*)w)[c] : to_f32(((const T*)w)[c]);
}

// Sum over the 2^log lanes of a team.
__device__ __forceinline__ float team_sum(float v, int log) {
  for (int k = 0; k < log; ++k) v += __shfl_xor(v, 1 << k, 64);
  return v;
}

// ---------------------------------------------------------------------------
// Held groups.  A team has 2^row_log rows of 2^lane_log lanes (as many as hold a pixel's
// vectors of the group); teams of a workgroup take neighbouring groups.  A team keeps to one
// group's channels over all its samples, so weights are read once and the weights' gradients
// stay in registers.
// ---------------------------------------------------------------------------

struct HeldPlan {
  int lane_log, row_log;
  uint32_t teams;    // of a workgroup that work
  uint32_t rows;     // samples that all teams take at once
  uint32_t grid;
  uint32_t partials;  // rows of the weights' gradients
  int runs;          // of a lane
};

template <typename T, int V, int E, bool BACKWARD>
__global__ void __launch_bounds__(256) group_norm_held_kernel(GnCall k, HeldPlan plan,
                                                              float* __restrict__ partial) {
  const int lane_log = plan.lane_log, team_log = lane_log + plan.row_log;
  const uint32_t lane = threadIdx.x & ((1u << lane_log) - 1);
  const uint32_t row = (threadIdx.x >> lane_log) & ((1u << plan.row_log) - 1);
  const uint32_t team = threadIdx.x >> team_log;
  const uint64_t id = (uint64_t)blockIdx.x * plan.teams + team;
  const bool works = team < plan.teams && id < (uint64_t)plan.rows * k.groups;
  const uint32_t group = (uint32_t)(id % k.groups);
  const bool live = works && lane * V < k.each;
  const uint32_t c0 = group * k.each + lane * V;
  const float inv = 1.f / (float)(k.pixels * k.each);
  float w[V], b[V], dw[V] = {}, db[V] = {};
#pragma unroll
  for (int v = 0; v < V; ++v) {
    w[v] = live ? column<T>(k.weight, k.wide_weights, c0 + v, 1.f) : 0.f;
    b[v] = live ? column<T>(k.bias, k.wide_weights, c0 + v, 0.f) : 0.f;
  }
  for (uint64_t n = id / k.groups; works && n < k.samples; n += plan.rows) {
    const T* x = (const T*)k.x + (int64_t)n * k.x_sample + c0;
    Run<T, V> in[E], grad[BACKWARD ? E : 1];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const uint32_t p = row + ((uint32_t)e << plan.row_log);
      const bool ok = live && p < k.pixels;
      if (ok) in[e].load(x + (int64_t)p * k.x_pitch);
      if constexpr (BACKWARD)
        if (ok)
          grad[e].load((const T*)k.dy + (int64_t)n * k.dy_sample + (int64_t)p * k.dy_pitch + c0);
    }
    float xh[E][V], sum = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const bool ok = live && row + ((uint32_t)e << plan.row_log) < k.pixels;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        xh[e][v] = ok ? to_f32(in[e].v[v]) : 0.f;
        sum += xh[e][v];
      }
    }
    const float mean = team_sum(sum, team_log) * inv;
    float squares = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const bool ok = live && row + ((uint32_t)e << plan.row_log) < k.pixels;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        xh[e][v] = ok ? xh[e][v] - mean : 0.f;
        squares = fmaf(xh[e][v], xh[e][v], squares);
      }
    }
    const float rstd = __builtin_amdgcn_rsqf(fmaf(team_sum(squares, team_log), inv, k.eps));
    T* y = (T*)k.y + (n * k.pixels) * k.width + c0;
    if constexpr (!BACKWARD) {
      if (k.stats && lane == 0 && row == 0) k.stats[n * k.groups + group] = {mean, rstd};
      with_act(k.act, [&](auto act) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const uint32_t p = row + ((uint32_t)e << plan.row_log);
          if (!live || p >= k.pixels) continue;
          Run<T, V> out;
#pragma unroll
          for (int v = 0; v < V; ++v)
            out.v[v] = from_f32<T>(
                act_value<act.value, T>(fmaf(xh[e][v] * rstd, w[v], b[v])));
          out.store(y + (uint64_t)p * k.width);
        }
      });
    } else {
      float dz[E][V], s1 = 0.f, s2 = 0.f;
      with_act(k.act, [&](auto act) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const bool ok = live && row + ((uint32_t)e << plan.row_log) < k.pixels;
#pragma unroll
          for (int v = 0; v < V; ++v) {
            xh[e][v] *= rstd;
            const float z = fmaf(xh[e][v], w[v], b[v]);
            dz[e][v] = ok ? to_f32(grad[e].v[v]) * act_slope<act.value, T>(z) : 0.f;
            dw[v] = fmaf(dz[e][v], xh[e][v], dw[v]);
            db[v] += dz[e][v];
            dz[e][v] *= w[v];
            s1 += dz[e][v];
            s2 = fmaf(dz[e][v], xh[e][v], s2);
          }
        }
      });
      if (k.y) {
        s1 = team_sum(s1, team_log) * inv;
        s2 = team_sum(s2, team_log) * inv;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const uint32_t p = row + ((uint32_t)e << plan.row_log);
          if (!live || p >= k.pixels) continue;
          Run<T, V> out;
#pragma unroll
          for (int v = 0; v < V; ++v)
            out.v[v] = from_f32<T>(rstd * (dz[e][v] - s1 - xh[e][v] * s2));
          out.store(y + (uint64_t)p * k.width);
        }
      }
    }
  }
  if constexpr (BACKWARD) {
    if (!partial) return;
#pragma unroll
    for (int v = 0; v < V; ++v)
      for (int j = lane_log; j < team_log; ++j) {
        dw[v] += __shfl_xor(dw[v], 1 << j, 64);
        db[v] += __shfl_xor(db[v], 1 << j, 64);
      }
    if (plan.teams < k.groups) {  // no two teams of a workgroup have the same channels
      if (live && row == 0) {
        float* out = partial + id / k.groups * 2 * k.width + c0;
#pragma unroll
        for (int v = 0; v < V; ++v) out[v] = dw[v], out[k.width + v] = db[v];
      }
      return;
    }
    __shared__ float s[2][256 * V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      s[0][threadIdx.x * V + v] = dw[v];
      s[1][threadIdx.x * V + v] = db[v];
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < 2 * k.width; i += 256) {
      const uint32_t c = i < k.width ? i : i - k.width;
      const uint32_t at = (((c / k.each) << team_log) * V) + c % k.each;
      const float* from = s[i < k.width ? 0 : 1] + at;
      float a = 0.f;
      for (uint32_t t = 0; t < plan.teams; t += k.groups) a += from[((uint64_t)t << team_log) * V];
      partial[(uint64_t)blockIdx.x * 2 * k.width + i] = a;
    }
  }
}

// dw and db: the partial rows' sums, 8 columns by 128 interleaved runs of rows a workgroup.
template <typename W>
__global__ void __launch_bounds__(1024) group_norm_join_kernel(uint32_t parts, uint32_t width,
                                                               const float* __restrict__ partial,
                                                               W* __restrict__ dweight,
                                                               W* __restrict__ dbias) {
  __shared__ float s[1024];
  const uint32_t c = blockIdx.x * 8 + threadIdx.x % 8, k = threadIdx.x / 8;
  float a = 0.f;
  if (c < 2 * width) {
#pragma unroll 8
    for (uint32_t p = k; p < parts; p += 128) a += partial[(uint64_t)p * 2 * width + c];
  }
  s[threadIdx.x] = a;
  for (uint32_t h = 64; h > 0; h >>= 1) {
    __syncthreads();
    if (k < h) s[threadIdx.x] += s[threadIdx.x + 8 * h];
  }
  if (k == 0 && c < 2 * width) {
    W* out = c < width ? dweight : dbias;
    if (out) out[c < width ? c : c - width] = from_f32<W>(s[threadIdx.x]);
  }
}

// ---------------------------------------------------------------------------
// Streamed groups.
// ---------------------------------------------------------------------------

struct StreamPlan {
  uint32_t tiles, columns;  // tiles of channels, vectors of a tile
  uint32_t threads_rows;    // pixels that a workgroup takes at once
  uint32_t chunks;          // of a sample's pixels
  uint64_t chunk;           // pixels of one
  uint64_t items;           // samples * tiles * chunks
};

struct Item {
  uint64_t n, first, last;  // sample, pixels
  uint32_t chunk, column;   // this thread's first channel
  uint32_t row;
  bool live;
};

template <int V>
__device__ __forceinline__ Item item_of(const GnCall& k, const StreamPlan& plan, uint64_t i) {
  Item it;
  it.chunk = (uint32_t)(i % plan.chunks);
  const uint64_t rest = i / plan.chunks;
  const uint32_t tile = (uint32_t)(rest % plan.tiles);
  it.n = rest / plan.tiles;
  it.first = it.chunk * plan.chunk;
  it.last = min(it.first + plan.chunk, k.pixels);
  it.row = threadIdx.x / plan.columns;
  const uint32_t vector = tile * plan.columns + threadIdx.x % plan.columns;
  it.column = vector * V;
  it.live = it.row < plan.threads_rows && vector < k.width / V;
  return it;
}

// Pixels of [first, last) that row r of a workgroup takes.
__device__ __forceinline__ uint32_t row_count(uint64_t pixels, uint32_t r, uint32_t rows) {
  return pixels > r ? (uint32_t)((pixels - r + rows - 1) / rows) : 0;
}

// Each channel's mean and sum of squared differences over a chunk of pixels.
template <typename T, int V>
__global__ void __launch_bounds__(256) group_norm_stats_kernel(GnCall k, StreamPlan plan,
                                                               float2* __restrict__ partial) {
  __shared__ float s_mean[256 * V], s_m2[256 * V];
  for (uint64_t i = blockIdx.x; i < plan.items; i += gridDim.x) {
    const Item it = item_of<V>(k, plan, i);
    const uint32_t rows = plan.threads_rows;
    float pivot[V] = {}, sum[V] = {}, squares[V] = {};
    if (it.live && it.first + it.row < it.last) {
      const T* x = (const T*)k.x + (int64_t)it.n * k.x_sample + it.column;
      Run<T, V> run;
      run.load(x + (int64_t)(it.first + it.row) * k.x_pitch);
#pragma unroll
      for (int v = 0; v < V; ++v) pivot[v] = to_f32(run.v[v]);
#pragma unroll 4
      for (uint64_t p = it.first + it.row + rows; p < it.last; p += rows) {
        run.load(x + (int64_t)p * k.x_pitch);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float d = to_f32(run.v[v]) - pivot[v];
          sum[v] += d;
          squares[v] = fmaf(d, d, squares[v]);
        }
      }
    }
    const uint32_t count = row_count(it.last - it.first, it.row, rows);
    const float inv = count ? 1.f / (float)count : 0.f;
    __syncthreads();  // (the last item's values are read)
    if (it.row < rows) {
      const uint32_t at = threadIdx.x * V;  // rows of `columns` vectors
#pragma unroll
      for (int v = 0; v < V; ++v) {
        s_mean[at + v] = fmaf(sum[v], inv, pivot[v]);
        s_m2[at + v] = fmaxf(fmaf(-sum[v] * inv, sum[v], squares[v]), 0.f);
      }
    }
    __syncthreads();
    const uint32_t wide = plan.columns * V, tile = it.column / wide * wide;
    const float all = 1.f / (float)(it.last - it.first);
    for (uint32_t c = threadIdx.x; c < wide && tile + c < k.width; c += 256) {
      float mean = 0.f, m2 = 0.f;
      for (uint32_t r = 0; r < rows; ++r)
        mean = fmaf(s_mean[r * wide + c],
                    (float)row_count(it.last - it.first, r, rows) * all, mean);
      for (uint32_t r = 0; r < rows; ++r) {
        const float d = s_mean[r * wide + c] - mean;
        const float n = (float)row_count(it.last - it.first, r, rows);
        m2 += n > 0.f ? fmaf(n * d, d, s_m2[r * wide + c]) : 0.f;
      }
      partial[(it.n * plan.chunks + it.chunk) * k.width + tile + c] = {mean, m2};
    }
  }
}

__device__ __forceinline__ double sum_of_workgroup(double v, double* s) {
#pragma unroll
  for (int off = 32; off; off >>= 1) v += __shfl_xor(v, off, 64);
  __syncthreads();
  if (threadIdx.x % 64 == 0) s[threadIdx.x / 64] = v;
  __syncthreads();
  return (s[0] + s[1]) + (s[2] + s[3]);
}

// Mean and rstd of each sample's group, a workgroup each, in 64 bits.
__global__ void __launch_bounds__(256) group_norm_finish_kernel(GnCall k, StreamPlan plan,
                                                                const float2* __restrict__ partial) {
  __shared__ double s[4];
  for (uint64_t i = blockIdx.x; i < k.samples * k.groups; i += gridDim.x) {
    const uint64_t n = i / k.groups;
    const float2* from = partial + n * plan.chunks * k.width + i % k.groups * k.each;
    const uint64_t entries = (uint64_t)plan.chunks * k.each;
    const auto entry = [&](uint64_t e) { return from[e / k.each * k.width + e % k.each]; };
    const auto pixels = [&](uint64_t e) {
      const uint64_t first = e / k.each * plan.chunk;
      return (double)(min(first + plan.chunk, k.pixels) - first);
    };
    const double m = (double)k.pixels * k.each;
    double a = 0;
    for (uint64_t e = threadIdx.x; e < entries; e += 256) a += entry(e).x * pixels(e);
    const double mean = sum_of_workgroup(a, s) / m;
    double q = 0;
    for (uint64_t e = threadIdx.x; e < entries; e += 256) {
      const float2 p = entry(e);
      const double d = p.x - mean;
      q += p.y + pixels(e) * d * d;
    }
    q = sum_of_workgroup(q, s) / m;
    if (threadIdx.x == 0) k.stats[i] = {(float)mean, (float)(1.0 / sqrt(q + (double)k.eps))};
  }
}

// What a thread needs of its channels.
template <typename T, int V>
struct Columns {
  float mean[V], rstd[V], w[V], b[V];
  __device__ __forceinline__ void load(const GnCall& k, const Item& it) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const uint32_t c = it.column + v;
      const float2 st = k.stats[it.n * k.groups + c / k.each];
      mean[v] = st.x, rstd[v] = st.y;
      w[v] = column<T>(k.weight, k.wide_weights, c, 1.f);
      b[v] = column<T>(k.bias, k.wide_weights, c, 0.f);
    }
  }
};

template <typename T, int V>
__global__ void __launch_bounds__(256) group_norm_apply_kernel(GnCall k, StreamPlan plan) {
  for (uint64_t i = blockIdx.x; i < plan.items; i += gridDim.x) {
    const Item it = item_of<V>(k, plan, i);
    if (!it.live) continue;
    Columns<T, V> col;
    col.load(k, it);
    const T* x = (const T*)k.x + (int64_t)it.n * k.x_sample + it.column;
    T* y = (T*)k.y + it.n * k.pixels * k.width + it.column;
    with_act(k.act, [&](auto act) {
#pragma unroll 4
      for (uint64_t p = it.first + it.row; p < it.last; p += plan.threads_rows) {
        Run<T, V> run;
        run.load(x + (int64_t)p * k.x_pitch);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float xh = (to_f32(run.v[v]) - col.mean[v]) * col.rstd[v];
          run.v[v] = from_f32<T>(act_value<act.value, T>(fmaf(xh, col.w[v], col.b[v])));
        }
        run.store(y + p * k.width);
      }
    });
  }
}

// Each channel's sums of dz and dz xhat over a chunk of pixels.
template <typename T, int V>
__global__ void __launch_bounds__(256) group_norm_sums_kernel(GnCall k, StreamPlan plan,
                                                              float2* __restrict__ partial) {
  __shared__ float s[2][256 * V];
  for (uint64_t i = blockIdx.x; i < plan.items; i += gridDim.x) {
    const Item it = item_of<V>(k, plan, i);
    float db[V] = {}, dw[V] = {};
    if (it.live) {
      Columns<T, V> col;
      col.load(k, it);
      const T* x = (const T*)k.x + (int64_t)it.n * k.x_sample + it.column;
      const T* dy = (const T*)k.dy + (int64_t)it.n * k.dy_sample + it.column;
      with_act(k.act, [&](auto act) {
#pragma unroll 2
        for (uint64_t p = it.first + it.row; p < it.last; p += plan.threads_rows) {
          Run<T, V> run, grad;
          run.load(x + (int64_t)p * k.x_pitch);
          grad.load(dy + (int64_t)p * k.dy_pitch);
#pragma unroll
          for (int v = 0; v < V; ++v) {
            const float xh = (to_f32(run.v[v]) - col.mean[v]) * col.rstd[v];
            const float dz =
                to_f32(grad.v[v]) * act_slope<act.value, T>(fmaf(xh, col.w[v], col.b[v]));
            db[v] += dz;
            dw[v] = fmaf(dz, xh, dw[v]);
          }
        }
      });
    }
    __syncthreads();
    if (it.row < plan.threads_rows) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        s[0][threadIdx.x * V + v] = db[v];
        s[1][threadIdx.x * V + v] = dw[v];
      }
    }
    __syncthreads();
    const uint32_t wide = plan.columns * V, tile = it.column / wide * wide;
    for (uint32_t c = threadIdx.x; c < wide && tile + c < k.width; c += 256) {
      float a = 0.f, b = 0.f;
      for (uint32_t r = 0; r < plan.threads_rows; ++r) {
        a += s[0][r * wide + c];
        b += s[1][r * wide + c];
      }
      partial[(it.n * plan.chunks + it.chunk) * k.width + tile + c] = {a, b};
    }
  }
}

// A sample's sums by channel (rows of dw, db for the join) and by group (sum(g) / m and
// sum(g xhat) / m), a workgroup for each group: 32 runs of chunks by 8 channels.
template <typename T>
__global__ void __launch_bounds__(256) group_norm_group_sums_kernel(
    GnCall k, StreamPlan plan, const float2* __restrict__ partial, float* __restrict__ rows,
    float2* __restrict__ sums) {
  __shared__ float s_a[256], s_b[256];
  for (uint64_t i = blockIdx.x; i < k.samples * k.groups; i += gridDim.x) {
    const uint64_t n = i / k.groups;
    const uint32_t c0 = (uint32_t)(i % k.groups) * k.each, lane = threadIdx.x % 8;
    float s1 = 0.f, s2 = 0.f;  // (of the threads below 8)
    for (uint32_t j = 0; j < k.each; j += 8) {
      const uint32_t c = c0 + j + lane;
      const bool ok = j + lane < k.each;
      float a = 0.f, b = 0.f;
      if (ok)
        for (uint32_t q = threadIdx.x / 8; q < plan.chunks; q += 32) {
          const float2 p = partial[(n * plan.chunks + q) * k.width + c];
          a += p.x, b += p.y;
        }
      s_a[threadIdx.x] = a, s_b[threadIdx.x] = b;
      for (uint32_t h = 128; h >= 8; h >>= 1) {
        __syncthreads();
        if (threadIdx.x < h) {
          s_a[threadIdx.x] += s_a[threadIdx.x + h];
          s_b[threadIdx.x] += s_b[threadIdx.x + h];
        }
      }
      if (threadIdx.x < 8 && ok) {
        a = s_a[lane], b = s_b[lane];
        const float w = column<T>(k.weight, k.wide_weights, c, 1.f);
        s1 = fmaf(w, a, s1);
        s2 = fmaf(w, b, s2);
        if (rows) rows[n * 2 * k.width + c] = b, rows[(n * 2 + 1) * k.width + c] = a;
      }
      __syncthreads();
    }
    for (int off = 4; off; off >>= 1) s1 += __shfl_xor(s1, off, 8), s2 += __shfl_xor(s2, off, 8);
    if (threadIdx.x == 0) {
      const double m = (double)k.pixels * k.each;
      sums[i] = {(float)(s1 / m), (float)(s2 / m)};
    }
  }
}

template <typename T, int V>
__global__ void __launch_bounds__(256) group_norm_dx_kernel(GnCall k, StreamPlan plan,
                                                            const float2* __restrict__ sums) {
  for (uint64_t i = blockIdx.x; i < plan.items; i += gridDim.x) {
    const Item it = item_of<V>(k, plan, i);
    if (!it.live) continue;
    Columns<T, V> col;
    col.load(k, it);
    float s1[V], s2[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float2 p = sums[it.n * k.groups + (it.column + v) / k.each];
      s1[v] = p.x, s2[v] = p.y;
    }
    const T* x = (const T*)k.x + (int64_t)it.n * k.x_sample + it.column;
    const T* dy = (const T*)k.dy + (int64_t)it.n * k.dy_sample + it.column;
    T* dx = (T*)k.y + it.n * k.pixels * k.width + it.column;
    with_act(k.act, [&](auto act) {
#pragma unroll 2
      for (uint64_t p = it.first + it.row; p < it.last; p += plan.threads_rows) {
        Run<T, V> run, grad;
        run.load(x + (int64_t)p * k.x_pitch);
        grad.load(dy + (int64_t)p * k.dy_pitch);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float xh = (to_f32(run.v[v]) - col.mean[v]) * col.rstd[v];
          const float g = to_f32(grad.v[v]) *
                          act_slope<act.value, T>(fmaf(xh, col.w[v], col.b[v])) * col.w[v];
          run.v[v] = from_f32<T>(col.rstd[v] * (g - s1[v] - xh * s2[v]));
        }
        run.store(dx + p * k.width);
      }
    });
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

static int log2_up(uint64_t n) {
  int k = 0;
  while ((1ull << k) < n) ++k;
  return k;
}

static uint32_t size_of(int32_t dtype) { return dtype == TGS_F32 ? 4 : 2; }

// Values of a lane's load: the most of 16 bytes, four values and one that n (the channels of a
// group where a team holds it, of a pixel otherwise) are a whole number of.
static uint32_t vector_of(uint32_t n, int32_t dtype) {
  for (uint32_t v = 16 / size_of(dtype); v >= 4; v /= 2)
    if (n % v == 0) return v;
  return 1;
}

static bool held_plan(uint64_t samples, uint64_t pixels, uint32_t groups, uint32_t each,
                      uint32_t v, HeldPlan& plan) {
  plan.lane_log = log2_up(each / v);
  if (plan.lane_log > 6 || pixels > 64 * HELD_RUNS) return false;
  plan.row_log = std::min(6 - plan.lane_log, log2_up(pixels));
  plan.runs = (int)((pixels + (1u << plan.row_log) - 1) >> plan.row_log);
  if (plan.runs > HELD_RUNS) return false;
  const uint32_t teams = 256 >> (plan.lane_log + plan.row_log);
  if (teams >= groups) {
    const uint32_t each_wg = teams / groups;  // samples of a workgroup at once
    plan.teams = each_wg * groups;
    plan.grid = (uint32_t)std::min<uint64_t>((samples + each_wg - 1) / each_wg, 2048);
    plan.rows = plan.grid * each_wg;
    plan.partials = plan.grid;
  } else {
    plan.teams = teams;
    plan.rows = (uint32_t)std::min<uint64_t>(
        samples, std::max<uint64_t>(1, 2048ull * teams / groups));
    plan.grid = (uint32_t)(((uint64_t)plan.rows * groups + teams - 1) / teams);
    plan.partials = plan.rows;
  }
  return true;
}

static StreamPlan stream_plan(uint64_t samples, uint64_t pixels, uint32_t width, uint32_t v) {
  StreamPlan plan;
  const uint32_t vectors = width / v;
  plan.tiles = (vectors + TILE_VECTORS - 1) / TILE_VECTORS;
  plan.columns = (vectors + plan.tiles - 1) / plan.tiles;
  plan.threads_rows = 256 / plan.columns;
  // about 2048 workgroups, each with 8 pixels a thread at least
  const uint64_t wanted = std::max<uint64_t>(1, 2048 / std::max<uint64_t>(1, samples * plan.tiles));
  const uint64_t least = 8ull * plan.threads_rows;
  plan.chunk = std::max((pixels + wanted - 1) / wanted, least);
  plan.chunk = (plan.chunk + plan.threads_rows - 1) / plan.threads_rows * plan.threads_rows;
  plan.chunks = (uint32_t)((pixels + plan.chunk - 1) / plan.chunk);
  plan.items = samples * plan.tiles * plan.chunks;
  return plan;
}

static uint32_t capped(uint64_t n) { return (uint32_t)std::min<uint64_t>(n, 1u << 20); }

static bool gn_sizes_ok(uint64_t samples, uint64_t pixels, uint32_t width, uint32_t groups,
                        int32_t dtype) {
  return width > 0 && width <= 65536 && groups > 0 && width % groups == 0 &&
         dtype >= TGS_F32 && dtype <= TGS_F16 && samples < (1ull << 40) && pixels < (1ull << 40);
}

static bool gn_held(uint64_t samples, uint64_t pixels, uint32_t width, uint32_t groups,
                    int32_t dtype, HeldPlan& plan) {
  const uint32_t each = width / groups;
  return held_plan(samples, pixels, groups, each, vector_of(each, dtype), plan);
}

// Calls f(T, V) as a value and a constant.
template <typename F>
static void with_vector(int32_t dtype, uint32_t v, F&& f) {
  with_dtype(dtype, "tgs_group_norm", [&](auto tag) {
    using T = decltype(tag);
    if (v == 1)
      f(tag, std::integral_constant<int, 1>());
    else if (v == 4 || sizeof(T) == 4)
      f(tag, std::integral_constant<int, 4>());
    else
      f(tag, std::integral_constant<int, 16 / sizeof(T)>());
    return TGS_OK;
  });
}

template <bool BACKWARD>
static void held_launch(const GnCall& k, const HeldPlan& plan, int32_t dtype, float* partial,
                        hipStream_t stream) {
  with_vector(dtype, vector_of(k.each, dtype), [&](auto tag, auto v) {
    using T = decltype(tag);
    const auto launch = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3(plan.grid), dim3(256), 0, stream, k, plan, partial);
    };
    if (plan.runs == 1)
      launch(group_norm_held_kernel<T, v.value, 1, BACKWARD>);
    else if (plan.runs == 2)
      launch(group_norm_held_kernel<T, v.value, 2, BACKWARD>);
    else if (plan.runs <= 4)
      launch(group_norm_held_kernel<T, v.value, 4, BACKWARD>);
    else
      launch(group_norm_held_kernel<T, v.value, 8, BACKWARD>);
  });
}

extern "C" uint64_t tgs_group_norm_stats_size(uint64_t samples, uint64_t pixels, uint32_t width,
                                              uint32_t groups, int32_t dtype) {
  HeldPlan plan;
  if (!gn_sizes_ok(samples, pixels, width, groups, dtype) || samples == 0 || pixels == 0 ||
      gn_held(samples, pixels, width, groups, dtype, plan))
    return 0;
  return samples * groups * sizeof(float2);
}

extern "C" uint64_t tgs_group_norm_fwd_workspace_size(uint64_t samples, uint64_t pixels,
                                                      uint32_t width, uint32_t groups,
                                                      int32_t dtype) {
  HeldPlan held;
  if (!gn_sizes_ok(samples, pixels, width, groups, dtype) || samples == 0 || pixels == 0 ||
      gn_held(samples, pixels, width, groups, dtype, held))
    return 0;
  const StreamPlan plan = stream_plan(samples, pixels, width, vector_of(width, dtype));
  return samples * plan.chunks * width * sizeof(float2);
}

extern "C" uint64_t tgs_group_norm_bwd_workspace_size(uint64_t samples, uint64_t pixels,
                                                      uint32_t width, uint32_t groups,
                                                      int32_t dtype) {
  HeldPlan held;
  if (!gn_sizes_ok(samples, pixels, width, groups, dtype) || samples == 0 || pixels == 0) return 0;
  if (gn_held(samples, pixels, width, groups, dtype, held))
    return (uint64_t)held.partials * 2 * width * sizeof(float);
  const StreamPlan plan = stream_plan(samples, pixels, width, vector_of(width, dtype));
  return samples * sizeof(float2) * ((plan.chunks + 1ull) * width + groups);
}

#define GN_CHECK_CALL(name)                                                                      \
  TGS_CHECK_ARG(gn_sizes_ok(samples, pixels, width, groups, dtype) ||                            \
                    (dtype < TGS_F32 || dtype > TGS_F16),                                        \
                name ": width %u must lie in 1..65536 and be a multiple of the %u groups, "      \
                     "samples and pixels below 2^40", width, groups);                            \
  TGS_CHECK_ARG(dtype >= TGS_F32 && dtype <= TGS_F16,                                            \
                name ": dtype must be 0 (float32), 1 (bfloat16) or 2 (float16), got %d", dtype); \
  TGS_CHECK_ARG(weight_dtype == dtype || weight_dtype == TGS_F32,                                \
                name ": the weights have x's type or float32");                                  \
  TGS_CHECK_ARG(activation >= 0 && activation <= ACT_NONE, name ": activation %d", activation);  \
  TGS_CHECK_ARG(eps >= 0x1p-80f && eps <= 0x1p80f,                                               \
                name ": eps must lie in 2^-80..2^80 (squares below it leave float32)")

extern "C" int tgs_group_norm_fwd(uint64_t samples, uint64_t pixels, uint32_t width,
                                  uint32_t groups, int32_t dtype, int32_t activation,
                                  const void* x, int64_t x_sample, int64_t x_pitch,
                                  const void* weight, const void* bias, int32_t weight_dtype,
                                  float eps, void* y, float* stats, void* workspace,
                                  uint64_t workspace_bytes, hipStream_t stream) {
  GN_CHECK_CALL("tgs_group_norm_fwd");
  if (samples == 0 || pixels == 0) return TGS_OK;
  TGS_CHECK_ARG(x && y, "tgs_group_norm_fwd: null pointer");
  TGS_CHECK_ARG(x_pitch >= (int64_t)width || pixels == 1, "tgs_group_norm_fwd: pitch below width");
  GnCall k = {samples, pixels, width, groups, width / groups, activation,
              weight_dtype != dtype, x, nullptr, x_sample, x_pitch, 0, 0, weight, bias, eps, y,
              (float2*)stats};
  HeldPlan held;
  if (gn_held(samples, pixels, width, groups, dtype, held)) {
    k.stats = nullptr;
    held_launch<false>(k, held, dtype, nullptr, stream);
    TGS_RETURN_LAUNCH("tgs_group_norm_fwd");
  }
  TGS_CHECK_ARG(stats, "tgs_group_norm_fwd: null stats");
  if (workspace_bytes <
      tgs_group_norm_fwd_workspace_size(samples, pixels, width, groups, dtype)) {
    tgs_set_error("tgs_group_norm_fwd: workspace too small");
    return TGS_ERR_WORKSPACE;
  }
  TGS_CHECK_ARG(workspace && (uintptr_t)workspace % 8 == 0 && (uintptr_t)stats % 8 == 0,
                "tgs_group_norm_fwd: the workspace and the stats start on 8 bytes");
  const uint32_t v = vector_of(width, dtype);
  const StreamPlan plan = stream_plan(samples, pixels, width, v);
  const dim3 grid(capped(plan.items)), by_group(capped(samples * groups));
  float2* partial = (float2*)workspace;
  with_vector(dtype, v, [&](auto tag, auto vec) {
    using T = decltype(tag);
    hipLaunchKernelGGL((group_norm_stats_kernel<T, vec.value>), grid, dim3(256), 0, stream, k,
                       plan, partial);
    hipLaunchKernelGGL(group_norm_finish_kernel, by_group, dim3(256), 0, stream, k, plan, partial);
    hipLaunchKernelGGL((group_norm_apply_kernel<T, vec.value>), grid, dim3(256), 0, stream, k,
                       plan);
  });
  TGS_RETURN_LAUNCH("tgs_group_norm_fwd");
}

extern "C" int tgs_group_norm_bwd(uint64_t samples, uint64_t pixels, uint32_t width,
                                  uint32_t groups, int32_t dtype, int32_t activation,
                                  const void* x, int64_t x_sample, int64_t x_pitch,
                                  const void* dy, int64_t dy_sample, int64_t dy_pitch,
                                  const void* weight, const void* bias, int32_t weight_dtype,
                                  float eps, const float* stats, void* dx, void* dweight,
                                  void* dbias, void* workspace, uint64_t workspace_bytes,
                                  hipStream_t stream) {
  GN_CHECK_CALL("tgs_group_norm_bwd");
  const bool sums = dweight || dbias, any = samples > 0 && pixels > 0;
  if (!sums && (!dx || !any)) return TGS_OK;
  TGS_CHECK_ARG(!any || (x && dy), "tgs_group_norm_bwd: null pointer");
  TGS_CHECK_ARG((x_pitch >= (int64_t)width && dy_pitch >= (int64_t)width) || pixels <= 1,
                "tgs_group_norm_bwd: pitch below width");
  if (any && workspace_bytes <
                 tgs_group_norm_bwd_workspace_size(samples, pixels, width, groups, dtype)) {
    tgs_set_error("tgs_group_norm_bwd: workspace too small");
    return TGS_ERR_WORKSPACE;
  }
  TGS_CHECK_ARG(!any || (workspace && (uintptr_t)workspace % 8 == 0),
                "tgs_group_norm_bwd: the workspace starts on 8 bytes");
  GnCall k = {samples, pixels, width, groups, width / groups, activation,
              weight_dtype != dtype, x, dy, x_sample, x_pitch, dy_sample, dy_pitch, weight, bias,
              eps, dx, (float2*)stats};
  const auto join = [&](uint32_t parts, const float* rows) {
    if (!sums) return;
    with_dtype(weight_dtype, "tgs_group_norm_bwd", [&](auto tag) {
      using W = decltype(tag);
      hipLaunchKernelGGL(group_norm_join_kernel<W>, dim3((2 * width + 7) / 8), dim3(1024), 0,
                         stream, parts, width, rows, (W*)dweight, (W*)dbias);
      return TGS_OK;
    });
  };
  HeldPlan held;
  if (!any) {
    join(0, nullptr);  // zeros
  } else if (gn_held(samples, pixels, width, groups, dtype, held)) {
    float* partial = sums ? (float*)workspace : nullptr;
    held_launch<true>(k, held, dtype, partial, stream);
    join(held.partials, partial);
  } else {
    TGS_CHECK_ARG(stats && (uintptr_t)stats % 8 == 0,
                  "tgs_group_norm_bwd: the stats of the forward are needed, on 8 bytes");
    TGS_CHECK_ARG(!sums || samples < (1ull << 32), "tgs_group_norm_bwd: 2^32 samples and more");
    const uint32_t v = vector_of(width, dtype);
    const StreamPlan plan = stream_plan(samples, pixels, width, v);
    const dim3 grid(capped(plan.items)), by_group(capped(samples * groups));
    float2* partial = (float2*)workspace;
    float* rows = (float*)(partial + samples * plan.chunks * width);
    float2* group_sums = (float2*)rows + samples * width;
    with_vector(dtype, v, [&](auto tag, auto vec) {
      using T = decltype(tag);
      hipLaunchKernelGGL((group_norm_sums_kernel<T, vec.value>), grid, dim3(256), 0, stream, k,
                         plan, partial);
      hipLaunchKernelGGL(group_norm_group_sums_kernel<T>, by_group, dim3(256), 0, stream, k, plan,
                         partial, sums ? rows : nullptr, group_sums);
      if (dx)
        hipLaunchKernelGGL((group_norm_dx_kernel<T, vec.value>), grid, dim3(256), 0, stream, k,
                           plan, group_sums);
    });
    join((uint32_t)samples, rows);
  }
  TGS_RETURN_LAUNCH("tgs_group_norm_bwd");
}
