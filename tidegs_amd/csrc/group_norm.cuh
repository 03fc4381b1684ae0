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
// Held (up to 4 runs of 16 bytes a lane of 64, or 8 of a workgroup's 256): a team of lanes
// keeps a group in registers, so x is read once and one launch does all.  The backward computes
// mean and rstd again.
//
// Streamed: workgroups take runs of pixels by up to 64 vectors of channels and leave each channel's
// mean and sum of squared differences (of dz and dz xhat in the backward); they are joined by
// group, by the workgroups that read x again and write where they are few, by a launch of its
// own otherwise.  The forward keeps mean and rstd for the backward.
//
// Pixels are dealt out to a streaming launch's workgroups a run of rows each in turn, so that all
// of them read one stretch of memory at a time, and the launch that reads x again begins at its
// end, which is still cached in part (backward of 4 x 960x540x64 bfloat16: 307 -> 268 us for both).
// Runs need their elements' alignment only, and where a group or a pixel is no whole number of
// them the last one overlaps the one before.
//
// Sums of squares are of differences from a value near by (a thread's first one, a mean), and
// partial ones are joined by their means, so no large mean cancels.  All joins are in a fixed
// order.  Sums are taken in 32 bits, those over a whole group's partial values in 64.
//
// 1M rows of 64 bfloat16 in 4 groups, held: forward 45 us (5.6 TB/s), backward 77 (5.0 TB/s) and 6
// for the weights' gradients.  1920x1080x32 bfloat16, silu, streamed: 27 + 7 + 49 us (4.9 and 5.4
// TB/s, x read twice); 4 x 960x540x64, both directions: 62 + 6 + 91 and 115 + 7 + 139 + 7 us (4.3,
// 5.8, 4.6 and 5.7 TB/s).  16 x 1020 pixels of 512 halves in 32 groups, held by workgroups: 13
// and 34 us, of 32-byte pieces of cache lines.
#pragma once

#include "activation.cuh"
#include "vector_io.cuh"

#define ACT_NONE 3
// Groups of up to so many runs a lane are held, of a workgroup's lanes and of a wavefront's (eight
// took 460 registers in the backward).  16 x 1020 pixels of 512 halves in 32 groups: forward 13 us
// held and 26 streamed, backward 34 and 32, in one launch less each.
#define HELD_RUNS 8
#define HELD_FEW 4
#define TILE_VECTORS 64  // vectors of channels of a streaming workgroup
// The workgroups that read partial values join them for themselves up to so many channels,
// channels of a group, partial values of a sample and values of x, if at least so many workgroups
// leave them: 3 x 241x137x48 float32, both directions: 65 us of kernels in five launches and in
// seven, and 4 us less of the host's time for each launch.
#define JOINED_WIDTH 512
#define JOINED_EACH 64
#define JOINED_ENTRIES 4096
#define JOINED_BELOW (1u << 24)
#define JOINED_WORKGROUPS 192

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
  int32_t once;   // whether y is stored past the caches
};

// Calls f with the activation as a constant.  The kernels do so around their loops: inside of them
// the four forms' registers add up (held backward of one run: 121, outside 86).
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

// Stores of a second pass that reads what the first one left in the caches.  Large outputs go past
// them, measured with y alone and y read by the next kernel (bfloat16, 64 channels, silu, us, plain
// and past): 64 MB 66, 64 and 85.5, 86; 128 MB 94, 91.5 and 149, 147; 256 MB 187, 155 and 283, 262;
// 512 MB 355, 325 and 536, 520.  Held groups, read once, lose by it (128 MB: 92, 102 with y read),
// and so does dx (4 x 960x540x64, both directions: 411 past the caches, 399 plain).
#define ONCE_BYTES (96ull << 20)

template <typename T, int V>
__device__ __forceinline__ void store(const GnCall& k, const Run<T, V>& run, T* p) {
  if (k.once)
    run.store_once(p);
  else
    run.store(p);
}

// Sum over a team: 2^log lanes of a wavefront, or (WIDE) the workgroup.
template <bool WIDE>
__device__ __forceinline__ float team_sum(float v, int log) {
  if constexpr (WIDE) {
    __shared__ float s[4];
    v = tgs_wave_sum(v);
    __syncthreads();
    if (threadIdx.x % 64 == 0) s[threadIdx.x / 64] = v;
    __syncthreads();
    return (s[0] + s[1]) + (s[2] + s[3]);
  } else {
    for (int k = 0; k < log; ++k) v += __shfl_xor(v, 1 << k, 64);
    return v;
  }
}

// ---------------------------------------------------------------------------
// Held groups.  A team has 2^row_log rows of 2^lane_log lanes (as many as hold a pixel's
// vectors of the group); teams of a workgroup take neighbouring groups.  A team keeps to one
// group's channels over all its samples, so weights are read once and the weights' gradients
// stay in registers.  WIDE: the workgroup is one team, and neighbouring groups, which share cache
// lines, go to one XCD's workgroups (they are dealt out round robin).
//
// TAIL: the group is no whole number of runs, and the last one ends where it ends: what it has in
// common with the run before counts once, in that one, and is written twice, the same.
// ---------------------------------------------------------------------------

struct HeldPlan {
  uint32_t v;         // values of a run
  bool tail;          // whether a group's last run overlaps the one before
  int lane_log, row_log;
  uint32_t teams;    // of a workgroup that work
  uint32_t rows;     // samples that all teams take at once
  uint32_t grid;
  uint32_t partials;  // rows of the weights' gradients
  int runs;           // of a lane
  bool wide;          // a team is a workgroup
};

template <typename T, int V, int E, bool BACKWARD, bool WIDE, bool TAIL>
__global__ void __launch_bounds__(256) group_norm_held_kernel(GnCall k, HeldPlan plan,
                                                              float* __restrict__ partial) {
  const int lane_log = plan.lane_log, team_log = lane_log + plan.row_log;
  const uint32_t lane = threadIdx.x & ((1u << lane_log) - 1);
  const uint32_t row = (threadIdx.x >> lane_log) & ((1u << plan.row_log) - 1);
  const uint32_t team = threadIdx.x >> team_log;
  uint64_t id = (uint64_t)blockIdx.x * plan.teams + team;
  if (WIDE && gridDim.x % 8 == 0) id = (blockIdx.x % 8) * (gridDim.x / 8) + blockIdx.x / 8;
  const bool works = team < plan.teams && id < (uint64_t)plan.rows * k.groups;
  const uint32_t group = (uint32_t)(id % k.groups);
  const bool live = works && lane * V < k.each;
  const uint32_t in_group = TAIL ? min(lane * V, k.each - V) : lane * V;
  const uint32_t c0 = group * k.each + in_group, skip = lane * V - in_group;
  const auto counts = [&](int v) { return !TAIL || (uint32_t)v >= skip; };
  const float inv = 1.f / (float)(k.pixels * k.each);
  float w[V], b[V], dw[V] = {}, db[V] = {};
#pragma unroll
  for (int v = 0; v < V; ++v) {
    w[v] = live ? column<T>(k.weight, k.wide_weights, c0 + v, 1.f) : 0.f;
    b[v] = live ? column<T>(k.bias, k.wide_weights, c0 + v, 0.f) : 0.f;
  }
  with_act(k.act, [&](auto act) {
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
          sum += counts(v) ? xh[e][v] : 0.f;
        }
      }
      const float mean = team_sum<WIDE>(sum, team_log) * inv;
      float squares = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const bool ok = live && row + ((uint32_t)e << plan.row_log) < k.pixels;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          xh[e][v] = ok ? xh[e][v] - mean : 0.f;
          squares = counts(v) ? fmaf(xh[e][v], xh[e][v], squares) : squares;
        }
      }
      const float rstd = __builtin_amdgcn_rsqf(fmaf(team_sum<WIDE>(squares, team_log), inv, k.eps));
      T* y = (T*)k.y + (n * k.pixels) * k.width + c0;
      if constexpr (!BACKWARD) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const uint32_t p = row + ((uint32_t)e << plan.row_log);
          if (!live || p >= k.pixels) continue;
          Run<T, V> out;
#pragma unroll
          for (int v = 0; v < V; ++v)
            out.v[v] = from_f32<T>(act_value<act.value, T>(fmaf(xh[e][v] * rstd, w[v], b[v])));
          out.store(y + (uint64_t)p * k.width);
        }
      } else {
        // Few runs keep xhat and dz w for the second pass over the team's values.  Many compute
        // them again: kept, the two take 128 registers of eight runs, 460 in all.
        constexpr bool KEEP = E <= HELD_FEW / 2;
        float g[KEEP ? E : 1][V], s1 = 0.f, s2 = 0.f;
        const auto ok = [&](int e) {
          return live && row + ((uint32_t)e << plan.row_log) < k.pixels;
        };
        const auto both = [&](int e, int v, float& xhat, float& dz) {
          xhat = (to_f32(in[e].v[v]) - mean) * rstd;
          dz = to_f32(grad[e].v[v]) * act_slope<act.value, T>(fmaf(xhat, w[v], b[v]));
        };
#pragma unroll
        for (int e = 0; e < E; ++e) {
          if (!ok(e)) continue;
#pragma unroll
          for (int v = 0; v < V; ++v) {
            float xhat, dz;
            both(e, v, xhat, dz);
            dw[v] = fmaf(dz, xhat, dw[v]);
            db[v] += dz;
            dz *= w[v];
            s1 += counts(v) ? dz : 0.f;
            s2 = counts(v) ? fmaf(dz, xhat, s2) : s2;
            if constexpr (KEEP) xh[e][v] = xhat, g[e][v] = dz;
          }
        }
        if (!k.y) continue;
        s1 = team_sum<WIDE>(s1, team_log) * inv;
        s2 = team_sum<WIDE>(s2, team_log) * inv;
        if constexpr (!KEEP) {
#pragma unroll
          for (int e = 0; e < E; ++e) in[e].forget(), grad[e].forget();
        }
#pragma unroll
        for (int e = 0; e < E; ++e) {
          if (!ok(e)) continue;
          Run<T, V> out;
#pragma unroll
          for (int v = 0; v < V; ++v) {
            float xhat, dz;
            if constexpr (KEEP) {
              xhat = xh[e][v], dz = g[e][v];
            } else {
              both(e, v, xhat, dz);
              dz *= w[v];
            }
            out.v[v] = from_f32<T>(rstd * (dz - s1 - xhat * s2));
          }
          out.store(y + (uint64_t)(row + ((uint32_t)e << plan.row_log)) * k.width);
        }
      }
    }
  });
  if constexpr (BACKWARD) {
    if (!partial) return;
    // over the rows of a wavefront
    const int in_wave = min(team_log, 6);
#pragma unroll
    for (int v = 0; v < V; ++v)
      for (int j = lane_log; j < in_wave; ++j) {
        dw[v] += __shfl_xor(dw[v], 1 << j, 64);
        db[v] += __shfl_xor(db[v], 1 << j, 64);
      }
    if (!WIDE && plan.teams < k.groups) {  // no two teams of a workgroup have the same channels
      if (live && row == 0) {
        float2* out = (float2*)partial + id / k.groups * k.width + c0;
#pragma unroll
        for (int v = 0; v < V; ++v) out[v] = {db[v], dw[v]};
      }
      return;
    }
    // WIDE: over the wavefronts (one row of each, all rows where a row is longer than one);
    // otherwise over the teams of the same group
    __shared__ float2 s[256 * V];
    const int rows_log = WIDE ? max(6 - lane_log, 0) : 0;
    const uint32_t at = WIDE ? ((row >> rows_log) << lane_log) + lane : threadIdx.x;
    if (!WIDE || (row & ((1u << rows_log) - 1)) == 0) {
#pragma unroll
      for (int v = 0; v < V; ++v) s[at * V + v] = {db[v], dw[v]};
    }
    __syncthreads();
    const uint32_t channels = WIDE ? k.each : k.width, step = WIDE ? 1 : k.groups;
    const uint32_t count = WIDE ? 1u << (plan.row_log - rows_log) : plan.teams;
    const uint32_t stride = (1u << (WIDE ? lane_log : team_log)) * V;
    float2* out = (float2*)partial + (WIDE ? id / k.groups * k.width + group * k.each
                                           : (uint64_t)blockIdx.x * k.width);
    const uint32_t last = (k.each - 1) / V * V;  // the last run's first channel without overlap
    for (uint32_t c = threadIdx.x; c < channels; c += 256) {
      const uint32_t team0 = WIDE ? 0 : c / k.each, in = c - team0 * k.each;
      const uint32_t of = TAIL && in >= last ? last + in - (k.each - V) : in;
      const float2* from = s + (team0 << team_log) * V + of;
      float2 a = {0.f, 0.f};
      for (uint32_t t = 0; t < count; t += step) {
        const float2 p = from[t * stride];
        a.x += p.x, a.y += p.y;
      }
      out[c] = a;
    }
  }
}

// ---------------------------------------------------------------------------
// Streamed groups.
// ---------------------------------------------------------------------------

struct StreamPlan {
  uint32_t vectors;         // of a pixel; the last one ends where the pixel does, and may overlap
                            // the one before (what both have is computed and written twice)
  uint32_t tiles, columns;  // tiles of channels, vectors of a tile
  uint32_t threads_rows;    // pixels that a workgroup takes at once
  uint32_t chunks;          // of a sample's pixels: every chunks-th run of threads_rows
  uint32_t at_once;         // samples of a launch's grid
};

// The partial values of a sample, as the launch that left them cut its pixels.
struct Parts {
  uint32_t chunks, rows;
  bool joined;  // by the workgroups that read them
};

// A workgroup's part: a chunk of the pixels (the grid's x) by a tile of channels (its y), of every
// sample that its z comes to.
struct Item {
  uint64_t first;        // this thread's first pixel
  uint32_t step;         // to its next
  uint32_t column;       // this thread's first channel
  uint32_t tile;         // the tile's first channel, and its number of channels
  uint32_t wide;
  uint32_t row;
  bool live;
  uint32_t last, overlap;  // the last vector's first channel without overlap, and its overlap
  // Where channel c of the tile is in a row of the tile's vectors.
  __device__ __forceinline__ uint32_t place(uint32_t c) const {
    return tile + c >= last ? c + overlap : c;
  }
};

template <int V>
__device__ __forceinline__ Item item_of(const GnCall& k, const StreamPlan& plan) {
  Item it;
  it.row = threadIdx.x / plan.columns;
  it.first = (uint64_t)blockIdx.x * plan.threads_rows + it.row;
  it.step = plan.chunks * plan.threads_rows;
  const uint32_t vector = blockIdx.y * plan.columns + threadIdx.x - it.row * plan.columns;
  it.column = min(vector * V, k.width - V);
  it.tile = blockIdx.y * plan.columns * V;
  it.wide = min(plan.columns * V, k.width - it.tile);
  it.live = it.row < plan.threads_rows && vector < plan.vectors;
  it.last = (plan.vectors - 1) * V;
  it.overlap = it.last - (k.width - V);
  return it;
}

// Pixels of `pixels` from `first` on in steps of `step`.
__device__ __forceinline__ uint32_t count_from(uint64_t first, uint64_t pixels, uint32_t step) {
  return first < pixels ? (uint32_t)((pixels - first + step - 1) / step) : 0;
}

// For every `step`th pixel from p on: U loads on their way before the first is used; past the
// end the last pixel's, unused (so that the rest of a chunk is not loaded one by one).
template <typename T, int V, int U, typename L, typename F>
__device__ __forceinline__ void for_pixels(uint64_t p, uint64_t last, uint32_t step, L&& load,
                                           F&& use) {
  for (; p < last; p += U * (uint64_t)step) {
    Run<T, V> run[U];
#pragma unroll
    for (int u = 0; u < U; ++u) load(min(p + u * (uint64_t)step, last - 1), run[u]);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (p + u * (uint64_t)step < last) use(p + u * (uint64_t)step, run[u]);
  }
}

// The same over pairs of runs.
template <typename T, int V, int U, typename L, typename F>
__device__ __forceinline__ void for_pixel_pairs(uint64_t p, uint64_t last, uint32_t step, L&& load,
                                                F&& use) {
  for (; p < last; p += U * (uint64_t)step) {
    Run<T, V> a[U], b[U];
#pragma unroll
    for (int u = 0; u < U; ++u) load(min(p + u * (uint64_t)step, last - 1), a[u], b[u]);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (p + u * (uint64_t)step < last) use(p + u * (uint64_t)step, a[u], b[u]);
  }
}

// f(r, c) over the rows of a tile's channels in LDS, c in 0..it.wide - 1: `parts` threads of a
// channel take a share of the rows each.
struct TileRows {
  uint32_t c, part, parts;
  bool live;
  __device__ __forceinline__ TileRows(const Item& it, uint32_t rows) {
    parts = min(max(256u / it.wide, 1u), rows);
    part = threadIdx.x / it.wide;
    c = threadIdx.x - part * it.wide;
    live = part < parts;
  }
};

// Each channel's mean and sum of squared differences over a chunk of pixels.
template <typename T, int V>
__global__ void __launch_bounds__(256) group_norm_stats_kernel(GnCall k, StreamPlan plan,
                                                               float2* __restrict__ partial) {
  __shared__ float2 s[256 * V];
  __shared__ float2 s_part[256];
  const Item it = item_of<V>(k, plan);
  const uint32_t rows = plan.threads_rows;
  const uint64_t run = (uint64_t)blockIdx.x * rows;  // the chunk's first pixel
  // Rows have one pixel more than the last one has, or as many, those with more first.
  const uint32_t count = count_from(it.first, k.pixels, it.step);
  const uint32_t least = count_from(run + rows - 1, k.pixels, it.step);
  const uint32_t longer = count_from(run, k.pixels, it.step) > least
                              ? (uint32_t)((k.pixels - run) % it.step) : 0;
  const float inv = count ? 1.f / (float)count : 0.f;
  const float all = 1.f / (float)((uint64_t)least * rows + longer);
  for (uint64_t n = blockIdx.z; n < k.samples; n += gridDim.z) {
    float pivot[V] = {}, sum[V] = {}, squares[V] = {};
    if (it.live && count) {
      const T* x = (const T*)k.x + (int64_t)n * k.x_sample + it.column;
      bool begun = false;
      for_pixels<T, V, 8>(it.first, k.pixels, it.step, [&](uint64_t p, Run<T, V>& r) {
        r.load(x + (int64_t)p * k.x_pitch);
      }, [&](uint64_t, const Run<T, V>& r) {
        if (!begun) {
#pragma unroll
          for (int v = 0; v < V; ++v) pivot[v] = to_f32(r.v[v]);
          begun = true;
        }
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float d = to_f32(r.v[v]) - pivot[v];
          sum[v] += d;
          squares[v] = fmaf(d, d, squares[v]);
        }
      });
    }
    __syncthreads();  // (the last sample's values are read)
    if (it.row < rows) {
#pragma unroll
      for (int v = 0; v < V; ++v)
        s[threadIdx.x * V + v] = {fmaf(sum[v], inv, pivot[v]),
                                  fmaxf(fmaf(-sum[v] * inv, sum[v], squares[v]), 0.f)};
    }
    __syncthreads();
    // rows joined from the first row's mean, near to which the others' are
    const uint32_t pitch = plan.columns * V;
    for (uint32_t c0 = 0; c0 < it.wide; c0 += 256) {
      const TileRows t(it, rows);
      const uint32_t c = it.wide > 256 ? c0 + threadIdx.x : t.c;
      const bool live = it.wide > 256 ? c < it.wide : t.live;
      float2 a = {0.f, 0.f};
      const uint32_t place = it.place(c);
      const float near = live ? s[place].x : 0.f;
      if (live)
        for (uint32_t r = t.part; r < rows; r += t.parts) {
          const float m = (float)(least + (r < longer));
          if (m == 0.f) break;
          const float2 p = s[r * pitch + place];
          const float d = p.x - near;
          a.x = fmaf(m, d, a.x);
          a.y += fmaf(m * d, d, p.y);
        }
      if (t.parts > 1) {
        s_part[threadIdx.x] = a;
        __syncthreads();
        if (threadIdx.x < it.wide)
          for (uint32_t j = 1; j < t.parts; ++j) {
            const float2 p = s_part[threadIdx.x + j * it.wide];
            a.x += p.x, a.y += p.y;
          }
      }
      if (live && t.part == 0)
        partial[(n * plan.chunks + blockIdx.x) * k.width + it.tile + c] = {
            fmaf(a.x, all, near), fmaxf(fmaf(-a.x * all, a.x, a.y), 0.f)};
    }
  }
}

// Pixels of a chunk.
__device__ __forceinline__ float chunk_pixels(const GnCall& k, const Parts& parts, uint32_t q) {
  const uint64_t round = (uint64_t)parts.chunks * parts.rows, before = (uint64_t)q * parts.rows;
  const uint64_t rest = k.pixels % round;
  const uint64_t more = rest > before ? min(rest - before, (uint64_t)parts.rows) : 0;
  return (float)(k.pixels / round * parts.rows + more);
}

template <int WAVES>
__device__ __forceinline__ double sum_of_workgroup(double v, double* s) {
#pragma unroll
  for (int off = 32; off; off >>= 1) v += __shfl_xor(v, off, 64);
  __syncthreads();
  if (threadIdx.x % 64 == 0) s[threadIdx.x / 64] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) v += s[w];
  return v;
}

// f(chunk, channel) over a group's partial values: as many threads side by side as there are
// channels, up to 64, the others on further chunks.
template <typename F>
__device__ __forceinline__ void for_entries(const Parts& parts, uint32_t each, F&& f) {
  const uint32_t across = each < 64 ? each : 64, along = blockDim.x / across;
  const uint32_t c0 = threadIdx.x % across, q0 = threadIdx.x / across;
  if (q0 >= along) return;
  for (uint32_t c = c0; c < each; c += across) {
#pragma unroll 4
    for (uint32_t q = q0; q < parts.chunks; q += along) f(q, c);
  }
}

// sum(g) / m and sum(g xhat) / m of each sample's group, a workgroup each.
template <typename T>
__global__ void __launch_bounds__(1024) group_norm_group_sums_kernel(
    GnCall k, Parts parts, const float2* __restrict__ partial, float2* __restrict__ sums) {
  __shared__ double s[16];
  for (uint64_t i = blockIdx.x; i < k.samples * k.groups; i += gridDim.x) {
    const uint64_t n = i / k.groups;
    const uint32_t c0 = (uint32_t)(i % k.groups) * k.each;
    const float2* from = partial + n * parts.chunks * k.width + c0;
    const double m = (double)k.pixels * k.each;
    double a = 0, b = 0;
    for_entries(parts, k.each, [&](uint32_t j, uint32_t c) {
      const float2 p = from[(uint64_t)j * k.width + c];
      const float w = column<T>(k.weight, k.wide_weights, c0 + c, 1.f);
      a += (double)w * p.x;
      b += (double)w * p.y;
    });
    a = sum_of_workgroup<16>(a, s) / m;
    b = sum_of_workgroup<16>(b, s) / m;
    if (threadIdx.x == 0) sums[i] = {(float)a, (float)b};
  }
}

// The same two joins by a workgroup of 256 for itself, all groups of a sample at once (their
// channels are one tile): threads by channel over the chunks, then by channel over its group.
// s: 2 floats for each of 256 threads or of the channels, whichever are more.

// The sums of entry(q, c) over the chunks q, each channel's in s[c].
template <typename F>
__device__ __forceinline__ void sum_by_channel(const GnCall& k, const Parts& parts, float2* s,
                                               F&& entry) {
  const uint32_t along = k.width < 256 ? 256 / k.width : 1;  // threads of a channel
  __syncthreads();
  for (uint32_t t = threadIdx.x; t < along * k.width; t += 256) {
    const uint32_t c = t % k.width;
    float2 a = {0.f, 0.f};
#pragma unroll 16
    for (uint32_t q = t / k.width; q < parts.chunks; q += along) {
      const float2 p = entry(q, c);
      a.x += p.x, a.y += p.y;
    }
    s[t] = a;
  }
  __syncthreads();
  if (along > 1) {
    float2 a = {0.f, 0.f};
    if (threadIdx.x < k.width)
      for (uint32_t j = 0; j < along; ++j) {
        const float2 p = s[j * k.width + threadIdx.x];
        a.x += p.x, a.y += p.y;
      }
    __syncthreads();
    if (threadIdx.x < k.width) s[threadIdx.x] = a;
    __syncthreads();
  }
}

// s[group] = f(group), for the at most two groups of a thread; f reads s.
template <typename F>
__device__ __forceinline__ void replace_by_group(const GnCall& k, float2* s, F&& f) {
  float2 a[2];
#pragma unroll
  for (int j = 0; j < 2; ++j)
    if (threadIdx.x + 256 * j < k.groups) a[j] = f(threadIdx.x + 256 * j);
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 2; ++j)
    if (threadIdx.x + 256 * j < k.groups) s[threadIdx.x + 256 * j] = a[j];
  __syncthreads();
}

// s[group] = {mean, rstd}
__device__ __forceinline__ void join_stats(const GnCall& k, const Parts& parts,
                                           const float2* partial, uint64_t n, float2* s) {
  const float2* from = partial + n * parts.chunks * k.width;
  const float pixels = (float)k.pixels, inv = 1.f / pixels;
  // differences from the first chunk's mean, near to which the others' are
  sum_by_channel(k, parts, s, [&](uint32_t q, uint32_t c) {
    const float2 p = from[q * k.width + c];
    const float d = p.x - from[c].x, nd = chunk_pixels(k, parts, q) * d;
    return make_float2(nd, fmaf(nd, d, p.y));
  });
  for (uint32_t c = threadIdx.x; c < k.width; c += 256) {
    const float2 a = s[c];
    s[c] = {fmaf(a.x, inv, from[c].x), fmaxf(fmaf(-a.x * inv, a.x, a.y), 0.f)};
  }
  __syncthreads();
  replace_by_group(k, s, [&](uint32_t g) {
    const float2* channel = s + g * k.each;
    float mean = 0.f, m2 = 0.f;
    for (uint32_t j = 0; j < k.each; ++j) mean += channel[j].x;
    mean /= (float)k.each;
    for (uint32_t j = 0; j < k.each; ++j) {
      const float d = channel[j].x - mean;
      m2 += fmaf(pixels * d, d, channel[j].y);
    }
    return make_float2(mean, 1.f / sqrtf(fmaf(m2, inv / (float)k.each, k.eps)));
  });
}

// s[group] = {sum(g) / m, sum(g xhat) / m}
template <typename T>
__device__ __forceinline__ void join_sums(const GnCall& k, const Parts& parts,
                                          const float2* partial, uint64_t n, float2* s) {
  const float2* from = partial + n * parts.chunks * k.width;
  const float inv = 1.f / (float)(k.pixels * k.each);
  sum_by_channel(k, parts, s, [&](uint32_t q, uint32_t c) {
    const float w = column<T>(k.weight, k.wide_weights, c, 1.f);
    const float2 p = from[q * k.width + c];
    return make_float2(w * p.x, w * p.y);
  });
  replace_by_group(k, s, [&](uint32_t g) {
    float2 a = {0.f, 0.f};
    for (uint32_t j = 0; j < k.each; ++j) {
      const float2 p = s[g * k.each + j];
      a.x += p.x, a.y += p.y;
    }
    return make_float2(a.x * inv, a.y * inv);
  });
}

// What a thread needs of its channels, z = (x - mean) w rstd + b; `stats` of this sample's groups.
template <typename T, int V>
struct Columns {
  float mean[V], rstd[V], factor[V], b[V];
  __device__ __forceinline__ void load(const GnCall& k, const Item& it, const float2* stats) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const uint32_t c = it.column + v;
      const float2 st = stats[c / k.each];
      mean[v] = st.x, rstd[v] = st.y;
      factor[v] = column<T>(k.weight, k.wide_weights, c, 1.f) * rstd[v];
      b[v] = column<T>(k.bias, k.wide_weights, c, 0.f);
    }
  }
};

// JOINED: mean and rstd are joined here, and kept by the workgroup of a sample's first chunk.
template <typename T, int V, bool JOINED>
__global__ void __launch_bounds__(256) group_norm_apply_kernel(GnCall k, StreamPlan plan,
                                                               Parts parts,
                                                               const float2* __restrict__ partial) {
  __shared__ float2 s[JOINED ? JOINED_WIDTH : 1];
  const Item it = item_of<V>(k, plan);
  for (uint64_t m = blockIdx.z; m < k.samples; m += gridDim.z) {
    const uint64_t n = k.samples - 1 - m;
    const float2* stats = k.stats + n * k.groups;
    if constexpr (JOINED) {
      join_stats(k, parts, partial, n, s);
      if (blockIdx.x == 0)
        for (uint32_t g = threadIdx.x; g < k.groups; g += 256) k.stats[n * k.groups + g] = s[g];
      stats = s;
    }
    if (!it.live) continue;
    Columns<T, V> col;
    col.load(k, it, stats);
    const int64_t end = (int64_t)k.pixels - 1;
    const T* x = (const T*)k.x + (int64_t)n * k.x_sample + end * k.x_pitch + it.column;
    T* y = (T*)k.y + (n * k.pixels + end) * k.width + it.column;
    with_act(k.act, [&](auto act) {
      for_pixels<T, V, 4>(it.first, k.pixels, it.step,
                          [&](uint64_t p, Run<T, V>& r) { r.load(x - (int64_t)p * k.x_pitch); },
                          [&](uint64_t p, const Run<T, V>& r) {
        Run<T, V> out;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float d = to_f32(r.v[v]) - col.mean[v];
          out.v[v] = from_f32<T>(act_value<act.value, T>(fmaf(d, col.factor[v], col.b[v])));
        }
        store(k, out, y - p * k.width);
      });
    });
  }
}

// Each channel's sums of dz and dz xhat over a chunk of pixels.
template <typename T, int V>
__global__ void __launch_bounds__(256) group_norm_sums_kernel(GnCall k, StreamPlan plan,
                                                              float2* __restrict__ partial) {
  __shared__ float2 s[256 * V];
  __shared__ float2 s_part[256];
  const Item it = item_of<V>(k, plan);
  for (uint64_t n = blockIdx.z; n < k.samples; n += gridDim.z) {
    float db[V] = {}, dw[V] = {};  // (dw of x - mean, times rstd at the end)
    Columns<T, V> col;
    if (it.live) {
      col.load(k, it, k.stats + n * k.groups);
      const T* x = (const T*)k.x + (int64_t)n * k.x_sample + it.column;
      const T* dy = (const T*)k.dy + (int64_t)n * k.dy_sample + it.column;
      with_act(k.act, [&](auto act) {
        for_pixel_pairs<T, V, 2>(it.first, k.pixels, it.step,
                                 [&](uint64_t p, Run<T, V>& r, Run<T, V>& g) {
          r.load(x + (int64_t)p * k.x_pitch);
          g.load(dy + (int64_t)p * k.dy_pitch);
        }, [&](uint64_t, const Run<T, V>& r, const Run<T, V>& g) {
#pragma unroll
          for (int v = 0; v < V; ++v) {
            const float d = to_f32(r.v[v]) - col.mean[v];
            const float dz =
                to_f32(g.v[v]) * act_slope<act.value, T>(fmaf(d, col.factor[v], col.b[v]));
            db[v] += dz;
            dw[v] = fmaf(dz, d, dw[v]);
          }
        });
      });
    }
    __syncthreads();
    if (it.row < plan.threads_rows) {
#pragma unroll
      for (int v = 0; v < V; ++v)
        s[threadIdx.x * V + v] = {db[v], it.live ? dw[v] * col.rstd[v] : 0.f};
    }
    __syncthreads();
    const uint32_t pitch = plan.columns * V;
    for (uint32_t c0 = 0; c0 < it.wide; c0 += 256) {
      const TileRows t(it, plan.threads_rows);
      const uint32_t c = it.wide > 256 ? c0 + threadIdx.x : t.c;
      const bool live = it.wide > 256 ? c < it.wide : t.live;
      float2 a = {0.f, 0.f};
      if (live)
        for (uint32_t r = t.part; r < plan.threads_rows; r += t.parts) {
          const float2 p = s[r * pitch + it.place(c)];
          a.x += p.x, a.y += p.y;
        }
      if (t.parts > 1) {
        s_part[threadIdx.x] = a;
        __syncthreads();
        if (threadIdx.x < it.wide)
          for (uint32_t j = 1; j < t.parts; ++j) {
            const float2 p = s_part[threadIdx.x + j * it.wide];
            a.x += p.x, a.y += p.y;
          }
      }
      if (live && t.part == 0)
        partial[(n * plan.chunks + blockIdx.x) * k.width + it.tile + c] = a;
    }
  }
}

// from: the groups' sums, or (JOINED) the partial ones.
template <typename T, int V, bool JOINED>
__global__ void __launch_bounds__(256) group_norm_dx_kernel(GnCall k, StreamPlan plan,
                                                            Parts parts,
                                                            const float2* __restrict__ from) {
  __shared__ float2 s[JOINED ? JOINED_WIDTH : 1];
  const Item it = item_of<V>(k, plan);
  for (uint64_t m = blockIdx.z; m < k.samples; m += gridDim.z) {
    const uint64_t n = k.samples - 1 - m;
    const float2* sums = from + n * k.groups;
    if constexpr (JOINED) {
      join_sums<T>(k, parts, from, n, s);
      sums = s;
    }
    if (!it.live) continue;
    Columns<T, V> col;
    col.load(k, it, k.stats + n * k.groups);
    // dx = factor dz - s1 - xhat s2 (rstd twice in s2 would leave float32 for large spreads)
    float s1[V], s2[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float2 p = sums[(it.column + v) / k.each];
      s1[v] = p.x * col.rstd[v], s2[v] = p.y * col.rstd[v];
    }
    const int64_t end = (int64_t)k.pixels - 1;
    const T* x = (const T*)k.x + (int64_t)n * k.x_sample + end * k.x_pitch + it.column;
    const T* dy = (const T*)k.dy + (int64_t)n * k.dy_sample + end * k.dy_pitch + it.column;
    T* dx = (T*)k.y + (n * k.pixels + end) * k.width + it.column;
    with_act(k.act, [&](auto act) {
      for_pixel_pairs<T, V, 2>(it.first, k.pixels, it.step,
                               [&](uint64_t p, Run<T, V>& r, Run<T, V>& g) {
        r.load(x - (int64_t)p * k.x_pitch);
        g.load(dy - (int64_t)p * k.dy_pitch);
      }, [&](uint64_t p, const Run<T, V>& r, const Run<T, V>& g) {
        Run<T, V> out;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float d = to_f32(r.v[v]) - col.mean[v];
          const float dz =
              to_f32(g.v[v]) * act_slope<act.value, T>(fmaf(d, col.factor[v], col.b[v]));
          out.v[v] = from_f32<T>(fmaf(-d * col.rstd[v], s2[v], fmaf(dz, col.factor[v], -s1[v])));
        }
        out.store(dx - p * k.width);
      });
    });
  }
}

// ---------------------------------------------------------------------------
// Launches
// ---------------------------------------------------------------------------

// The plans of the four streaming launches.
struct StreamPlans {
  uint32_t v;
  bool joined;
  StreamPlan stats, apply, sums, dx;
  Parts parts_of(const StreamPlan& plan) const { return {plan.chunks, plan.threads_rows, joined}; }
  // Whether a launch's partial values are joined by channel first: a group has too many of them
  // for one workgroup.
  bool by_channel(const StreamPlan& plan, uint32_t each) const {
    return !joined && (uint64_t)plan.chunks * each > JOINED_ENTRIES;
  }
};

static inline dim3 grid_of(const StreamPlan& plan) {
  return dim3(plan.chunks, plan.tiles, plan.at_once);
}

static inline uint32_t capped(uint64_t n) { return (uint32_t)std::min<uint64_t>(n, 1u << 20); }

// Mean and rstd of each sample's group from the partial values; partial values joined over the
// chunks (group_norm.hip).
void gn_finish(const GnCall& k, const Parts& parts, const float2* partial, hipStream_t stream);
Parts gn_channels(const GnCall& k, const Parts& parts, bool stats, const float2* partial,
                  float2* out, hipStream_t stream);

// Rows of db and dw by channel, whose sum is the weights' gradients.
struct SumRows {
  const float2* first;
  uint32_t count;
};

// By type, in a translation unit each (group_norm_f32.hip and its like).
template <typename T>
void gn_held(const GnCall& k, const HeldPlan& plan, bool backward, float* partial,
             hipStream_t stream);
template <typename T>
void gn_streamed_fwd(const GnCall& k, const StreamPlans& plans, float2* partial,
                     hipStream_t stream);
// (k.y null: no dx)
template <typename T>
SumRows gn_streamed_bwd(const GnCall& k, const StreamPlans& plans, float2* workspace,
                        hipStream_t stream);

#ifdef GN_TYPE

// Calls f with the values of a run as a constant.
template <typename T, typename F>
static void with_run(uint32_t v, F&& f) {
  constexpr int WIDEST = 16 / sizeof(T);
  if (v == 1)
    f(std::integral_constant<int, 1>());
  else if (v == 4 || WIDEST == 4)
    f(std::integral_constant<int, 4>());
  else
    f(std::integral_constant<int, WIDEST>());
}

template <typename T, int V, int E, bool BACKWARD>
static void held_launch(const GnCall& k, const HeldPlan& plan, float* partial,
                        hipStream_t stream) {
  const auto start = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(plan.grid), dim3(256), 0, stream, k, plan, partial);
  };
  const auto tail = [&](auto wide) {
    if constexpr (V > 1)  // (single values have no tail)
      if (plan.tail) return start(group_norm_held_kernel<T, V, E, BACKWARD, wide.value, true>);
    start(group_norm_held_kernel<T, V, E, BACKWARD, wide.value, false>);
  };
  if (plan.wide)
    tail(std::true_type());
  else if constexpr (E <= HELD_FEW)
    tail(std::false_type());
}

template <typename T>
void gn_held(const GnCall& k, const HeldPlan& plan, bool backward, float* partial,
             hipStream_t stream) {
  with_run<T>(plan.v, [&](auto v) {
    const auto runs = [&](auto e) {
      if (backward)
        held_launch<T, v.value, e.value, true>(k, plan, partial, stream);
      else
        held_launch<T, v.value, e.value, false>(k, plan, partial, stream);
    };
    if (plan.runs == 1)
      runs(std::integral_constant<int, 1>());
    else if (plan.runs == 2)
      runs(std::integral_constant<int, 2>());
    else if (plan.runs <= 4)
      runs(std::integral_constant<int, 4>());
    else
      runs(std::integral_constant<int, 8>());
  });
}

template <typename T>
void gn_streamed_fwd(const GnCall& k, const StreamPlans& plans, float2* partial,
                     hipStream_t stream) {
  const Parts parts = plans.parts_of(plans.stats);
  with_run<T>(plans.v, [&](auto v) {
    hipLaunchKernelGGL((group_norm_stats_kernel<T, v.value>), grid_of(plans.stats), dim3(256), 0,
                       stream, k, plans.stats, partial);
    if (plans.by_channel(plans.stats, k.each)) {
      float2* channels = partial + k.samples * parts.chunks * k.width;
      gn_finish(k, gn_channels(k, parts, true, partial, channels, stream), channels, stream);
    } else if (!parts.joined) {
      gn_finish(k, parts, partial, stream);
    }
    const auto apply = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, grid_of(plans.apply), dim3(256), 0, stream, k, plans.apply, parts,
                         partial);
    };
    if (parts.joined)
      apply(group_norm_apply_kernel<T, v.value, true>);
    else
      apply(group_norm_apply_kernel<T, v.value, false>);
  });
}

template <typename T>
SumRows gn_streamed_bwd(const GnCall& k, const StreamPlans& plans, float2* workspace,
                        hipStream_t stream) {
  Parts parts = plans.parts_of(plans.sums);
  float2* partial = workspace;
  with_run<T>(plans.v, [&](auto v) {
    hipLaunchKernelGGL((group_norm_sums_kernel<T, v.value>), grid_of(plans.sums), dim3(256), 0,
                       stream, k, plans.sums, partial);
    if (plans.by_channel(plans.sums, k.each)) {
      float2* channels = partial + k.samples * parts.chunks * k.width;
      parts = gn_channels(k, parts, false, partial, channels, stream);
      partial = channels;
    }
    if (!k.y) return;
    float2* group_sums = partial + k.samples * parts.chunks * k.width;
    if (!parts.joined)
      hipLaunchKernelGGL(group_norm_group_sums_kernel<T>, dim3(capped(k.samples * k.groups)),
                         dim3(1024), 0, stream, k, parts, partial, group_sums);
    const auto launch = [&](auto kernel, const float2* from) {
      hipLaunchKernelGGL(kernel, grid_of(plans.dx), dim3(256), 0, stream, k, plans.dx, parts,
                         from);
    };
    if (parts.joined)
      launch(group_norm_dx_kernel<T, v.value, true>, partial);
    else
      launch(group_norm_dx_kernel<T, v.value, false>, group_sums);
  });
  return {partial, (uint32_t)(k.samples * parts.chunks)};
}

template void gn_held<GN_TYPE>(const GnCall&, const HeldPlan&, bool, float*, hipStream_t);
template void gn_streamed_fwd<GN_TYPE>(const GnCall&, const StreamPlans&, float2*, hipStream_t);
template SumRows gn_streamed_bwd<GN_TYPE>(const GnCall&, const StreamPlans&, float2*,
                                          hipStream_t);
#endif
