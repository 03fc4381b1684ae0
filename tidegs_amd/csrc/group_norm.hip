// Group norm: the kernels that go by no type of x, the plans and the entry points
// (group_norm.cuh has the mathematics and the other kernels).
#include "group_norm.cuh"

// db and dw, which alternate in the partial rows: the rows' sums, 8 values by 128 interleaved
// runs of rows a workgroup.
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
    W* out = c % 2 ? dweight : dbias;
    if (out) out[c / 2] = from_f32<W>(s[threadIdx.x]);
  }
}

// Each channel's partial values joined over the chunks, 64 channels by 16 runs of chunks a
// workgroup: for groups of many channels, whose values one workgroup would read for long (one
// group of 862 channels of 36471 pixels: 231 us the forward, 104 with this launch).
// STATS: means and sums of squared differences, otherwise sums.
template <bool STATS>
__global__ void __launch_bounds__(1024) group_norm_channels_kernel(
    GnCall k, Parts parts, const float2* __restrict__ partial, float2* __restrict__ out) {
  __shared__ float2 s[1024];
  const uint32_t c = blockIdx.x * 64 + threadIdx.x % 64;
  const bool live = c < k.width;
  for (uint64_t n = blockIdx.y; n < k.samples; n += gridDim.y) {
    const float2* from = partial + n * parts.chunks * k.width;
    float2 a = {0.f, 0.f};
    const float near = STATS && live ? from[c].x : 0.f;
    if (live) {
#pragma unroll 8
      for (uint32_t q = threadIdx.x / 64; q < parts.chunks; q += 16) {
        const float2 p = from[(uint64_t)q * k.width + c];
        if constexpr (STATS) {
          const float d = p.x - near, nd = chunk_pixels(k, parts, q) * d;
          a.x += nd, a.y += fmaf(nd, d, p.y);
        } else {
          a.x += p.x, a.y += p.y;
        }
      }
    }
    s[threadIdx.x] = a;
    for (uint32_t h = 512; h >= 64; h >>= 1) {
      __syncthreads();
      if (threadIdx.x < h) {
        s[threadIdx.x].x += s[threadIdx.x + h].x;
        s[threadIdx.x].y += s[threadIdx.x + h].y;
      }
    }
    if (threadIdx.x < 64 && live) {
      a = s[threadIdx.x];
      if constexpr (STATS) {
        const float mean = a.x / (float)k.pixels;
        a = {near + mean, fmaxf(fmaf(-mean, a.x, a.y), 0.f)};
      }
      out[n * k.width + c] = a;
    }
    __syncthreads();
  }
}

// Mean and rstd of each sample's group, a workgroup each: sums of 64 bits of differences from
// the group's first partial mean.
__global__ void __launch_bounds__(1024) group_norm_finish_kernel(
    GnCall k, Parts parts, const float2* __restrict__ partial) {
  __shared__ double s[16];
  for (uint64_t i = blockIdx.x; i < k.samples * k.groups; i += gridDim.x) {
    const uint64_t n = i / k.groups;
    const float2* from = partial + n * parts.chunks * k.width + i % k.groups * k.each;
    const double m = (double)k.pixels * k.each, near = from[0].x;
    double a = 0, q = 0;
    for_entries(parts, k.each, [&](uint32_t j, uint32_t c) {
      const float2 p = from[(uint64_t)j * k.width + c];
      const double d = p.x - near, nd = chunk_pixels(k, parts, j) * d;
      a += nd;
      q += p.y + nd * d;
    });
    a = sum_of_workgroup<16>(a, s) / m;
    q = sum_of_workgroup<16>(q, s) / m;
    if (threadIdx.x == 0)
      k.stats[i] = {(float)(near + a),
                    (float)(1.0 / sqrt(fmax(q - a * a, 0.0) + (double)k.eps))};
  }
}

Parts gn_channels(const GnCall& k, const Parts& parts, bool stats, const float2* partial,
                  float2* out, hipStream_t stream) {
  const dim3 grid((k.width + 63) / 64, (unsigned)std::min<uint64_t>(k.samples, 1024));
  if (stats)
    hipLaunchKernelGGL(group_norm_channels_kernel<true>, grid, dim3(1024), 0, stream, k, parts,
                       partial, out);
  else
    hipLaunchKernelGGL(group_norm_channels_kernel<false>, grid, dim3(1024), 0, stream, k, parts,
                       partial, out);
  return {1, parts.rows, false};
}

void gn_finish(const GnCall& k, const Parts& parts, const float2* partial, hipStream_t stream) {
  hipLaunchKernelGGL(group_norm_finish_kernel, dim3(capped(k.samples * k.groups)), dim3(1024), 0,
                     stream, k, parts, partial);
}

static int log2_up(uint64_t n) {
  int k = 0;
  while ((1ull << k) < n) ++k;
  return k;
}

static uint32_t size_of(int32_t dtype) { return dtype == TGS_F32 ? 4 : 2; }

// Values of a run: the most of 16 bytes and four values that n is a whole number of, or else
// the most that n has at least (the last run overlaps), or one.  (With runs of single values
// for what is no multiple, 2 x 250000 x 59 bfloat16 took 68 us in place of 52, the forward, and
// 20000 rows of 777 in one group, which no team held then, 1069 in place of 30.)
static uint32_t vector_of(uint32_t n, int32_t dtype) {
  const uint32_t widest = 16 / size_of(dtype);
  for (uint32_t v = widest; v >= 4; v /= 2)
    if (n % v == 0) return v;
  for (uint32_t v = widest; v >= 4; v /= 2)
    if (n > v) return v;
  return 1;
}

static bool held_plan(uint64_t samples, uint64_t pixels, uint32_t groups, uint32_t each,
                      uint32_t v, HeldPlan& plan) {
  plan.v = v;
  plan.tail = each % v != 0;
  plan.lane_log = log2_up((each + v - 1) / v);
  plan.wide = false;
  if (plan.lane_log > 8 || pixels > 256 * HELD_RUNS) return false;
  const int rows = log2_up(pixels);
  if (plan.lane_log > 6 || pixels > HELD_FEW * (64u >> plan.lane_log)) {
    plan.wide = true;  // (the rows fill the workgroup: idle ones cost nothing)
    plan.row_log = 8 - plan.lane_log;
    plan.runs = (int)((pixels + (1u << plan.row_log) - 1) >> plan.row_log);
    if (plan.runs > HELD_RUNS) return false;
    plan.teams = 1;
    plan.rows = (uint32_t)std::min<uint64_t>(samples, std::max<uint32_t>(1, 2048 / groups));
    plan.grid = plan.rows * groups;
    plan.partials = plan.rows;
    return true;
  }
  plan.row_log = std::min(6 - plan.lane_log, rows);
  plan.runs = (int)((pixels + (1u << plan.row_log) - 1) >> plan.row_log);
  const uint32_t teams = 256 >> (plan.lane_log + plan.row_log);
  if (teams >= groups) {
    const uint32_t each_wg = teams / groups;  // samples of a workgroup at once
    plan.teams = each_wg * groups;
    plan.grid = (uint32_t)std::min<uint64_t>((samples + each_wg - 1) / each_wg, 1280);
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

// About `workgroups` of them, each with 8 pixels a thread at least; `most` chunks of a sample.
static StreamPlan stream_plan(uint64_t samples, uint64_t pixels, uint32_t width, uint32_t v,
                              uint64_t workgroups, uint64_t most) {
  StreamPlan plan;
  plan.vectors = (width + v - 1) / v;
  plan.tiles = (plan.vectors + TILE_VECTORS - 1) / TILE_VECTORS;
  plan.columns = (plan.vectors + plan.tiles - 1) / plan.tiles;
  plan.threads_rows = 256 / plan.columns;
  const uint64_t others = std::max<uint64_t>(1, samples * plan.tiles);
  const uint64_t wanted = std::min(std::max<uint64_t>(1, workgroups / others), most);
  plan.chunks = (uint32_t)std::min(wanted, (pixels + 8 * plan.threads_rows - 1) /
                                               (8 * plan.threads_rows));
  plan.at_once = (uint32_t)std::min<uint64_t>(
      samples,
      std::max<uint64_t>(1, std::min<uint64_t>(65535, (1u << 23) / (plan.tiles * plan.chunks))));
  return plan;
}

static StreamPlans stream_plans(uint64_t samples, uint64_t pixels, uint32_t width, uint32_t groups,
                                int32_t dtype) {
  StreamPlans p;
  p.v = vector_of(width, dtype);
  const auto plan = [&](uint64_t workgroups, uint64_t most) {
    return stream_plan(samples, pixels, width, p.v, workgroups, most);
  };
  // (4 x 960x540x64 bfloat16, 1024 and 2048 workgroups: stats 59 and 70 us, sums 156 and 141, dx 187
  // and 166)
  constexpr uint64_t ANY = 1ull << 30;
  p.stats = plan(1024, ANY);
  p.apply = plan(2048, ANY);
  p.sums = plan(2048, ANY);
  p.dx = plan(2048, ANY);
  // Few partial values are joined by each workgroup that reads them, a launch less, if enough
  // workgroups are left where chunks are made fewer for it.
  const uint64_t most = std::max<uint64_t>(1, JOINED_ENTRIES / width);
  p.joined = width <= p.v * TILE_VECTORS && width <= JOINED_WIDTH &&
             width / groups <= JOINED_EACH && samples * pixels * width < JOINED_BELOW &&
             (p.stats.chunks <= most || samples * most >= JOINED_WORKGROUPS);
  if (p.joined) {
    p.stats = plan(1024, most);
    p.sums = plan(2048, most);
  }
  return p;
}

static bool gn_sizes_ok(uint64_t samples, uint64_t pixels, uint32_t width, uint32_t groups,
                        int32_t dtype) {
  return width > 0 && width <= 65536 && groups > 0 && width % groups == 0 &&
         dtype >= TGS_F32 && dtype <= TGS_F16 && samples < (1ull << 40) && pixels < (1ull << 40);
}

static bool gn_held(uint64_t samples, uint64_t pixels, uint32_t width, uint32_t groups,
                    int32_t dtype, HeldPlan& plan) {
  const uint32_t each = width / groups, v = vector_of(each, dtype);
  return held_plan(samples, pixels, groups, each, v, plan) ||
         // (fewer lanes, where runs of four values take too many)
         (v == 4 && each > 8 && dtype != TGS_F32 &&
          held_plan(samples, pixels, groups, each, 8, plan));
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
  const StreamPlans plans = stream_plans(samples, pixels, width, groups, dtype);
  const uint64_t rows =
      (uint64_t)plans.stats.chunks + (plans.by_channel(plans.stats, width / groups) ? 1 : 0);
  return samples * rows * width * sizeof(float2);
}

extern "C" uint64_t tgs_group_norm_bwd_workspace_size(uint64_t samples, uint64_t pixels,
                                                      uint32_t width, uint32_t groups,
                                                      int32_t dtype) {
  HeldPlan held;
  if (!gn_sizes_ok(samples, pixels, width, groups, dtype) || samples == 0 || pixels == 0) return 0;
  if (gn_held(samples, pixels, width, groups, dtype, held))
    return (uint64_t)held.partials * 2 * width * sizeof(float);
  const StreamPlans plans = stream_plans(samples, pixels, width, groups, dtype);
  const uint64_t rows =
      (uint64_t)plans.sums.chunks + (plans.by_channel(plans.sums, width / groups) ? 1 : 0);
  return samples * sizeof(float2) * (rows * width + groups);
}

// Calls f with a value of the (checked) type.
template <typename F>
static void by_type(int32_t dtype, F&& f) {
  with_dtype(dtype, "tgs_group_norm", [&](auto tag) {
    f(tag);
    return TGS_OK;
  });
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
              (float2*)stats, samples * pixels * width * size_of(dtype) >= ONCE_BYTES};
  HeldPlan held;
  if (gn_held(samples, pixels, width, groups, dtype, held)) {
    k.stats = nullptr;
    by_type(dtype, [&](auto tag) { gn_held<decltype(tag)>(k, held, false, nullptr, stream); });
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
  const StreamPlans plans = stream_plans(samples, pixels, width, groups, dtype);
  by_type(dtype, [&](auto tag) {
    gn_streamed_fwd<decltype(tag)>(k, plans, (float2*)workspace, stream);
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
              eps, dx, (float2*)stats, samples * pixels * width * size_of(dtype) >= ONCE_BYTES};
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
    by_type(dtype, [&](auto tag) { gn_held<decltype(tag)>(k, held, true, partial, stream); });
    join(held.partials, partial);
  } else {
    TGS_CHECK_ARG(stats && (uintptr_t)stats % 8 == 0,
                  "tgs_group_norm_bwd: the stats of the forward are needed, on 8 bytes");
    const StreamPlans plans = stream_plans(samples, pixels, width, groups, dtype);
    TGS_CHECK_ARG(!sums || samples * plans.sums.chunks < (1ull << 32),
                  "tgs_group_norm_bwd: too many samples for their sums");
    by_type(dtype, [&](auto tag) {
      const SumRows rows = gn_streamed_bwd<decltype(tag)>(k, plans, (float2*)workspace, stream);
      join(rows.count, (const float*)rows.first);
    });
  }
  TGS_RETURN_LAUNCH("tgs_group_norm_bwd");
}
