// What the gated feed-forward block's kernels share, and the interface of the kernels for
// narrow rows.
#pragma once

#include "activation.cuh"
#include "matrix.cuh"

// Eight values of a row from column c on (zeros past the width), as planes.
template <typename T>
__device__ __forceinline__ void load_fragment(const T* row, int c, int width, bool live, bool wide,
                                              frag_t<typename Planes<T>::E> (&out)[Planes<T>::N]) {
  using E = typename Planes<T>::E;
  constexpr int P = Planes<T>::N, V = Vec16<T>::N;
  T v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = (T)0.f;
  if (live) {
    if (wide) {  // rows on 16 bytes, a whole number of 16-byte runs
#pragma unroll
      for (int e = 0; e < 8; e += V)
        if (c + e < width) *(Vec16<T>*)(v + e) = *(const Vec16<T>*)(row + c + e);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c + e < width) v[e] = row[c + e];
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    E p[P];
    split<T>(to_f32(v[e]), p);
#pragma unroll
    for (int s = 0; s < P; ++s) out[s][e] = p[s];
  }
}

// a b over the pairs of planes.
template <typename T>
__device__ __forceinline__ f32x4 mfma_planes(const frag_t<typename Planes<T>::E> (&a)[Planes<T>::N],
                                             const frag_t<typename Planes<T>::E> (&b)[Planes<T>::N],
                                             f32x4 c) {
  if constexpr (Planes<T>::N == 1) {
    return mfma32(a[0], b[0], c);
  } else {
    c = mfma32(a[2], b[0], c);
    c = mfma32(a[0], b[2], c);
    c = mfma32(a[1], b[1], c);
    c = mfma32(a[1], b[0], c);
    c = mfma32(a[0], b[1], c);
    return mfma32(a[0], b[0], c);
  }
}

// Calls f with the activation as a constant.
template <typename F>
__host__ __device__ __forceinline__ void with_activation(int act, F&& f) {
  if (act == ACT_SILU)
    f(std::integral_constant<int, ACT_SILU>());
  else if (act == ACT_GELU)
    f(std::integral_constant<int, ACT_GELU>());
  else
    f(std::integral_constant<int, ACT_RELU>());
}

// The block's sizes and tensors, as the entry points get them.
struct FfnCall {
  int64_t rows;
  int32_t width, hidden, out, act;
  int64_t x_pitch, dy_pitch;
  const void *x, *wg, *wu, *wd, *bg, *bu, *bd, *dy;
  void *y, *dx, *dwg, *dwu, *dwd, *dbg, *dbu, *dbd;
};

// ---------------------------------------------------------------------------
// Half precision's backward.  h, dg and du are rounded to the tensors' type for the products
// that sum them over rows; half keeps nothing below 2^-25, where the gradients of a mean over
// an image's pixels lie, though their sums do not (9000 rows with dy of 3e-7: dWg 35% off).  They
// are multiplied by powers of two before they are rounded and the 32-bit sums divided again,
// both exact.  The powers are the largest that cannot overflow, by bounds from the tensors'
// largest magnitudes: half's 40 binary places leave 2^-40 of the bound, some 2^-25 of the values
// themselves.  Never below 1, so a row far beyond the others takes nothing from them.
// ---------------------------------------------------------------------------

template <typename T>
constexpr bool LIFTED = std::is_same<T, f16_t>::value;

struct Lift {
  float h, back_h, d, back_d;  // of h; of dg and du
};
#define LIFT_BLOCKS 512                // of a tensor at most
#define LIFT_PEAKS (7 * LIFT_BLOCKS)   // floats of workspace
void ffn_lift(const FfnCall& c, Lift* lift, float* peaks, hipStream_t stream);

// ---------------------------------------------------------------------------
// Operands that the products cannot read where they lie (32-bit values, rows that do
// not start on 16 bytes, widths that are no multiple of 8) are laid out as planes
// with rows of a whole number of chunks, zeros behind the last value.
// ---------------------------------------------------------------------------

struct LayJob {
  const void* src;
  void* dst;
  int64_t rows, pitch, plane;  // plane: values between two planes of dst
  uint32_t cols, cols8;
  uint32_t blocks;  // of the launch, up to and with this job's
};
#define LAY_JOBS 5
struct LayJobs {
  LayJob job[LAY_JOBS];
};

template <typename T>
__global__ void __launch_bounds__(256) ffn_lay_kernel(LayJobs jobs) {
  using E = typename Planes<T>::E;
  constexpr int P = Planes<T>::N;
  int k = 0;
  uint32_t first = 0;
  while (blockIdx.x >= jobs.job[k].blocks) first = jobs.job[k++].blocks;
  const LayJob& job = jobs.job[k];
  const uint32_t chunks = job.cols8 / 8;
  const uint64_t i = (uint64_t)(blockIdx.x - first) * 256 + threadIdx.x;
  const int64_t row = (int64_t)(i / chunks);
  const uint32_t c = (uint32_t)(i % chunks) * 8;
  if (row >= job.rows) return;
  const T* src = (const T*)job.src + row * job.pitch;
  frag_t<E> out[P];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    E p[P];
    split<T>(c + e < job.cols ? to_f32(src[c + e]) : 0.f, p);
#pragma unroll
    for (int q = 0; q < P; ++q) out[q][e] = p[q];
  }
  E* dst = (E*)job.dst + row * job.cols8 + c;
#pragma unroll
  for (int q = 0; q < P; ++q) *(frag_t<E>*)(dst + q * job.plane) = out[q];
}

// Partial sums joined in a fixed order and rounded: out[r, c] = sum_s partial[s, r, c].
// The rows are those of up to three tensors one after another in `partial`.
struct JoinJob {
  const float* partial;
  int64_t part;       // values between two partial sums
  int64_t pitch;      // of a row of them
  int32_t parts, cols, groups;  // groups: threads of a value
  int64_t rows;
  void* out;          // [rows, cols]
  const void* bias;   // [cols], added to the sums; nullable
  const float* factor;  // of the sums, half's; nullable
  uint32_t blocks;    // of the launch, up to and with this job's
};
#define JOIN_JOBS 6
struct JoinJobs {
  JoinJob job[JOIN_JOBS];
};

// A job's workgroup takes 256 / groups values, each summed by `groups` threads over parts g,
// g + groups, ... and then over the threads: one thread per value took 62 us for 256 parts of
// 49k values, a load after another; eight take 10.
template <typename T>
__global__ void __launch_bounds__(256) ffn_join_kernel(JoinJobs jobs) {
  __shared__ float s[256];
  int k = 0;
  uint32_t first = 0;
  while (blockIdx.x >= jobs.job[k].blocks) first = jobs.job[k++].blocks;
  const JoinJob& job = jobs.job[k];
  const int each = 256 / job.groups, e = threadIdx.x % each, g = threadIdx.x / each;
  const int64_t i = (int64_t)(blockIdx.x - first) * each + e;
  const bool live = i < job.rows * job.cols;
  float acc = 0.f;
  if (live) {
    const float* p = job.partial + i / job.cols * job.pitch + i % job.cols;
#pragma unroll 8
    for (int part = g; part < job.parts; part += job.groups) acc += p[part * job.part];
  }
  s[threadIdx.x] = acc;
  for (int h = job.groups >> 1; h > 0; h >>= 1) {
    __syncthreads();
    if (g < h) s[threadIdx.x] += s[threadIdx.x + h * each];
  }
  if (live && g == 0) {
    float v = s[threadIdx.x];
    if (LIFTED<T> && job.factor) v *= *job.factor;
    ((T*)job.out)[i] = from_f32<T>(v + (job.bias ? to_f32(((const T*)job.bias)[i % job.cols]) : 0.f));
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

static inline int64_t round8(int64_t n) { return (n + 7) / 8 * 8; }

// Hands out parts of a workspace; with a null base it only counts.
struct Carver {
  char* base;
  uint64_t used = 0;
  template <typename U>
  U* take(int64_t n) {
    U* p = base ? (U*)(base + used) : nullptr;
    used += ((uint64_t)n * sizeof(U) + 255) / 256 * 256;
    return p;
  }
};

static inline int64_t tiles(int64_t n, int64_t t) { return (n + t - 1) / t; }

// Whether a product can read a matrix where it lies.
template <typename T>
static bool in_place(const void* p, int64_t cols, int64_t pitch) {
  return Planes<T>::N == 1 && cols % 8 == 0 && pitch <= MX_PITCH && aligned16((const T*)p, pitch);
}

template <typename T>
struct Layer {
  using E = typename Planes<T>::E;
  LayJobs jobs;
  int n = 0;
  uint32_t blocks = 0;
  // The operand that holds a matrix: itself, or a copy that the next launch lays out.
  Operand<E> operand(const void* p, int64_t rows, int64_t cols, int64_t pitch, E* copy) {
    if (in_place<T>(p, cols, pitch)) return {(const E*)p, 0, pitch};
    const int64_t cols8 = round8(cols);
    blocks += (uint32_t)tiles(rows * (cols8 / 8), 256);
    jobs.job[n++] = LayJob{p, copy, rows, pitch, rows * cols8, (uint32_t)cols, (uint32_t)cols8, blocks};
    return {copy, rows * cols8, cols8};
  }
  void launch(hipStream_t s) {
    if (n) hipLaunchKernelGGL(ffn_lay_kernel<T>, dim3(blocks), dim3(256), 0, s, jobs);
    n = 0;
    blocks = 0;
  }
};

template <typename T>
static const void* row_at(const void* p, int64_t row, int64_t pitch) {
  return (const T*)p + row * pitch;
}

// Parts that a sum over `steps` is split into where `tiles` workgroups would leave the chip
// idle: up to a workgroup a CU, none shorter than four steps (more cost the partial sums'
// traffic what they save: 8000 rows of 300-900-300 in two parts 63 us, in one 51).  The partial
// sums of tiles_ * part values then stay within SPLIT_TILES tiles' values.
#define SPLIT_TILES 256
static inline int split_parts(int64_t tiles_, int64_t steps) {
  return (int)std::max<int64_t>(1, std::min<int64_t>(SPLIT_TILES / std::max<int64_t>(tiles_, 1),
                                                     steps / 4));
}

// The join of a call's partial sums, one launch.
template <typename T>
struct Joiner {
  JoinJobs jobs;
  int n = 0;
  uint32_t blocks = 0;
  void add(const float* partial, int64_t part, int64_t pitch, int64_t parts, int64_t rows,
           int64_t cols, void* to, const void* bias = nullptr, const float* factor = nullptr) {
    if (!to) return;
    // (many values in few parts keep the chip busy with a thread each)
    const int groups = parts > (rows * cols < 65536 ? 4 : 32) ? 8 : 1;
    blocks += (uint32_t)tiles(rows * cols, 256 / groups);
    jobs.job[n++] = JoinJob{partial, part, pitch, (int32_t)parts, (int32_t)cols, groups, rows, to,
                            bias, factor, blocks};
  }
  void launch(hipStream_t s) {
    if (n) hipLaunchKernelGGL(ffn_join_kernel<T>, dim3(blocks), dim3(256), 0, s, jobs);
  }
};

// Few rows (gated_ffn_few.hip): the weights' bytes are the work.
#define FEW_ROWS 32
template <typename T>
struct FewKernels {
  static uint64_t workspace(int64_t rows, int32_t hidden);
  static void forward(const FfnCall& c, void* workspace, hipStream_t stream);
};

// Narrow rows (gated_ffn_rows.cuh): whether a call's sizes are theirs, the workspace they
// take and their launches.
template <typename T>
struct RowKernels {
  static bool takes(int32_t width, int32_t out);
  static uint64_t workspace(int64_t rows, int32_t width, int32_t hidden, int32_t out, bool back);
  static void forward(const FfnCall& c, void* workspace, hipStream_t stream);
  static void backward(const FfnCall& c, void* workspace, hipStream_t stream);
};
