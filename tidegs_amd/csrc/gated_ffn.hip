// Gated feed-forward block, forward and backward:
//
//   g = x Wg' + bg, u = x Wu' + bu, h = act(g) u, y = h Wd' + bd
//   dh = dy Wd, dg = dh u act'(g), du = dh act(g)
//   dx = dg Wg + du Wu, dWg = dg' x, dWu = du' x, dWd = dy' h, db. = column sums
//
// x [rows, width], Wg and Wu [hidden, width], Wd [out, hidden], row-major (x and dy at
// a pitch).  The backward computes g and u again.
#include "decoder_common.cuh"

enum { ACT_SILU = 0, ACT_GELU = 1, ACT_RELU = 2 };

// act(g) and its derivative.
__device__ __forceinline__ float2 activation(int act, float g) {
  if (act == ACT_RELU) return g > 0.f ? make_float2(g, 1.f) : make_float2(0.f * g, 0.f);
  if (act == ACT_SILU) {
    const float s = 1.f / (1.f + expf(-g));
    return make_float2(g * s, s * (1.f + g * (1.f - s)));
  }
  const float phi = 0.5f * (1.f + erff(g * 0.70710678118654752f));
  return make_float2(g * phi, phi + g * 0.39894228040143268f * expf(-0.5f * g * g));
}

// A matrix by its strides, of the call's element type or of 32-bit values.
struct Mat {
  const void* p;
  int64_t row, col;  // strides (values)
  int wide;          // 32-bit values whatever the call's type
};

template <typename T>
__device__ __forceinline__ float at(const Mat& m, int64_t r, int64_t c) {
  const int64_t i = r * m.row + c * m.col;
  return m.wide ? ((const float*)m.p)[i] : to_f32(((const T*)m.p)[i]);
}

// C[m,n] = sum_k A[m,k] B[k,n] (+ A2 B2) + bias[n], 16 x 16 tiles through LDS.
template <typename T>
__global__ void __launch_bounds__(256) ffn_product_kernel(int64_t M, int64_t N, int64_t K, Mat A,
                                                          Mat B, Mat A2, Mat B2,
                                                          const T* __restrict__ bias, void* C,
                                                          int c_wide) {
  __shared__ float s_a[16][17], s_b[16][17];
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  const int64_t tiles_n = (N + 15) / 16;
  const int64_t m = blockIdx.x / tiles_n * 16 + ty, n = blockIdx.x % tiles_n * 16 + tx;
  const int64_t mb = m - ty + tx;  // the row this thread loads of A where k runs along ty
  double acc = 0.0;
  for (int pair = 0; pair < (A2.p ? 2 : 1); ++pair) {
    const Mat& a = pair ? A2 : A;
    const Mat& b = pair ? B2 : B;
    for (int64_t k0 = 0; k0 < K; k0 += 16) {
      s_a[tx][ty] = mb < M && k0 + ty < K ? at<T>(a, mb, k0 + ty) : 0.f;
      s_b[ty][tx] = n < N && k0 + ty < K ? at<T>(b, k0 + ty, n) : 0.f;
      __syncthreads();
#pragma unroll
      for (int k = 0; k < 16; ++k) acc += (double)s_a[ty][k] * (double)s_b[k][tx];
      __syncthreads();
    }
  }
  if (m >= M || n >= N) return;
  const float v = (float)acc + (bias ? to_f32(bias[n]) : 0.f);
  if (c_wide)
    ((float*)C)[m * N + n] = v;
  else
    ((T*)C)[m * N + n] = from_f32<T>(v);
}

// g -> h in place of g (forward); g, u, dh -> dg, du, h in their places (backward).
__global__ void __launch_bounds__(256) ffn_gate_kernel(uint64_t n, int act, float* __restrict__ g,
                                                       float* __restrict__ u,
                                                       float* __restrict__ dh) {
  for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < n;
       i += (uint64_t)gridDim.x * 256) {
    const float2 a = activation(act, g[i]);
    const float uu = u[i];
    if (!dh) {
      g[i] = a.x * uu;
      continue;
    }
    const float d = dh[i];
    g[i] = d * uu * a.y;
    u[i] = d * a.x;
    dh[i] = a.x * uu;
  }
}

// Sums of a matrix's columns, one wavefront per column.
template <typename T>
__global__ void __launch_bounds__(64) ffn_column_sum_kernel(int64_t rows, Mat A,
                                                            T* __restrict__ out) {
  float acc = 0.f;
  for (int64_t r = threadIdx.x; r < rows; r += 64) acc += at<T>(A, r, blockIdx.x);
  acc = tgs_wave_sum(acc);
  if (threadIdx.x == 0) out[blockIdx.x] = from_f32<T>(acc);
}

template <typename T>
static void product(hipStream_t s, int64_t M, int64_t N, int64_t K, Mat A, Mat B, const T* bias,
                    void* C, int c_wide, Mat A2 = Mat{}, Mat B2 = Mat{}) {
  hipLaunchKernelGGL(ffn_product_kernel<T>, dim3((unsigned)(((M + 15) / 16) * ((N + 15) / 16))),
                     dim3(256), 0, s, M, N, K, A, B, A2, B2, bias, C, c_wide);
}

static int check_sizes(const char* name, uint64_t rows, uint32_t width, uint32_t hidden,
                       uint32_t out, int32_t activation) {
  TGS_CHECK_ARG(width > 0 && hidden > 0 && out > 0, "%s: width, hidden and out are positive", name);
  TGS_CHECK_ARG(width <= 65536 && hidden <= 65536 && out <= 65536,
                "%s: width, hidden and out go up to 65536", name);
  TGS_CHECK_ARG(rows <= 0x7FFFFFFFull, "%s: rows go up to 2^31 - 1", name);
  TGS_CHECK_ARG(activation >= 0 && activation <= 2,
                "%s: activation must be 0 (silu), 1 (gelu) or 2 (relu)", name);
  return TGS_OK;
}

extern "C" uint64_t tgs_gated_ffn_fwd_workspace_size(uint64_t rows, uint32_t width, uint32_t hidden,
                                                     uint32_t out, int32_t dtype) {
  (void)width, (void)out, (void)dtype;
  return 2 * rows * hidden * sizeof(float);
}

extern "C" uint64_t tgs_gated_ffn_bwd_workspace_size(uint64_t rows, uint32_t width, uint32_t hidden,
                                                     uint32_t out, int32_t dtype) {
  (void)width, (void)out, (void)dtype;
  return 3 * rows * hidden * sizeof(float);
}

extern "C" int tgs_gated_ffn_fwd(uint64_t rows, uint32_t width, uint32_t hidden, uint32_t out,
                                 int32_t dtype, int32_t activation, const void* x, int64_t x_pitch,
                                 const void* w_gate, const void* w_up, const void* w_down,
                                 const void* b_gate, const void* b_up, const void* b_down, void* y,
                                 void* workspace, uint64_t workspace_bytes, hipStream_t stream) {
  return with_dtype(dtype, "tgs_gated_ffn_fwd", [&](auto tag) -> int {
    using T = decltype(tag);
    if (const int rc = check_sizes("tgs_gated_ffn_fwd", rows, width, hidden, out, activation))
      return rc;
    if (rows == 0) return TGS_OK;
    TGS_CHECK_ARG(x && w_gate && w_up && w_down && y, "tgs_gated_ffn_fwd: null pointer");
    TGS_CHECK_ARG(x_pitch >= (int64_t)width || rows == 1, "tgs_gated_ffn_fwd: pitch below width");
    if (workspace_bytes < tgs_gated_ffn_fwd_workspace_size(rows, width, hidden, out, dtype)) {
      tgs_set_error("tgs_gated_ffn_fwd: workspace too small");
      return TGS_ERR_WORKSPACE;
    }
    const int64_t M = rows, D = width, F = hidden, O = out;
    float *g = (float*)workspace, *u = g + M * F;
    const Mat X{x, x_pitch, 1, 0};
    product<T>(stream, M, F, D, X, Mat{w_gate, 1, D, 0}, (const T*)b_gate, g, 1);
    product<T>(stream, M, F, D, X, Mat{w_up, 1, D, 0}, (const T*)b_up, u, 1);
    hipLaunchKernelGGL(ffn_gate_kernel, dim3(std::min<int64_t>((M * F + 255) / 256, 65536)),
                       dim3(256), 0, stream, (uint64_t)(M * F), activation, g, u, (float*)nullptr);
    product<T>(stream, M, O, F, Mat{g, F, 1, 1}, Mat{w_down, 1, F, 0}, (const T*)b_down, y, 0);
    TGS_RETURN_LAUNCH("tgs_gated_ffn_fwd");
  });
}

extern "C" int tgs_gated_ffn_bwd(uint64_t rows, uint32_t width, uint32_t hidden, uint32_t out,
                                 int32_t dtype, int32_t activation, const void* x, int64_t x_pitch,
                                 const void* w_gate, const void* w_up, const void* w_down,
                                 const void* b_gate, const void* b_up, const void* dy,
                                 int64_t dy_pitch, void* dx, void* dw_gate, void* dw_up,
                                 void* dw_down, void* db_gate, void* db_up, void* db_down,
                                 void* workspace, uint64_t workspace_bytes, hipStream_t stream) {
  return with_dtype(dtype, "tgs_gated_ffn_bwd", [&](auto tag) -> int {
    using T = decltype(tag);
    if (const int rc = check_sizes("tgs_gated_ffn_bwd", rows, width, hidden, out, activation))
      return rc;
    TGS_CHECK_ARG(w_gate && w_up && w_down && (rows == 0 || (x && dy)),
                  "tgs_gated_ffn_bwd: null pointer");
    TGS_CHECK_ARG((x_pitch >= (int64_t)width && dy_pitch >= (int64_t)out) || rows <= 1,
                  "tgs_gated_ffn_bwd: pitch below width");
    if (workspace_bytes < tgs_gated_ffn_bwd_workspace_size(rows, width, hidden, out, dtype)) {
      tgs_set_error("tgs_gated_ffn_bwd: workspace too small");
      return TGS_ERR_WORKSPACE;
    }
    const int64_t M = rows, D = width, F = hidden, O = out;
    float *g = (float*)workspace, *u = g + M * F, *dh = u + M * F;
    const Mat X{x, x_pitch, 1, 0}, DY{dy, dy_pitch, 1, 0};
    const Mat G{g, F, 1, 1}, U{u, F, 1, 1}, H{dh, F, 1, 1};
    if (M) {
      product<T>(stream, M, F, D, X, Mat{w_gate, 1, D, 0}, (const T*)b_gate, g, 1);
      product<T>(stream, M, F, D, X, Mat{w_up, 1, D, 0}, (const T*)b_up, u, 1);
      product<T>(stream, M, F, O, DY, Mat{w_down, F, 1, 0}, (const T*)nullptr, dh, 1);
      hipLaunchKernelGGL(ffn_gate_kernel, dim3(std::min<int64_t>((M * F + 255) / 256, 65536)),
                         dim3(256), 0, stream, (uint64_t)(M * F), activation, g, u, dh);
      if (dx)
        product<T>(stream, M, D, F, G, Mat{w_gate, D, 1, 0}, (const T*)nullptr, dx, 0, U,
                   Mat{w_up, D, 1, 0});
    }
    const T* none = nullptr;
    if (dw_gate) product<T>(stream, F, D, M, Mat{g, 1, F, 1}, X, none, dw_gate, 0);
    if (dw_up) product<T>(stream, F, D, M, Mat{u, 1, F, 1}, X, none, dw_up, 0);
    if (dw_down) product<T>(stream, O, F, M, Mat{dy, 1, dy_pitch, 0}, H, none, dw_down, 0);
    const auto sums = [&](const Mat& A, int64_t n, void* db) {
      if (db)
        hipLaunchKernelGGL(ffn_column_sum_kernel<T>, dim3((unsigned)n), dim3(64), 0, stream, M, A,
                           (T*)db);
    };
    sums(G, F, db_gate);
    sums(U, F, db_up);
    sums(DY, O, db_down);
    TGS_RETURN_LAUNCH("tgs_gated_ffn_bwd");
  });
}
