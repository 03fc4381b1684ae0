// The gated feed-forward block over narrow rows (width and out up to 128): the hidden values
// of a row never leave the registers.
//
// A wavefront holds 16 RT rows of x as the second operand of its products and walks the
// hidden columns in chunks of 32.  The products are taken transposed: g' = Wg x', so a
// lane's accumulators hold four hidden columns of one row, which is, for the two
// 16-column tiles of a chunk together, the layout of the second operand of y' = Wd h' over
// those 32 columns (the tiles' rows are dealt so that the lane's eight are neighbours).
// The gate and the rounding happen in place and no value crosses a lane.
//
// The weights are laid out once per call, fragment by fragment as a lane reads them, chunk
// after chunk; the wavefronts of a workgroup share the chunk in LDS, copied there without
// registers while the chunk before it is multiplied.
#pragma once

#include "gated_ffn.cuh"

// KB of a chunk of 32 hidden columns: fragments and 1 KB for the biases.
template <typename T, int DK, int OT>
struct ForwardChunk {
  static constexpr int P = Planes<T>::N;
  static constexpr int FRAGMENTS = 4 * DK + OT;  // Wg and Wu: two tiles by DK each; Wd: OT
  static constexpr int KB = FRAGMENTS * P + 1;
};

struct PackArgs {
  const void *wg, *wu, *wd, *bg, *bu;
  char* out;
  int32_t width, hidden, out_n, chunks, dk, ot, kb;
};

// The hidden column of row r of tile t of a chunk.
__device__ __forceinline__ int dealt(int chunk, int t, int r) {
  return chunk * 32 + (r >> 2) * 8 + t * 4 + (r & 3);
}

// One wavefront per fragment (and one per chunk for its biases).
template <typename T>
__global__ void __launch_bounds__(64) ffn_pack_kernel(PackArgs a) {
  using E = typename Planes<T>::E;
  constexpr int P = Planes<T>::N;
  const int lane = threadIdx.x;
  const int per = 4 * a.dk + a.ot + 1;
  const int chunk = blockIdx.x / per, q = blockIdx.x % per;
  char* base = a.out + (int64_t)chunk * a.kb * 1024;
  if (q == per - 1) {
    const int f = chunk * 32 + (lane & 31);
    const T* b = (const T*)(lane < 32 ? a.bg : a.bu);
    ((float*)(base + (a.kb - 1) * 1024))[lane] = b && f < a.hidden ? to_f32(b[f]) : 0.f;
    return;
  }
  frag_t<E> out[P];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int k = (lane >> 4) * 8 + j;
    float v = 0.f;
    if (q < 4 * a.dk) {  // [gate, up][tile][k step]
      const T* w = (const T*)(q < 2 * a.dk ? a.wg : a.wu);
      const int f = dealt(chunk, q / a.dk & 1, lane & 15), d = q % a.dk * 32 + k;
      if (f < a.hidden && d < a.width) v = to_f32(w[(int64_t)f * a.width + d]);
    } else {
      const int o = (q - 4 * a.dk) * 16 + (lane & 15), f = chunk * 32 + k;
      if (o < a.out_n && f < a.hidden) v = to_f32(((const T*)a.wd)[(int64_t)o * a.hidden + f]);
    }
    E p[P];
    split<T>(v, p);
#pragma unroll
    for (int s = 0; s < P; ++s) out[s][j] = p[s];
  }
#pragma unroll
  for (int s = 0; s < P; ++s) ((frag_t<E>*)(base + (q * P + s) * 1024))[lane] = out[s];
}

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

template <typename T>
struct ForwardArgs {
  const T* x;
  T* y;
  const char* packed;
  const T* bd;
  int64_t rows, x_pitch;
  int32_t width, out, chunks, act;
  int32_t wide;      // x is read 16 bytes at a time
  int32_t wide_out;  // y is written four values at a time
};

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

// KB kilobytes to LDS by WAVES wavefronts, without registers.
template <int KB, int WAVES>
__device__ __forceinline__ void copy_chunk(char* lds, const char* src) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const rsrc_t r = buffer_of(src, KB * 1024);
#pragma unroll
  for (int j = 0; j < KB; j += WAVES)
    if (j + wave < KB)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)(lds + (j + wave) * 1024), 16,
                                               (j + wave) * 1024 + (threadIdx.x & 63) * 16, 0, 0, 0);
}

#define FR_WAVES 8

template <typename T, int DK, int OT, int RT>
__global__ void __launch_bounds__(64 * FR_WAVES) ffn_rows_fwd_kernel(ForwardArgs<T> a) {
  using E = typename Planes<T>::E;
  constexpr int P = Planes<T>::N;
  using C = ForwardChunk<T, DK, OT>;
  __shared__ __attribute__((aligned(1024))) char lds[2 * C::KB * 1024];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  constexpr int TILE = 16 * RT * FR_WAVES;
  const int64_t tiles = (a.rows + TILE - 1) / TILE;
  for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const int64_t m0 = tile * TILE + wave * 16 * RT + (lane & 15);
    copy_chunk<C::KB, FR_WAVES>(lds, a.packed);
    frag_t<E> x[RT][DK][P];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const int64_t m = m0 + i * 16;
#pragma unroll
      for (int k = 0; k < DK; ++k)
        load_fragment<T>(a.x + m * a.x_pitch, k * 32 + (lane >> 4) * 8, a.width, m < a.rows, a.wide,
                         x[i][k]);
    }
    f32x4 y[OT][RT] = {};
    for (int c = 0; c < a.chunks; ++c) {
      __syncthreads();  // the chunk is there, and nobody reads the one before it
      const char* cur = lds + (c & 1) * C::KB * 1024;
      if (c + 1 < a.chunks)
        copy_chunk<C::KB, FR_WAVES>(lds + (~c & 1) * C::KB * 1024,
                                    a.packed + (int64_t)(c + 1) * C::KB * 1024);
      const auto fragment = [&](int q, frag_t<E>(&f)[P]) {
#pragma unroll
        for (int s = 0; s < P; ++s) f[s] = ((const frag_t<E>*)(cur + (q * P + s) * 1024))[lane];
      };
      const float* bias = (const float*)(cur + (C::KB - 1) * 1024) + (lane >> 4) * 8;
      frag_t<E> h[RT][P];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        f32x4 g[RT], u[RT];
        const f32x4 bg = *(const f32x4*)(bias + t * 4), bu = *(const f32x4*)(bias + 32 + t * 4);
#pragma unroll
        for (int i = 0; i < RT; ++i) g[i] = bg, u[i] = bu;
#pragma unroll
        for (int k = 0; k < DK; ++k) {
          frag_t<E> w[P];
          fragment(t * DK + k, w);
#pragma unroll
          for (int i = 0; i < RT; ++i) g[i] = mfma_planes<T>(w, x[i][k], g[i]);
          fragment((2 + t) * DK + k, w);
#pragma unroll
          for (int i = 0; i < RT; ++i) u[i] = mfma_planes<T>(w, x[i][k], u[i]);
        }
        with_activation(a.act, [&](auto act) {
#pragma unroll
          for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              E p[P];
              split<T>(activation<T, act.value>(g[i][r]).x * u[i][r], p);
#pragma unroll
              for (int s = 0; s < P; ++s) h[i][s][t * 4 + r] = p[s];
            }
        });
      }
#pragma unroll
      for (int o = 0; o < OT; ++o) {
        frag_t<E> w[P];
        fragment(4 * DK + o, w);
#pragma unroll
        for (int i = 0; i < RT; ++i) y[o][i] = mfma_planes<T>(w, h[i], y[o][i]);
      }
    }
    __syncthreads();  // (the next rows' first chunk goes where the last one lay)
#pragma unroll
    for (int o = 0; o < OT; ++o) {
      const int n = o * 16 + (lane >> 4) * 4;
      float bd[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) bd[r] = a.bd && n + r < a.out ? to_f32(a.bd[n + r]) : 0.f;
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        const int64_t m = m0 + i * 16;
        if (m >= a.rows || n >= a.out) continue;
        T* at = a.y + m * a.out + n;
        if (a.wide_out) {
          four_t<T> v;
#pragma unroll
          for (int r = 0; r < 4; ++r) v[r] = from_f32<T>(y[o][i][r] + bd[r]);
          *(four_t<T>*)at = v;
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (n + r < a.out) at[r] = from_f32<T>(y[o][i][r] + bd[r]);
        }
      }
    }
  }
}

// Calls f(DK, OT) as constants.
template <typename F>
static void with_narrow(int width, int out, F&& f) {
  const auto by_out = [&](auto dk) {
    if (out <= 16) return f(dk, std::integral_constant<int, 1>());
    if (out <= 32) return f(dk, std::integral_constant<int, 2>());
    if (out <= 48) return f(dk, std::integral_constant<int, 3>());
    if (out <= 64) return f(dk, std::integral_constant<int, 4>());
    return f(dk, std::integral_constant<int, 8>());
  };
  if (width <= 32) return by_out(std::integral_constant<int, 1>());
  if (width <= 64) return by_out(std::integral_constant<int, 2>());
  return by_out(std::integral_constant<int, 4>());
}

#define NARROW 128

template <typename T>
bool RowKernels<T>::takes(int64_t rows, int32_t width, int32_t hidden, int32_t out) {
  (void)rows, (void)hidden;
  return width <= NARROW && out <= NARROW;
}

template <typename T>
uint64_t RowKernels<T>::workspace(int32_t width, int32_t hidden, int32_t out) {
  uint64_t kb = 0;
  with_narrow(width, out, [&](auto dk, auto ot) { kb = ForwardChunk<T, dk.value, ot.value>::KB; });
  return kb * 1024 * ((hidden + 31) / 32);
}

template <typename T>
void RowKernels<T>::forward(const FfnCall& c, void* workspace, hipStream_t stream) {
  const int chunks = (c.hidden + 31) / 32;
  with_narrow(c.width, c.out, [&](auto dk, auto ot) {
    constexpr int DK = dk.value, OT = ot.value;
    using C = ForwardChunk<T, DK, OT>;
    const PackArgs pack{c.wg, c.wu, c.wd, c.bg, c.bu, (char*)workspace, c.width, c.hidden, c.out,
                        chunks, DK, OT, C::KB};
    hipLaunchKernelGGL(ffn_pack_kernel<T>, dim3(chunks * (C::FRAGMENTS + 1)), dim3(64), 0, stream,
                       pack);
    const ForwardArgs<T> a{(const T*)c.x, (T*)c.y, (const char*)workspace, (const T*)c.bd, c.rows,
                           c.x_pitch, c.width, c.out, chunks, c.act,
                           c.width % Vec16<T>::N == 0 && aligned16((const T*)c.x, c.x_pitch),
                           c.out % 4 == 0 && aligned16((const T*)c.y, 0)};
    const auto launch = [&](auto kernel, int rt) {
      const int64_t tiles = (c.rows + 16 * rt * FR_WAVES - 1) / (16 * rt * FR_WAVES);
      hipLaunchKernelGGL(kernel, dim3((unsigned)std::min<int64_t>(tiles, 512)), dim3(64 * FR_WAVES),
                         0, stream, a);
    };
    constexpr int MANY = Planes<T>::N == 1 && DK <= 2 && OT <= 4 ? 4 : 2;
    if (c.rows >= 16 * MANY * FR_WAVES * 256)
      launch(ffn_rows_fwd_kernel<T, DK, OT, MANY>, MANY);
    else
      launch(ffn_rows_fwd_kernel<T, DK, OT, 1>, 1);
  });
}
