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
// h, dg and du of 16-bit tensors are rounded to their type there, once, as a stored hidden
// tensor is: y, dx and the weights' gradients come out 0.0023 of themselves off in bfloat16,
// where rounding the results alone takes 0.0017.  A second plane of them, as the kernels for few
// rows keep, would be as many products with them again.
//
// The weights are laid out once per call, fragment by fragment as a lane reads them, chunk
// after chunk; the wavefronts of a workgroup share the chunk in LDS, copied there without
// registers while the chunk before it is multiplied.
//
// Bound by the gate's arithmetic: 1M rows of 64-256-64 bfloat16 issue vector instructions in
// 60% of the SIMDs' cycles, among them an exponential and a reciprocal a hidden value at a
// quarter of the rate, beside matrix instructions in 34%, with no LDS bank conflicts; the
// backward in one kernel in 41% beside 28%, waiting for LDS and its barriers.
//   1M rows bfloat16 of 64-256-48, forward: 115 us, 780 TFLOP/s; of 64-256-64: forward 135
//     (730), backward in one kernel 387 (680, the hidden products included)
//   300k rows float32 of 59-128-3 (six products a product): 78, 143 and 138 us
#pragma once

#include "gated_ffn.cuh"

// A chunk of 32 hidden columns: fragments (times the planes) and 1 KB for the biases.
// DK, OK: k steps of 32 of the width and of the out; OT, DT: tiles of 16.
template <typename T, int DK, int OT>
struct ForwardChunk {  // Wg, Wu: two tiles by DK; Wd: OT tiles
  static constexpr int FRAGMENTS = 4 * DK + OT;
  static constexpr int KB = FRAGMENTS * Planes<T>::N + 1;
};
template <typename T, int DK, int OK>
struct BackwardChunk {  // Wg, Wu: two tiles by DK; Wd': two tiles by OK; Wg', Wu': 2 DK tiles
  static constexpr int FRAGMENTS = 8 * DK + 2 * OK;
  static constexpr int KB = FRAGMENTS * Planes<T>::N + 1;
};

// The columns of a chunk's fragment behind the last hidden one become zeros: there g and u are
// products with zeros, NaN where x is infinite, and would reach the row's other outputs.
// (Three planes make an infinity NaN by themselves.)
template <typename E, int P>
__device__ __forceinline__ void keep_hidden(frag_t<E> (&f)[P], int left) {
  if constexpr (P == 1) {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[0][e] = (int)(threadIdx.x & 63) / 16 * 8 + e < left ? f[0][e] : (E)0.f;
  }
}

struct PackArgs {
  const void *wg, *wu, *wd, *bg, *bu;
  char* out;
  int32_t width, hidden, out_n, dk, ot, ok, kb;  // ot: forward; ok: backward
};

// The hidden column of row r of tile t of a chunk.
__device__ __forceinline__ int dealt(int chunk, int t, int r) {
  return chunk * 32 + (r >> 2) * 8 + t * 4 + (r & 3);
}

// One wavefront per fragment (and one per chunk for its biases).
template <typename T, bool BACK>
__global__ void __launch_bounds__(64) ffn_pack_kernel(PackArgs a) {
  using E = typename Planes<T>::E;
  constexpr int P = Planes<T>::N;
  const int lane = threadIdx.x, row = lane & 15;
  const int per = (BACK ? 8 * a.dk + 2 * a.ok : 4 * a.dk + a.ot) + 1;
  const int chunk = blockIdx.x / per;
  const int q = blockIdx.x % per;
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
    const void* w;
    int r, c, rows, cols;  // of the weight's element
    if (q < 4 * a.dk) {  // [gate, up][tile][k step]
      w = q < 2 * a.dk ? a.wg : a.wu;
      r = dealt(chunk, q / a.dk & 1, row), c = q % a.dk * 32 + k;
      rows = a.hidden, cols = a.width;
    } else if (!BACK) {
      w = a.wd;
      r = (q - 4 * a.dk) * 16 + row, c = chunk * 32 + k;
      rows = a.out_n, cols = a.hidden;
    } else if (q < 4 * a.dk + 2 * a.ok) {  // Wd' [tile][k step]
      const int i = q - 4 * a.dk;
      w = a.wd;
      r = i % a.ok * 32 + k, c = dealt(chunk, i / a.ok, row);
      rows = a.out_n, cols = a.hidden;
    } else {  // Wg', Wu' [gate, up][tile]
      const int i = q - 4 * a.dk - 2 * a.ok;
      w = i < 2 * a.dk ? a.wg : a.wu;
      r = chunk * 32 + k, c = i % (2 * a.dk) * 16 + row;
      rows = a.hidden, cols = a.width;
    }
    E p[P];
    split<T>(r < rows && c < cols ? to_f32(((const T*)w)[(int64_t)r * cols + c]) : 0.f, p);
#pragma unroll
    for (int s = 0; s < P; ++s) out[s][j] = p[s];
  }
#pragma unroll
  for (int s = 0; s < P; ++s) ((frag_t<E>*)(base + (q * P + s) * 1024))[lane] = out[s];
}

template <typename T>
struct ForwardArgs {
  const T* x;
  T* y;
  const char* packed;
  const T* bd;
  int64_t rows, x_pitch;
  int32_t width, out, chunks, hidden;
  float* parts;      // not null: [gridDim.y, rows, out], chunks dealt over gridDim.y
  int32_t wide;      // x is read 16 bytes at a time
  int32_t wide_out;  // y is written four values at a time
};

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

#define FR_WAVES 8  // of a workgroup

// Up to four values of a partial row.
__device__ __forceinline__ void put_part(float* at, f32x4 v, int left) {
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (r < left) at[r] = v[r];
}

// Up to four values of a result's row, in one store where its rows allow that.
template <typename T>
__device__ __forceinline__ void put_four(T* at, f32x4 v, int left, bool whole) {
  if (whole) {
    four_t<T> t;
#pragma unroll
    for (int r = 0; r < 4; ++r) t[r] = from_f32<T>(v[r]);
    *(four_t<T>*)at = t;
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (r < left) at[r] = from_f32<T>(v[r]);
  }
}

template <typename T, int DK, int OT, int RT, int ACT>
__global__ void __launch_bounds__(64 * FR_WAVES) ffn_rows_fwd_kernel(ForwardArgs<T> a) {
  using E = typename Planes<T>::E;
  constexpr int P = Planes<T>::N;
  using C = ForwardChunk<T, DK, OT>;
  __shared__ __attribute__((aligned(1024))) char lds[2 * C::KB * 1024];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  constexpr int TILE = 16 * RT * FR_WAVES;
  const int64_t m0 = (int64_t)blockIdx.x * TILE + wave * 16 * RT + (lane & 15);
  // this workgroup's chunks
  const int first = a.chunks * blockIdx.y / gridDim.y;
  const int chunks = a.chunks * (blockIdx.y + 1) / gridDim.y - first;
  const char* packed = a.packed + (int64_t)first * C::KB * 1024;
  copy_chunk<C::KB, FR_WAVES>(lds, packed);
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
  for (int c = 0; c < chunks; ++c) {
    stage_barrier();  // the chunk is there, and nobody reads the one before it
    const char* cur = lds + (c & 1) * C::KB * 1024;
    if (c + 1 < chunks)
      copy_chunk<C::KB, FR_WAVES>(lds + (~c & 1) * C::KB * 1024,
                                  packed + (int64_t)(c + 1) * C::KB * 1024);
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
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        float v[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = activation<ACT, T>(g[i][r]).x * u[i][r];
        four_t<E> p[P];
        split4<T>(v, p);
        set_half<E, P>(h[i], t, p);
      }
    }
    if (P == 1 && (first + c + 1) * 32 > a.hidden)
#pragma unroll
      for (int i = 0; i < RT; ++i) keep_hidden<E, P>(h[i], a.hidden - (first + c) * 32);
#pragma unroll
    for (int o = 0; o < OT; ++o) {
      frag_t<E> w[P];
      fragment(4 * DK + o, w);
#pragma unroll
      for (int i = 0; i < RT; ++i) y[o][i] = mfma_planes<T>(w, h[i], y[o][i]);
    }
  }
#pragma unroll
  for (int o = 0; o < OT; ++o) {
    const int n = o * 16 + (lane >> 4) * 4;
    f32x4 bd;
#pragma unroll
    for (int r = 0; r < 4; ++r) bd[r] = a.bd && n + r < a.out ? to_f32(a.bd[n + r]) : 0.f;
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const int64_t m = m0 + i * 16;
      if (m >= a.rows || n >= a.out) continue;
      if (a.parts)
        put_part(a.parts + ((int64_t)blockIdx.y * a.rows + m) * a.out + n, y[o][i], a.out - n);
      else
        put_four(a.y + m * a.out + n, y[o][i] + bd, a.out - n, a.wide_out);
    }
  }
}

// ---------------------------------------------------------------------------
// dx: the forward's walk with dh = dy Wd beside g and u, and dx' = Wg' dg' + Wu' du' in
// place of y.
// ---------------------------------------------------------------------------

template <typename T>
struct BackwardArgs {
  const T *x, *dy;
  T* dx;
  const char* packed;
  int64_t rows, x_pitch, dy_pitch;
  int32_t width, out, chunks, hidden;
  float* parts;                    // not null: [gridDim.y, rows, width], as the forward's
  int32_t wide, wide_dy, wide_dx;  // 16 bytes at a time; dx: four values
  const Lift* lift;                // half's
};

template <typename T, int DK, int OK, int RT, int ACT>
__global__ void __launch_bounds__(64 * FR_WAVES) ffn_rows_dx_kernel(BackwardArgs<T> a) {
  using E = typename Planes<T>::E;
  constexpr int P = Planes<T>::N, DT = 2 * DK;
  using C = BackwardChunk<T, DK, OK>;
  constexpr int BUFFERS = P == 3 ? 1 : 2;  // one, so that two workgroups share a CU
  __shared__ __attribute__((aligned(1024))) char lds[BUFFERS * C::KB * 1024];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  constexpr int TILE = 16 * RT * FR_WAVES;
  const int64_t m0 = (int64_t)blockIdx.x * TILE + wave * 16 * RT + (lane & 15);
  // this workgroup's chunks
  const int first = a.chunks * blockIdx.y / gridDim.y;
  const int chunks = a.chunks * (blockIdx.y + 1) / gridDim.y - first;
  const char* packed = a.packed + (int64_t)first * C::KB * 1024;
  copy_chunk<C::KB, FR_WAVES>(lds, packed);
  frag_t<E> x[RT][DK][P], dy[RT][OK][P];
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    const int64_t m = m0 + i * 16;
    const int c = (lane >> 4) * 8;
#pragma unroll
    for (int k = 0; k < DK; ++k)
      load_fragment<T>(a.x + m * a.x_pitch, k * 32 + c, a.width, m < a.rows, a.wide, x[i][k]);
#pragma unroll
    for (int k = 0; k < OK; ++k)
      load_fragment<T>(a.dy + m * a.dy_pitch, k * 32 + c, a.out, m < a.rows, a.wide_dy, dy[i][k]);
  }
  f32x4 dx[DT][RT] = {};
  Lift lift;
  if constexpr (LIFTED<T>) lift = *a.lift;
  for (int c = 0; c < chunks; ++c) {
    if (BUFFERS == 1 && c) {
      stage_barrier();
      copy_chunk<C::KB, FR_WAVES>(lds, packed + (int64_t)c * C::KB * 1024);
    }
    stage_barrier();  // the chunk is there, and nobody reads the one before it
    const char* cur = lds + (BUFFERS == 2 ? (c & 1) * C::KB * 1024 : 0);
    if (BUFFERS == 2 && c + 1 < chunks)
      copy_chunk<C::KB, FR_WAVES>(lds + (~c & 1) * C::KB * 1024,
                                  packed + (int64_t)(c + 1) * C::KB * 1024);
    const auto fragment = [&](int q, frag_t<E>(&f)[P]) {
#pragma unroll
      for (int s = 0; s < P; ++s) f[s] = ((const frag_t<E>*)(cur + (q * P + s) * 1024))[lane];
    };
    const float* bias = (const float*)(cur + (C::KB - 1) * 1024) + (lane >> 4) * 8;
    frag_t<E> dg[RT][P], du[RT][P];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      f32x4 g[RT], u[RT], dh[RT] = {};
      const f32x4 bg = *(const f32x4*)(bias + t * 4), bu = *(const f32x4*)(bias + 32 + t * 4);
#pragma unroll
      for (int i = 0; i < RT; ++i) g[i] = bg, u[i] = bu;
      frag_t<E> w[P];
#pragma unroll
      for (int k = 0; k < DK; ++k) {
        fragment(t * DK + k, w);
#pragma unroll
        for (int i = 0; i < RT; ++i) g[i] = mfma_planes<T>(w, x[i][k], g[i]);
        fragment((2 + t) * DK + k, w);
#pragma unroll
        for (int i = 0; i < RT; ++i) u[i] = mfma_planes<T>(w, x[i][k], u[i]);
      }
#pragma unroll
      for (int k = 0; k < OK; ++k) {
        fragment(4 * DK + t * OK + k, w);
#pragma unroll
        for (int i = 0; i < RT; ++i) dh[i] = mfma_planes<T>(w, dy[i][k], dh[i]);
      }
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        float vg[4], vu[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float2 v = activation<ACT, T>(g[i][r]);
          float d = dh[i][r];
          if constexpr (LIFTED<T>) d *= lift.d;
          vg[r] = d * u[i][r] * v.y;
          vu[r] = d * v.x;
        }
        four_t<E> p[P];
        split4<T>(vg, p);
        set_half<E, P>(dg[i], t, p);
        split4<T>(vu, p);
        set_half<E, P>(du[i], t, p);
      }
    }
    if (P == 1 && (first + c + 1) * 32 > a.hidden)
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        keep_hidden<E, P>(dg[i], a.hidden - (first + c) * 32);
        keep_hidden<E, P>(du[i], a.hidden - (first + c) * 32);
      }
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      frag_t<E> w[P];
      fragment(4 * DK + 2 * OK + d, w);
#pragma unroll
      for (int i = 0; i < RT; ++i) dx[d][i] = mfma_planes<T>(w, dg[i], dx[d][i]);
      fragment(4 * DK + 2 * OK + DT + d, w);
#pragma unroll
      for (int i = 0; i < RT; ++i) dx[d][i] = mfma_planes<T>(w, du[i], dx[d][i]);
    }
  }
#pragma unroll
  for (int d = 0; d < DT; ++d) {
    const int n = d * 16 + (lane >> 4) * 4;
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const int64_t m = m0 + i * 16;
      if (m >= a.rows || n >= a.width) continue;
      if constexpr (LIFTED<T>) dx[d][i] *= lift.back_d;
      if (a.parts) {
        put_part(a.parts + ((int64_t)blockIdx.y * a.rows + m) * a.width + n, dx[d][i], a.width - n);
        continue;
      }
      put_four(a.dx + m * a.width + n, dx[d][i], a.width - n, a.wide_dx);
    }
  }
}

// ---------------------------------------------------------------------------
// The weights' gradients.  A wavefront owns 16 FT hidden columns: their weights and the
// accumulators of their gradients stay in its registers while it walks the rows, 32 at a
// time.  g, u and dh are taken with the rows first (the same fragments, exchanged), so a
// lane holds, of one hidden column, the rows that the second operand of
// dWg' = x' dg wants of it; x' and dy' come out of LDS by the transposing read from the
// tile that x and dy are read from as they lie.  The wavefronts of a workgroup share the
// tile; the rows are dealt over gridDim.x workgroups, whose partial sums a second launch
// joins.  db of the hidden products adds up beside, dbd is dy' times ones.
// ---------------------------------------------------------------------------

template <typename T>
struct WeightArgs {
  using E = typename Planes<T>::E;
  Operand<E> x, dy;
  const T *wg, *wu, *wd, *bg, *bu;
  float *dwgu, *dwd, *sums, *dy_sums;  // [gridDim.x, ...]; dy_sums nullable
  int64_t rows;
  int32_t width, hidden, out, add;
  T* dx;  // where dx is taken along; its packed weights, their chunks, four values at a time
  const char* packed;
  int32_t chunks, wide_dx;
  const Lift* lift;  // half's
};

// Rows of a tile in LDS, of STEPS k steps of 32 (64 bytes each), and what its 16-byte
// chunks are exchanged with: the rows that one read touches together differ in bits 0, 1
// and 3.
template <int STEPS>
struct RowTile {
  static constexpr int PITCH = STEPS * 64, CHUNKS = STEPS * 4;
  __device__ static __forceinline__ int turn(int row) {
    if constexpr (STEPS == 1) return ((row >> 1) & 1) | ((row >> 2) & 2);
    if constexpr (STEPS == 2) return (row & 3) | ((row >> 1) & 4);
    return ((row & 3) | ((row >> 1) & 4)) << 1;
  }
  template <typename E, int ROWS>
  __device__ static __forceinline__ void load(char* lds, const E* p, int64_t pitch, int64_t m0,
                                              int64_t rows, int32_t cols8, int waves) {
    constexpr int PER = 64 / CHUNKS;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (int j = wave; j < ROWS / PER; j += waves) {
      const int first = j * PER;
      const int64_t left = rows - m0 - first;
      const rsrc_t r = buffer_of(
          p + (m0 + first) * pitch,
          left > 0 ? (uint32_t)(((left < PER ? left : PER) - 1) * pitch + cols8) * 2 : 0);
      const int row = first + lane / CHUNKS, c = (lane % CHUNKS) ^ turn(row);
      uint32_t off = (uint32_t)(lane / CHUNKS * pitch + c * 8) * 2;
      if (c * 8 >= cols8) off = MX_OUTSIDE;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)(lds + first * PITCH), 16, off, 0, 0, 0);
    }
  }
  // Rows first: tile t of the 32 rows from `row` on, dealt as a chunk's hidden columns are.
  template <typename E>
  __device__ static __forceinline__ frag_t<E> rows(const char* lds, int row, int t, int k) {
    const int lane = threadIdx.x & 63;
    const int r = row + dealt(0, t, lane & 15);
    return *(const frag_t<E>*)(lds + r * PITCH + ((k * 4 + (lane >> 4)) ^ turn(r)) * 16);
  }
  // Columns first: 16 columns from `col` on by the 32 rows.
  template <typename E>
  __device__ static __forceinline__ frag_t<E> columns(const char* lds, int row, int col) {
    const int lane = threadIdx.x & 63;
    const int r = row + (lane >> 4) * 8 + ((lane >> 2) & 3), c = (col >> 3) + ((lane >> 1) & 1);
    typedef short s4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s4 lds_s4;
    const char* at = lds + (lane & 1) * 8;
    union {
      s4 h[2];
      frag_t<E> f;
    } u;
    u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(at + r * PITCH + (c ^ turn(r)) * 16));
    u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds_s4*)(at + (r + 4) * PITCH + (c ^ turn(r + 4)) * 16));
    return u.f;
  }
};

// Wavefronts of a workgroup at most: two a SIMD, or one with twice the registers where three
// planes of more than 128 columns of x and dy together need them.
template <typename T, int DK, int OK>
constexpr int weight_waves() {
  return Planes<T>::N == 3 && DK + OK > 4 ? 4 : FR_WAVES;
}

template <typename T>
constexpr int weight_rows() {  // of a staged tile
  return Planes<T>::N == 1 ? 64 : 32;
}

// DX: the wavefronts of a workgroup that takes dx along (0: it does not).  It holds every
// hidden column, so dg and du of 32 rows, exchanged through LDS, are all that dx of these
// rows wants: tiles of 16 rows and columns, dealt over the wavefronts.  Wg' and Wu' stay in
// LDS.  Of 1M rows of 64-256-64 bfloat16 that saves the hidden products, the gate and the
// reads of x and dy that a kernel of its own for dx repeats.  FULL: they have a hidden column
// each (32 DX of them); a loop of known length over these spills less (1M rows of 64-256-64:
// 545 us against 566, both directions).
template <typename T, int DK, int OK, int FT, int ACT, int DX, bool FULL>
__global__ void __launch_bounds__((64 * (DX ? DX : weight_waves<T, DK, OK>())), (DX ? 2 : 1))
    ffn_rows_dw_kernel(WeightArgs<T> a) {
  using E = typename Planes<T>::E;
  constexpr int P = Planes<T>::N, DT = 2 * DK, OT = 2 * OK, ROWS = weight_rows<T>();
  using X = RowTile<DK>;
  using Y = RowTile<OK>;
  constexpr int XB = ROWS * X::PITCH, YB = ROWS * Y::PITCH, BYTES = P * (XB + YB);
  using C = BackwardChunk<T, DK, OK>;
  // dg, then du, by hidden columns: of a tile's rows, or of half of them where that lets two
  // workgroups share a CU
  constexpr int EXCHANGED = DX == 8 ? 64 : 32;
  using G = RowTile<EXCHANGED / 32>;
  constexpr int COLUMNS = DX * 16 * FT, WB = 2 * DT * 1024;  // WB: Wg' and Wu' of 32 columns
  static_assert(!DX || (P == 1 && FT == 2), "a wavefront's hidden columns are a chunk");
  __shared__ __attribute__((aligned(1024))) char
      lds[2 * BYTES + DX * WB + (DX ? 2 * COLUMNS * G::PITCH : 0)];
  const int lane = threadIdx.x & 63, waves = blockDim.x >> 6;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int f0 = (blockIdx.y * waves + wave) * 16 * FT;
  const bool sum_dy = a.dy_sums && blockIdx.y == 0;
  const int width8 = (a.width + 7) & ~7, out8 = (a.out + 7) & ~7;

  frag_t<E> wg[FT][DK][P], wu[FT][DK][P], wd[FT][OK][P];
  float bg[FT], bu[FT];
#pragma unroll
  for (int i = 0; i < FT; ++i) {
    const int f = f0 + i * 16 + (lane & 15);
    const bool live = f < a.hidden;
    bg[i] = a.bg && live ? to_f32(a.bg[f]) : 0.f;
    bu[i] = a.bu && live ? to_f32(a.bu[f]) : 0.f;
#pragma unroll
    for (int k = 0; k < DK; ++k) {
      const int c = k * 32 + (lane >> 4) * 8;
      load_fragment<T>(a.wg + (int64_t)f * a.width, c, a.width, live, false, wg[i][k]);
      load_fragment<T>(a.wu + (int64_t)f * a.width, c, a.width, live, false, wu[i][k]);
    }
#pragma unroll
    for (int k = 0; k < OK; ++k)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int o = k * 32 + (lane >> 4) * 8 + j;
        E p[P];
        split<T>(live && o < a.out ? to_f32(a.wd[(int64_t)o * a.hidden + f]) : 0.f, p);
#pragma unroll
        for (int s = 0; s < P; ++s) wd[i][k][s][j] = p[s];
      }
  }
  f32x4 dwg[FT][DT] = {}, dwu[FT][DT] = {}, dwd[FT][OT] = {};
  float dys[8] = {};  // of eight columns of dy, over every blockDim.x / Y::CHUNKS-th row
  float sg[FT] = {}, su[FT] = {};
  Lift lift;
  if constexpr (LIFTED<T>) lift = *a.lift;
  const int64_t tiles = (a.rows + ROWS - 1) / ROWS;
  const auto stage = [&](int64_t tile, char* to) {
#pragma unroll
    for (int s = 0; s < P; ++s) {
      X::template load<E, ROWS>(to + s * XB, a.x.p + s * a.x.plane, a.x.pitch, tile * ROWS, a.rows,
                                width8, waves);
      Y::template load<E, ROWS>(to + P * XB + s * YB, a.dy.p + s * a.dy.plane, a.dy.pitch,
                                tile * ROWS, a.rows, out8, waves);
    }
  };
  if (blockIdx.x < tiles) stage(blockIdx.x, lds);
  char* const wx = lds + 2 * BYTES;
  char* const exchange = wx + DX * WB;
  if (DX && blockIdx.x < tiles)
    for (int c = 0; c < a.chunks; ++c)
      copy_chunk<WB / 1024, DX ? DX : 1>(wx + c * WB, a.packed + ((int64_t)c * C::KB + 4 * DK + 2 * OK) * 1024);
  // dx of the exchanged rows, from m0 on: a wavefront takes 16 of them by 32 columns.
  const auto take_dx = [&](int64_t m0) {
    for (int q = wave; q < DK * EXCHANGED / 16; q += DX) {
      const int m16 = q % (EXCHANGED / 16) * 16, d = q / (EXCHANGED / 16) * 2;
      f32x4 v[2] = {};  // (in the order of the kernel that takes dx alone)
      const auto add = [&](int c, auto whole) {
        const frag_t<E>* w = (const frag_t<E>*)(wx + c * WB + d * 1024) + lane;
        frag_t<E> g[P], u[P];
        g[0] = G::template columns<E>(exchange, c * 32, m16);
        u[0] = G::template columns<E>(exchange, COLUMNS + c * 32, m16);
        if constexpr (!whole.value) {
          keep_hidden<E, P>(g, a.hidden - c * 32);
          keep_hidden<E, P>(u, a.hidden - c * 32);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) v[i] = mfma32(w[i * 64], g[0], v[i]);
#pragma unroll
        for (int i = 0; i < 2; ++i) v[i] = mfma32(w[(DT + i) * 64], u[0], v[i]);
      };
      const int whole = FULL ? DX : a.hidden / 32;
#pragma unroll 4
      for (int c = 0; c < whole; ++c) add(c, std::true_type());
      if (!FULL && whole < a.chunks) add(whole, std::false_type());
      const int64_t m = m0 + m16 + (lane & 15);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int n = (d + i) * 16 + (lane >> 4) * 4;
        if constexpr (LIFTED<T>) v[i] *= lift.back_d;
        if (m < a.rows && n < a.width) put_four(a.dx + m * a.width + n, v[i], a.width - n, a.wide_dx);
      }
    }
  };
  int turn = 0;
  for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x, turn ^= 1) {
    stage_barrier();  // the tile is there, and nobody reads the one before it
    const char* xs = lds + turn * BYTES;
    const char* ys = xs + P * XB;
    if (tile + gridDim.x < tiles) stage(tile + gridDim.x, lds + (turn ^ 1) * BYTES);
    if (sum_dy)
      for (int row = threadIdx.x / Y::CHUNKS; row < ROWS; row += blockDim.x / Y::CHUNKS)
#pragma unroll
        for (int s = P - 1; s >= 0; --s) {
          const int c = (threadIdx.x % Y::CHUNKS) ^ Y::turn(row);
          const frag_t<E> v = *(const frag_t<E>*)(ys + s * YB + row * Y::PITCH + c * 16);
#pragma unroll
          for (int j = 0; j < 8; ++j) dys[j] += (float)v[j];
        }
    if (!DX && f0 >= a.hidden) continue;
#pragma unroll 1
    for (int row = 0; row < ROWS; row += 32) {
      frag_t<E> dg[FT][P], du[FT][P], h[FT][P];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        f32x4 g[FT], u[FT], dh[FT] = {};
#pragma unroll
        for (int i = 0; i < FT; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) g[i][r] = bg[i], u[i][r] = bu[i];
#pragma unroll
        for (int k = 0; k < DK; ++k) {
          frag_t<E> x[P];
#pragma unroll
          for (int s = 0; s < P; ++s) x[s] = X::template rows<E>(xs + s * XB, row, t, k);
#pragma unroll
          for (int i = 0; i < FT; ++i) {
            g[i] = mfma_planes<T>(x, wg[i][k], g[i]);
            u[i] = mfma_planes<T>(x, wu[i][k], u[i]);
          }
        }
#pragma unroll
        for (int k = 0; k < OK; ++k) {
          frag_t<E> y[P];
#pragma unroll
          for (int s = 0; s < P; ++s) {
            y[s] = Y::template rows<E>(ys + s * YB, row, t, k);
            if (P == 3 && t) y[s] = negated<E>(y[s]);
          }
#pragma unroll
          for (int i = 0; i < FT; ++i) dh[i] = mfma_planes<T>(y, wd[i][k], dh[i]);
        }
#pragma unroll
        for (int i = 0; i < FT; ++i) {
          float vg[4], vu[4], vh[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float2 v = activation<ACT, T>(g[i][r]);
            float d = P == 3 && t ? -dh[i][r] : dh[i][r];
            if constexpr (LIFTED<T>) d *= lift.d;
            vg[r] = d * u[i][r] * v.y;
            vu[r] = d * v.x;
            vh[r] = v.x * u[i][r];
            if constexpr (LIFTED<T>) vh[r] *= lift.h;
            sg[i] += vg[r];
            su[i] += vu[r];
          }
          four_t<E> p[P];
          split4<T>(vg, p);
          set_half<E, P>(dg[i], t, p);
          split4<T>(vu, p);
          set_half<E, P>(du[i], t, p);
          split4<T>(vh, p);
          set_half<E, P>(h[i], t, p);
        }
      }
      if constexpr (DX > 0) {
        if (row && EXCHANGED < ROWS) lds_barrier();  // nobody reads those of the rows before
#pragma unroll
        for (int i = 0; i < FT; ++i) {
          const int f = wave * 16 * FT + i * 16 + (lane & 15);
          char* at = exchange + f * G::PITCH +
                     (((EXCHANGED == 64 ? row / 8 : 0) + (lane >> 4)) ^ G::turn(f)) * 16;
          *(frag_t<E>*)at = dg[i][0];
          *(frag_t<E>*)(at + COLUMNS * G::PITCH) = du[i][0];
        }
      }
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        frag_t<E> x[P];
#pragma unroll
        for (int s = 0; s < P; ++s) x[s] = X::template columns<E>(xs + s * XB, row, d * 16);
#pragma unroll
        for (int i = 0; i < FT; ++i) {
          dwg[i][d] = mfma_planes<T>(x, dg[i], dwg[i][d]);
          dwu[i][d] = mfma_planes<T>(x, du[i], dwu[i][d]);
        }
      }
#pragma unroll
      for (int o = 0; o < OT; ++o) {
        frag_t<E> y[P];
#pragma unroll
        for (int s = 0; s < P; ++s) y[s] = Y::template columns<E>(ys + s * YB, row, o * 16);
#pragma unroll
        for (int i = 0; i < FT; ++i) dwd[i][o] = mfma_planes<T>(h[i], y, dwd[i][o]);
      }
      if constexpr (DX && EXCHANGED < ROWS) {
        lds_barrier();  // dg and du are there
        take_dx(tile * ROWS + row);
      }
    }
    if constexpr (DX && EXCHANGED == ROWS) {
      lds_barrier();
      take_dx(tile * ROWS);
    }
  }

  const auto put = [&](float* at, float v) { *at = a.add ? *at + v : v; };
  float* gu_part = a.dwgu + (int64_t)blockIdx.x * 2 * a.hidden * a.width;
  float* d_part = a.dwd + (int64_t)blockIdx.x * a.out * a.hidden;
  float* s_part = a.sums + (int64_t)blockIdx.x * 2 * a.hidden;
#pragma unroll
  for (int i = 0; i < FT; ++i) {
    const int f = f0 + i * 16 + (lane & 15);
    sg[i] += __shfl_xor(sg[i], 16, 64);
    sg[i] += __shfl_xor(sg[i], 32, 64);
    su[i] += __shfl_xor(su[i], 16, 64);
    su[i] += __shfl_xor(su[i], 32, 64);
    if (lane < 16 && f < a.hidden) {
      put(s_part + f, sg[i]);
      put(s_part + a.hidden + f, su[i]);
    }
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int n = d * 16 + (lane >> 4) * 4 + r;
        if (f < a.hidden && n < a.width) {
          put(gu_part + (int64_t)f * a.width + n, dwg[i][d][r]);
          put(gu_part + (int64_t)(a.hidden + f) * a.width + n, dwu[i][d][r]);
        }
      }
#pragma unroll
    for (int o = 0; o < OT; ++o) {
      const int n = o * 16 + (lane & 15);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int ff = f0 + i * 16 + (lane >> 4) * 4 + r;
        if (n < a.out && ff < a.hidden) put(d_part + (int64_t)n * a.hidden + ff, dwd[i][o][r]);
      }
    }
  }
  if (sum_dy) {
    float* sum = (float*)lds;  // [blockDim.x / Y::CHUNKS][Y::CHUNKS * 8]
    stage_barrier();
#pragma unroll
    for (int j = 0; j < 8; ++j) sum[threadIdx.x * 8 + j] = dys[j];
    __syncthreads();
    for (int n = threadIdx.x; n < a.out; n += blockDim.x) {
      float v = 0.f;
      for (int r = n; r < (int)blockDim.x * 8; r += Y::CHUNKS * 8) v += sum[r];
      put(a.dy_sums + (int64_t)blockIdx.x * a.out + n, v);
    }
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

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
bool RowKernels<T>::takes(int32_t width, int32_t out) {
  return width <= NARROW && out <= NARROW;
}

// Calls f(DK, OK) as constants.
template <typename F>
static void with_narrow_back(int width, int out, F&& f) {
  const auto by_out = [&](auto dk) {
    if (out <= 32) return f(dk, std::integral_constant<int, 1>());
    if (out <= 64) return f(dk, std::integral_constant<int, 2>());
    return f(dk, std::integral_constant<int, 4>());
  };
  if (width <= 32) return by_out(std::integral_constant<int, 1>());
  if (width <= 64) return by_out(std::integral_constant<int, 2>());
  return by_out(std::integral_constant<int, 4>());
}

// Values that the partial sums of rows of `cols` may take, however the chunks are dealt.
static int64_t partial_values(int64_t rows, int64_t cols, int64_t hidden) {
  return std::min(rows * std::max<int64_t>(1, tiles(hidden, 32) / 4),
                  (int64_t)SPLIT_TILES * 16 * FR_WAVES) * cols;
}

#define ROW_PASS (1 << 20)  // rows whose x and dy are laid out at a time
// Rows of one launch of the kernels that take tiles of 128 rows on: a launch has less than 2^32
// threads, four a row.
#define ROW_LAUNCH (1 << 29)

// The backward's workspace.
template <typename T, int DK, int OK>
struct RowPlan {
  using E = typename Planes<T>::E;
  static constexpr int FT = Planes<T>::N == 1 && DK <= 2 && OK <= 2 ? 2 : 1;
  int64_t pass;
  int waves, columns, runs;  // of a workgroup; workgroups along hidden and along rows
  char* packed;
  E *x, *dy;
  float *parts, *dwgu, *dwd, *sums, *dy_sums;  // parts: of dx
  Lift* lift = nullptr;  // half's
  float* peaks = nullptr;
  uint64_t bytes;
  RowPlan(void* ws, int64_t rows, int64_t width, int64_t hidden, int64_t out) {
    constexpr int P = Planes<T>::N;
    pass = std::min<int64_t>(rows, ROW_PASS);
    const int64_t slices = tiles(hidden, 16 * FT);
    waves = (int)std::min<int64_t>(slices, weight_waves<T, DK, OK>());
    columns = (int)tiles(slices, waves);
    // workgroups that the chip holds at once, whole ones a CU (500k rows of 64-224-64: 7
    // wavefronts each, 256 workgroups; 292 of them left a second round to 36)
    runs = (int)std::max<int64_t>(
        1, std::min<int64_t>(tiles(pass, weight_rows<T>()), 256 * (weight_waves<T, DK, OK>() / waves) / columns));
    Carver c{(char*)ws};
    packed = c.take<char>(BackwardChunk<T, DK, OK>::KB * 1024 * tiles(hidden, 32));
    x = c.take<E>(P * pass * round8(width));
    dy = c.take<E>(P * pass * round8(out));
    parts = c.take<float>(partial_values(rows, width, hidden));
    dwgu = c.take<float>(runs * 2 * hidden * width);
    dwd = c.take<float>(runs * hidden * out);
    sums = c.take<float>(runs * 2 * hidden);
    dy_sums = c.take<float>(runs * out);
    if (LIFTED<T>) {
      lift = c.take<Lift>(1);
      peaks = c.take<float>(LIFT_PEAKS);
    }
    bytes = c.used;
  }
};

template <typename T>
uint64_t RowKernels<T>::workspace(int64_t rows, int32_t width, int32_t hidden, int32_t out,
                                  bool back) {
  uint64_t bytes = 0;
  if (back)
    with_narrow_back(width, out, [&](auto dk, auto ok) {
      bytes = RowPlan<T, dk.value, ok.value>(nullptr, rows, width, hidden, out).bytes;
    });
  else
    with_narrow(width, out, [&](auto dk, auto ot) {
      bytes = ForwardChunk<T, dk.value, ot.value>::KB * 1024 * tiles(hidden, 32) +
              partial_values(rows, out, hidden) * sizeof(float);
    });
  return bytes;
}

// Whether rows can be read 16 bytes at a time.
template <typename T>
static bool wide_rows(const void* p, int64_t cols, int64_t pitch) {
  return cols % Vec16<T>::N == 0 && aligned16((const T*)p, pitch);
}
template <typename T>
static bool wide_stores(const void* p, int64_t cols) {
  return cols % 4 == 0 && aligned16((const T*)p, 0);
}

// Wavefronts take 16 RT rows (a constant) where such fill the chip, 16 where they do not.
// Where even those leave CUs idle, the chunks of the hidden columns are dealt over
// several workgroups, whose partial sums a further launch joins (1000 rows of 64-4096-64:
// one workgroup walks 128 chunks in 65 us).
template <int RT, typename F>
static void with_rows(int64_t rows, int chunks, F&& f) {
  const auto launch = [&](auto rt) {
    const int64_t groups = tiles(rows, 16 * rt.value * FR_WAVES);
    f(rt, dim3((unsigned)groups, rt.value == RT && RT > 1 ? 1 : split_parts(groups, chunks)));
  };
  if (rows >= 16 * RT * FR_WAVES * 256)
    launch(std::integral_constant<int, RT>());
  else
    launch(std::integral_constant<int, 1>());
}

template <typename T>
void RowKernels<T>::forward(const FfnCall& c, void* workspace, hipStream_t stream) {
  const int chunks = (int)tiles(c.hidden, 32);
  with_narrow(c.width, c.out, [&](auto dk, auto ot) {
    constexpr int DK = dk.value, OT = ot.value;
    using C = ForwardChunk<T, DK, OT>;
    const PackArgs pack{c.wg, c.wu, c.wd, c.bg, c.bu, (char*)workspace, c.width, c.hidden, c.out,
                        DK, OT, 0, C::KB};
    hipLaunchKernelGGL((ffn_pack_kernel<T, false>), dim3(chunks * (C::FRAGMENTS + 1)), dim3(64), 0,
                       stream, pack);
    float* parts = (float*)((char*)workspace + C::KB * 1024 * chunks);
    // 32 rows share a fragment's reads, 16 leave room for a second workgroup: 500k rows
    // bfloat16 of 32-128-16: 27 and 30 us, 64-256-64: 77 and 76, 128-256-128: 191 and 145;
    // 300k rows float32 of 59-128-3: 114 and 96
    constexpr int RT = Planes<T>::N == 1 && DK <= 2 ? 2 : 1;
    for (int64_t r = 0; r < c.rows; r += ROW_LAUNCH) {
      const int64_t m = std::min<int64_t>(ROW_LAUNCH, c.rows - r);
      T* const y = (T*)c.y + r * c.out;
      ForwardArgs<T> a{(const T*)row_at<T>(c.x, r, c.x_pitch), y, (const char*)workspace,
                       (const T*)c.bd, m, c.x_pitch, c.width, c.out, chunks, c.hidden, nullptr,
                       wide_rows<T>(c.x, c.width, c.x_pitch), wide_stores<T>(c.y, c.out)};
      with_rows<RT>(m, chunks, [&](auto rt, dim3 grid) {
        if (grid.y > 1) a.parts = parts;
        with_activation(c.act, [&](auto act) {
          hipLaunchKernelGGL((ffn_rows_fwd_kernel<T, DK, OT, rt.value, act.value>), grid,
                             dim3(64 * FR_WAVES), 0, stream, a);
        });
        if (grid.y > 1) {
          Joiner<T> join;
          join.add(parts, m * c.out, c.out, grid.y, m, c.out, y, c.bd);
          join.launch(stream);
        }
      });
    }
  });
}

template <typename T>
void RowKernels<T>::backward(const FfnCall& c, void* workspace, hipStream_t stream) {
  with_narrow_back(c.width, c.out, [&](auto dk, auto ok) {
    constexpr int DK = dk.value, OK = ok.value;
    using C = BackwardChunk<T, DK, OK>;
    const RowPlan<T, DK, OK> p(workspace, c.rows, c.width, c.hidden, c.out);
    const int chunks = (int)tiles(c.hidden, 32);
    const bool weights = c.dwg || c.dwu || c.dwd || c.dbg || c.dbu || c.dbd;
    if (!c.dx && !weights) return;
    if (LIFTED<T>) ffn_lift(c, p.lift, p.peaks, stream);
    // dx with the weights' gradients where a workgroup of four or eight wavefronts has all hidden
    // columns (with one or two, most of its wavefronts would have none).  bfloat16, against two
    // kernels, with the weights' layout and the joins: 1M rows of 64-256-64 407 and 503 us,
    // 64-128-64 264 and 300; 500k of 32-256-32 147 and 178, 64-192-64 227 and 240, 64-160-64 218
    // and 218, 64-100-64 152 and 160
    constexpr bool ALONGSIDE = RowPlan<T, DK, OK>::FT == 2;
    const bool alongside = ALONGSIDE && c.dx && weights && p.columns == 1 && p.waves > 2;
    if (c.dx) {
      const PackArgs pack{c.wg, c.wu, c.wd, c.bg, c.bu, p.packed, c.width, c.hidden, c.out,
                          DK, 0, OK, C::KB};
      hipLaunchKernelGGL((ffn_pack_kernel<T, true>), dim3(chunks * (C::FRAGMENTS + 1)), dim3(64), 0,
                         stream, pack);
    }
    if (c.dx && !alongside) {
      // 500k rows bfloat16, 32 and 16 rows a wavefront: 128-256-128 244 and 281 us, 64-256-64
      // 115 and 108; float32 with 16 rows and one chunk buffer, where two workgroups share
      // a CU, against 32 and two: 300k of 59-128-3 147 and 175 us
      constexpr int RT = Planes<T>::N == 3 ? 1 : 2;
      for (int64_t r = 0; r < c.rows; r += ROW_LAUNCH) {
        const int64_t m = std::min<int64_t>(ROW_LAUNCH, c.rows - r);
        T* const dx = (T*)c.dx + r * c.width;
        BackwardArgs<T> a{(const T*)row_at<T>(c.x, r, c.x_pitch), (const T*)row_at<T>(c.dy, r, c.dy_pitch),
                          dx, p.packed, m, c.x_pitch, c.dy_pitch, c.width, c.out, chunks, c.hidden,
                          nullptr, wide_rows<T>(c.x, c.width, c.x_pitch),
                          wide_rows<T>(c.dy, c.out, c.dy_pitch), wide_stores<T>(c.dx, c.width), p.lift};
        with_rows<RT>(m, chunks, [&](auto rt, dim3 grid) {
          if (grid.y > 1) a.parts = p.parts;
          with_activation(c.act, [&](auto act) {
            hipLaunchKernelGGL((ffn_rows_dx_kernel<T, DK, OK, rt.value, act.value>), grid,
                               dim3(64 * FR_WAVES), 0, stream, a);
          });
          if (grid.y > 1) {
            Joiner<T> join;
            join.add(p.parts, m * c.width, c.width, grid.y, m, c.width, dx);
            join.launch(stream);
          }
        });
      }
    }
    if (!weights) return;
    Layer<T> lay;
    for (int64_t r = 0; r < c.rows; r += p.pass) {
      const int64_t m = std::min(p.pass, c.rows - r);
      WeightArgs<T> a{};
      a.x = lay.operand(row_at<T>(c.x, r, c.x_pitch), m, c.width, c.x_pitch, p.x);
      a.dy = lay.operand(row_at<T>(c.dy, r, c.dy_pitch), m, c.out, c.dy_pitch, p.dy);
      lay.launch(stream);
      a.wg = (const T*)c.wg, a.wu = (const T*)c.wu, a.wd = (const T*)c.wd;
      a.bg = (const T*)c.bg, a.bu = (const T*)c.bu;
      a.dwgu = p.dwgu, a.dwd = p.dwd, a.sums = p.sums, a.dy_sums = c.dbd ? p.dy_sums : nullptr;
      a.rows = m, a.width = c.width, a.hidden = c.hidden, a.out = c.out, a.add = r > 0;
      a.dx = c.dx ? (T*)c.dx + r * c.width : nullptr;
      a.packed = p.packed, a.chunks = chunks, a.wide_dx = wide_stores<T>(c.dx, c.width);
      a.lift = p.lift;
      const auto launch = [&](auto dx, auto full, int waves) {
        with_activation(c.act, [&](auto act) {
          hipLaunchKernelGGL((ffn_rows_dw_kernel<T, DK, OK, RowPlan<T, DK, OK>::FT, act.value, dx.value,
                                                 full.value>),
                             dim3(p.runs, p.columns), dim3(64 * waves), 0, stream, a);
        });
      };
      if constexpr (ALONGSIDE) {
        if (alongside) {
          const auto with = [&](auto dx) {
            if (c.hidden == 32 * dx.value)
              launch(dx, std::true_type(), dx.value);
            else
              launch(dx, std::false_type(), dx.value);
          };
          if (p.waves <= 4)
            with(std::integral_constant<int, 4>());
          else
            with(std::integral_constant<int, 8>());
          continue;
        }
      }
      launch(std::integral_constant<int, 0>(), std::false_type(), p.waves);
    }
    const int64_t F = c.hidden, D = c.width, O = c.out;
    const float* const back_d = LIFTED<T> ? &p.lift->back_d : nullptr;
    const float* const back_h = LIFTED<T> ? &p.lift->back_h : nullptr;
    Joiner<T> join;
    join.add(p.dwgu, 2 * F * D, D, p.runs, F, D, c.dwg, nullptr, back_d);
    join.add(p.dwgu + F * D, 2 * F * D, D, p.runs, F, D, c.dwu, nullptr, back_d);
    join.add(p.dwd, O * F, F, p.runs, O, F, c.dwd, nullptr, back_h);
    join.add(p.sums, 2 * F, F, p.runs, 1, F, c.dbg, nullptr, back_d);
    join.add(p.sums + F, 2 * F, F, p.runs, 1, F, c.dbu, nullptr, back_d);
    join.add(p.dy_sums, O, O, p.runs, 1, O, c.dbd);
    join.launch(stream);
  });
}
