// Matrix products on the matrix cores: a workgroup's tile of C[m, n] = sum_k A[m, k] B[n, k]
// in 32-bit accumulators.
//
// Operands are bfloat16 or half matrices ("planes") whose rows start on 16 bytes and are
// a whole number of 8-value chunks.  An operand's k may run along its rows (ALONG: row
// m holds its k's side by side) or across them (ACROSS: row k holds its m's side by
// side); both are staged as they lie, and an ACROSS operand is turned while it is read
// from LDS (the transposing 64-bit LDS read), so no product needs a transposed copy.
//
// 32-bit operands come as three bfloat16 planes hi + mid + lo = the value (8 bits each,
// split exactly up to 2^-27 of it) and are multiplied as the six products of planes
// whose sum is off by less than 2^-25: hi lo, lo hi, mid mid, mid hi, hi mid, hi hi.
// Six bfloat16 products run at 1/6 of that type's rate, 2.7 times the 32-bit matrix
// instructions' (an 8192^3 product of the vendor's: 1307 and 132 TFLOP/s).
//
// The staging copies go from memory to LDS without registers, 16 bytes a lane, 1 KB a
// wavefront; LDS chunks are permuted by row so that the fragments' reads meet no bank
// twice.  Chunks past an operand's end read as zero through the buffer's bounds.
#pragma once

#include "decoder_common.cuh"

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
template <typename E>
using frag_t = E __attribute__((ext_vector_type(8)));
template <typename E>
using four_t = E __attribute__((ext_vector_type(4)));

// One 16 x 16 x 32 step.  Lane l holds row l % 16 of either operand at k = (l / 16) * 8 + i
// and column l % 16 (the second operand's row), rows (l / 16) * 4 + i of the result.
__device__ __forceinline__ f32x4 mfma32(frag_t<bf16_t> a, frag_t<bf16_t> b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma32(frag_t<f16_t> a, frag_t<f16_t> b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// The planes that hold a tensor's values: itself, or three of bfloat16.
template <typename T>
struct Planes {
  using E = T;
  static constexpr int N = 1;
};
template <>
struct Planes<float> {
  using E = bf16_t;
  static constexpr int N = 3;
};

// v = sum of p[0..N).  What is not finite stays so in the first plane alone.
template <typename T>
__device__ __forceinline__ void split(float v, typename Planes<T>::E (&p)[Planes<T>::N]) {
  p[0] = (typename Planes<T>::E)v;
  if constexpr (Planes<T>::N == 3) {
    const float hi = (float)p[0];
    const float r = fabsf(hi) < __builtin_inff() ? v - hi : 0.f;
    p[1] = (bf16_t)r;
    p[2] = (bf16_t)(r - (float)p[1]);
  }
}

// The pairs of planes that a product multiplies, the smallest first.
template <typename T>
struct PlanePairs {
  static constexpr int N = 1;
  __device__ static __forceinline__ int a(int) { return 0; }
  __device__ static __forceinline__ int b(int) { return 0; }
};
template <>
struct PlanePairs<float> {
  static constexpr int N = 6;
  __device__ static __forceinline__ int a(int i) { return (0x201100 >> (4 * (5 - i))) & 3; }
  __device__ static __forceinline__ int b(int i) { return (0x021010 >> (4 * (5 - i))) & 3; }
};

enum Along { ALONG, ACROSS };

#define MX_BK 64  // k of one staged step

// A matrix operand: planes `plane` values apart, rows `pitch` values apart.  k runs to
// K and the other index to N.
template <typename E>
struct Operand {
  const E* p;
  int64_t plane;
  int64_t pitch;
};

typedef __attribute__((address_space(3))) void lds_void;
typedef __amdgpu_buffer_rsrc_t rsrc_t;

#define MX_OUTSIDE 0x80000000u  // an offset past every buffer here

__device__ __forceinline__ rsrc_t buffer_of(const void* p, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)bytes, 0x00027000);
}

// ROWS of an operand by MX_BK of its k, staged by the THREADS of a workgroup.
template <typename E, int ROWS, Along K_, int THREADS>
struct Stage {
  static constexpr int BYTES = ROWS * MX_BK * 2;
  static constexpr int WAVES = THREADS / 64;
  static constexpr int PASSES = BYTES / (1024 * WAVES);
  static_assert(PASSES * 1024 * WAVES == BYTES, "whole passes");
  static constexpr int CHUNKS = (K_ == ALONG ? MX_BK : ROWS) / 8;  // of an LDS row

  // Which unit of 32 bytes an ACROSS row's units are exchanged with: rows that one
  // transposing read touches together (bits 0, 1 and 3) meet different banks.
  __device__ static __forceinline__ int turn(int row) {
    if constexpr (ROWS >= 128) return (row & 3) | ((row >> 1) & 4);
    return ((row >> 1) & 1) | ((row >> 2) & 2);
  }

  // `rows` of the operand are there (from row0 on), k runs from k0 to K.  Row r of the
  // tile is row of(r) of the operand, the same distance from r for r of a run of 8.
  template <typename Of>
  __device__ static __forceinline__ void load(char* lds, const E* p, int64_t pitch, int64_t row0,
                                              int64_t rows, int64_t k0, int64_t K, Of&& of) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if constexpr (K_ == ALONG) {
#pragma unroll
      for (int j = 0; j < PASSES; ++j) {
        const int first = (j * WAVES + wave) * 8;  // row of lane 0
        const auto src = of(first);
        const int64_t at = row0 + src.row;
        const int64_t left = rows - at;
        const rsrc_t r = buffer_of(src.p + at * pitch + k0,
                                   left > 0 ? (uint32_t)(((left < 8 ? left : 8) - 1) * pitch +
                                                         ((K + 7) & ~7) - k0) * 2 : 0);
        const int c = (lane & 7) ^ (lane >> 3);
        uint32_t off = (uint32_t)((lane >> 3) * pitch + c * 8) * 2;
        if (k0 + c * 8 >= K) off = MX_OUTSIDE;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)(lds + first * 128), 16, off, 0, 0, 0);
      }
    } else {
      // row0 is this tile's first column of the operand's rows, which are its k
      constexpr int PER = 64 / CHUNKS;  // k rows of one wavefront's KB
#pragma unroll
      for (int j = 0; j < PASSES; ++j) {
        const int first = (j * WAVES + wave) * PER;
        const int64_t left = K - k0 - first;
        const rsrc_t r =
            buffer_of(p + (k0 + first) * pitch + row0,
                      left > 0 ? (uint32_t)(((left < PER ? left : PER) - 1) * pitch + rows - row0) * 2 : 0);
        const int row = first + lane / CHUNKS, pos = lane % CHUNKS;
        const int c = (((pos >> 1) ^ turn(row)) << 1) | (pos & 1);
        uint32_t off = (uint32_t)((lane / CHUNKS) * pitch + c * 8) * 2;
        if (row0 + c * 8 >= rows) off = MX_OUTSIDE;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)(lds + first * ROWS * 2), 16, off, 0, 0, 0);
      }
    }
  }

  // The fragment of rows row .. row + 15 at k step kk (32 values).
  __device__ static __forceinline__ frag_t<E> fragment(const char* lds, int row, int kk) {
    const int lane = threadIdx.x & 63;
    if constexpr (K_ == ALONG) {
      const int r = row + (lane & 15), c = (kk * 4 + (lane >> 4)) ^ (lane & 7);
      return *(const frag_t<E>*)(lds + r * 128 + c * 16);
    } else {
      const int k = kk * 32 + (lane >> 4) * 8 + ((lane >> 2) & 3);
      const int unit = (row >> 4) ^ turn(k);
      const char* at = lds + k * ROWS * 2 + unit * 32 + (lane & 3) * 8;
      typedef short s4 __attribute__((ext_vector_type(4)));
      typedef __attribute__((address_space(3))) s4 lds_s4;
      union {
        s4 h[2];
        frag_t<E> f;
      } u;
      u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(at));
      u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(at + 4 * ROWS * 2));
      return u.f;
    }
  }
};

// Which row of which matrix a tile's row is (runs of 8).
template <typename E>
struct RowOf {
  const E* p;
  int64_t row;
};

// A tile's place among `tiles_m` x `tiles_n`: workgroups go round the 8 XCDs, so each XCD is
// given a contiguous run of the order, and the order walks 8 tiles of m for each of n, so
// that what an XCD works on at once shares its operands in that XCD's L2.
__device__ __forceinline__ void tile_of(uint32_t bid, uint32_t tiles_m, uint32_t tiles_n,
                                        uint32_t& tm, uint32_t& tn) {
  const uint32_t n = tiles_m * tiles_n, per = n / 8, more = n % 8;
  const uint32_t xcd = bid % 8, at = bid / 8;
  const uint32_t t = xcd * per + (xcd < more ? xcd : more) + at;
  const uint32_t group = t / (8 * tiles_n), in = t % (8 * tiles_n);
  const uint32_t high = tiles_m - group * 8 < 8 ? tiles_m - group * 8 : 8;
  tm = group * 8 + in % high;
  tn = in / high;
}

// The main loop over `steps` staged steps: load(step, buffer) starts the copies of a step,
// and a step is multiplied while the next one's copies run.  acc[i][j] is the transposed
// 16 x 16 tile of rows a_row + 16 i of A and b_row + 16 j of B: lane l holds row l % 16 of A and
// rows (l / 16) * 4 + r of B.
template <typename E, typename SA, typename SB, int TM, int TN, typename Load>
__device__ __forceinline__ void product_loop(f32x4 (&acc)[TM][TN], char* lds, int steps, int a_row,
                                             int b_row, Load&& load) {
  constexpr int BYTES = SA::BYTES + SB::BYTES;
  load(0, lds);
#pragma unroll 1
  for (int s = 0; s < steps; ++s) {
    // everyone's copies of this step are there, and nobody reads the other buffer any more
    __syncthreads();
    const char* cur = lds + (s & 1) * BYTES;
    if (s + 1 < steps) load(s + 1, lds + ((s + 1) & 1) * BYTES);
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      frag_t<E> a[TM], b[TN];
#pragma unroll
      for (int i = 0; i < TM; ++i) a[i] = SA::fragment(cur, a_row + i * 16, kk);
#pragma unroll
      for (int j = 0; j < TN; ++j) b[j] = SB::fragment(cur + SA::BYTES, b_row + j * 16, kk);
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = mfma32(b[j], a[i], acc[i][j]);
    }
  }
  __syncthreads();
}
