// Matrix products on the matrix cores: a workgroup's tile of C[m, n] = sum_k A[m, k] B[n, k]
// in 32-bit accumulators.
//
// Operands are bfloat16 or half matrices ("planes") whose rows start on 16 bytes and are
// a whole number of 8-value chunks.  An operand's k may run along its rows (ALONG: row
// m holds its k's side by side) or across them (ACROSS: row k holds its m's side by
// side); both are staged as they lie, and an ACROSS operand is turned while it is read
// from LDS (the transposing 64-bit LDS read), so no product needs a transposed copy.
//
// 32-bit operands come as three bfloat16 planes hi + mid + lo = the value (each what the ones
// before it leave, rounded: exact) and are multiplied as six products of planes: hi lo,
// lo hi, mid mid, mid hi, hi mid, hi hi.  The three left out come to 2^-24 of the product at most
// (mid is below 2^-8 of the value and lo below 2^-17), to 2^-27 of it on the average.
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

// The matrix cores drop what lies below their accumulators' last bit, towards minus
// infinity: 2^-27 of a product, always the same way.  Sums over rows that cancel to the
// square root of their number gather it (db of 300k rows was off by 3.6e-6 of itself,
// beside 3.3e-7 of a sum of 32-bit products).  Where such sums follow, every other row's
// operand is negated, and its product back, so that the two halves' drift cancels: 3.6e-7.
template <typename E>
__device__ __forceinline__ frag_t<E> negated(frag_t<E> f) {
  union {
    frag_t<E> f;
    i32x4 w;
  } u;
  u.f = f;
  u.w ^= (i32x4)(int)0x80008000;
  return u.f;
}

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

// Four values at once, as kernels split what they compute, two values a word.  A 32-bit value that
// is not finite, or within 2^-9 of the largest, comes out as NaN.
template <typename T>
__device__ __forceinline__ void split4(const float (&v)[4],
                                       four_t<typename Planes<T>::E> (&out)[Planes<T>::N]) {
  if constexpr (Planes<T>::N == 1) {
#pragma unroll
    for (int r = 0; r < 4; ++r) out[0][r] = (typename Planes<T>::E)v[r];
  } else {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef bf16_t bf16x2 __attribute__((ext_vector_type(2)));
    union {
      uint32_t w[2];
      bf16x2 p[2];
      four_t<bf16_t> f;
    } u;
    float rest[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
    for (int q = 0; q < 3; ++q) {
#pragma unroll
      for (int k = 0; k < 2; ++k)
        u.p[k] = __builtin_convertvector((f32x2{rest[2 * k], rest[2 * k + 1]}), bf16x2);
      out[q] = u.f;
      if (q < 2)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          rest[2 * k] -= __uint_as_float(u.w[k] << 16);
          rest[2 * k + 1] -= __uint_as_float(u.w[k] & 0xFFFF0000u);
        }
    }
  }
}

// The halves of fragments.
template <typename E, int P>
__device__ __forceinline__ void set_half(frag_t<E> (&f)[P], int half, const four_t<E> (&v)[P]) {
#pragma unroll
  for (int q = 0; q < P; ++q)
#pragma unroll
    for (int r = 0; r < 4; ++r) f[q][half * 4 + r] = v[q][r];
}

enum Along { ALONG, ACROSS };

// k of one staged step: of one plane, or of all three, which are multiplied in one step (each
// plane staged once for the six products that it takes part in).
template <typename T>
constexpr int stage_k() {
  return Planes<T>::N == 1 ? 64 : 32;
}

// A matrix operand: planes `plane` values apart, rows `pitch` values apart.
template <typename E>
struct Operand {
  const E* p;
  int64_t plane;
  int64_t pitch;
};

typedef __attribute__((address_space(3))) void lds_void;
typedef __amdgpu_buffer_rsrc_t rsrc_t;

#define MX_OUTSIDE 0x80000000u  // an offset past every buffer here
#define MX_PITCH (1 << 22)      // of an operand at most: 256 rows stay within such offsets

__device__ __forceinline__ rsrc_t buffer_of(const void* p, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)bytes, 0x00027000);
}

// ROWS of an operand by BK of its k, staged by the THREADS of a workgroup.  Where each
// lane reads is worked out once; a step moves the buffer's base.
template <typename E, int ROWS, Along K_, int THREADS, int BK>
struct Stage {
  static constexpr int BYTES = ROWS * BK * 2;
  static constexpr int WAVES = THREADS / 64;
  static constexpr int PASSES = BYTES / (1024 * WAVES);
  static_assert(PASSES * 1024 * WAVES == BYTES, "whole passes");
  static constexpr int CHUNKS = (K_ == ALONG ? BK : ROWS) / 8;  // of an LDS row
  static constexpr int PER = 64 / CHUNKS;                          // LDS rows of one KB
  static constexpr int READS = K_ == ALONG ? 1 : 2;                // LDS reads of a fragment

  // What a row's chunks (ALONG) or units of 32 bytes (ACROSS) are exchanged with, so that the
  // rows that one read touches together meet different banks: 16 in a row, or those that
  // differ in bits 0, 1 and 3.
  __device__ static __forceinline__ int turn(int row) {
    if constexpr (K_ == ALONG) return BK == 64 ? row & 7 : (row >> 2) & 3;
    if constexpr (ROWS >= 128) return (row & 3) | ((row >> 1) & 4);
    return ((row >> 1) & 1) | ((row >> 2) & 2);
  }

  int64_t pitch, K;
  uint32_t off[PASSES];  // bytes, from the tile's first row (ALONG) or column (ACROSS)
  uint32_t last;         // ALONG: bytes to the last row's start
  int chunk;             // ALONG: the chunk of this lane

  // The tile is rows row0 .. (ALONG; row r of it is row of(r) of the operand) or columns
  // row0 .. (ACROSS) of an operand that has `rows` of them; k runs to K.
  template <typename Of>
  __device__ __forceinline__ void begin(int64_t pitch_, int64_t row0, int64_t rows, int64_t K_end,
                                        Of&& of) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    pitch = pitch_;
    K = K_end;
    const int left = (int)min((int64_t)ROWS, rows - row0);
#pragma unroll
    for (int j = 0; j < PASSES; ++j) {
      const int row = (j * WAVES + wave) * PER + lane / CHUNKS, pos = lane % CHUNKS;
      if constexpr (K_ == ALONG) {
        chunk = pos ^ turn(row);
        const int r = of(row);
        off[j] = r < left ? (uint32_t)(r * pitch + chunk * 8) * 2 : MX_OUTSIDE;
      } else {
        const int c = (((pos >> 1) ^ turn(row)) << 1) | (pos & 1);
        off[j] = c * 8 < left ? (uint32_t)(row * pitch + c * 8) * 2 : MX_OUTSIDE;
      }
    }
    last = (uint32_t)((left - 1) * pitch) * 2;
  }
  __device__ __forceinline__ void begin(int64_t pitch_, int64_t row0, int64_t rows, int64_t K_end) {
    begin(pitch_, row0, rows, K_end, [](int r) { return r; });
  }

  // Starts the copies of k0 .. k0 + BK - 1; `p` is the tile's first row's or column's
  // place in the plane, p2 that of the rows that `other` says come from another matrix.
  __device__ __forceinline__ void copy(char* lds, const E* p, int64_t k0) const {
    copy(lds, p, p, k0, [](int) { return false; });
  }
  template <typename Other>
  __device__ __forceinline__ void copy(char* lds, const E* p, const E* p2, int64_t k0,
                                       Other&& other) const {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int left = (int)min((int64_t)BK, K - k0);
    const int64_t at = K_ == ALONG ? k0 : k0 * pitch;
    // ALONG: chunks that start before K are there whole (operands end on chunks)
    const uint32_t bytes = K_ == ALONG ? last + ((left + 7) & ~7) * 2 : (uint32_t)(left * pitch) * 2;
    const rsrc_t r = buffer_of(p + at, bytes), r2 = buffer_of(p2 + at, bytes);
    const bool whole = K_ == ACROSS || chunk * 8 < left;
#pragma unroll
    for (int j = 0; j < PASSES; ++j) {
      const int first = (j * WAVES + wave) * PER;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(other(first) ? r2 : r,
                                               (lds_void*)(lds + (j * WAVES + wave) * 1024), 16,
                                               whole ? off[j] : MX_OUTSIDE, 0, 0, 0);
    }
  }

  // The fragment of rows row .. row + 15 at k step kk (32 values).
  __device__ static __forceinline__ frag_t<E> fragment(const char* lds, int row, int kk) {
    const int lane = threadIdx.x & 63;
    if constexpr (K_ == ALONG) {
      const int r = row + (lane & 15), c = (kk * 4 + (lane >> 4)) ^ turn(lane & 15);
      return *(const frag_t<E>*)(lds + r * BK * 2 + c * 16);
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

// The steps of a product's loop: k in BK from `from` to `to`, for each of `pairs` pairs of
// operands in turn.
struct Steps {
  int64_t k, from, to;
  int pair, pairs, BK;
  __device__ __forceinline__ Steps(int BK_, int64_t from_, int64_t to_, int pairs_)
      : k(from_), from(from_), to(to_), pair(from_ < to_ ? 0 : pairs_), pairs(pairs_), BK(BK_) {}
  __device__ __forceinline__ bool more() const { return pair < pairs; }
  __device__ __forceinline__ void next() {
    k += BK;
    if (k >= to) k = from, ++pair;
  }
};

// A workgroup's tile: WM x WN wavefronts of TM x TN tiles of 16.
template <int WM_, int WN_, int TM_, int TN_>
struct Tile {
  static constexpr int WM = WM_, WN = WN_, TM = TM_, TN = TN_;
  static constexpr int THREADS = 64 * WM * WN, M = 16 * WM * TM, N = 16 * WN * TN;
};

// Behind it every wavefront's copies to LDS have landed and its LDS reads are done.  The wait
// is spelled out: __syncthreads() orders LDS accesses, and the compiler does not
// count the copies among them at every barrier.
__device__ __forceinline__ void stage_barrier() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Behind it every wavefront's LDS accesses are done; copies to LDS may still be on their way.
__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// The main loop: copy(step, plane, a, b) starts the copies of a step's planes of the operands
// to a and b in LDS.  acc[i][j] is the transposed 16 x 16 tile of rows a_row + 16 i of A and
// b_row + 16 j of B: lane l holds row l % 16 of A and rows (l / 16) * 4 + r of B.
// FLIP: the products of every other of A's tiles come out negated.
//
// One plane: two buffers.  A step is two halves of k = 32, and the fragments of the half to
// come are read while a half is multiplied, so the matrix cores have operands in registers
// across the barrier in the middle of the step: behind it the step's buffer is read out and
// takes the copies of the step after next, and the next step's copies have landed.
//
// Three planes: one buffer and two workgroups a CU, one copying while the other multiplies;
// a step's 96 products a wavefront outlast its copies.  Pair after pair of planes, each in
// steps of its own, staged every plane twice as often and took 219 us for the forward
// of 1000 rows 1024-4096-1024.
template <typename E, int P>
struct Loop;

template <typename E>
struct Loop<E, 1> {
  template <typename SA, typename SB>
  static constexpr int bytes() {
    return 2 * (SA::BYTES + SB::BYTES);
  }
  template <bool FLIP, typename SA, typename SB, int TM, int TN, typename Copy>
  __device__ static __forceinline__ void run(f32x4 (&acc)[TM][TN], char* lds, Steps ahead, int a_row,
                                             int b_row, Copy&& copy) {
    constexpr int BYTES = SA::BYTES + SB::BYTES;
    static_assert(!FLIP, "of three planes' loop");
    if (!ahead.more()) return;
    frag_t<E> a[2][TM], b[2][TN];
    const auto read = [&](const char* from, int half) {
#pragma unroll
      for (int i = 0; i < TM; ++i) a[half][i] = SA::fragment(from, a_row + i * 16, half);
#pragma unroll
      for (int j = 0; j < TN; ++j) b[half][j] = SB::fragment(from + SA::BYTES, b_row + j * 16, half);
    };
    const auto multiply = [&](int half) {
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = mfma32(b[half][j], a[half][i], acc[i][j]);
    };
    // the reads dealt evenly among the products
    const auto mix = [] {
      constexpr int READS = TM * SA::READS + TN * SB::READS, PRODUCTS = TM * TN;
      constexpr int GROUPS = READS < PRODUCTS ? READS : PRODUCTS;
#pragma unroll
      for (int i = 0; i < GROUPS; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, PRODUCTS / GROUPS, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, (READS + GROUPS - 1) / GROUPS, 0);
      }
    };
    char *cur = lds, *other = lds + BYTES;
    copy(ahead, 0, cur, cur + SA::BYTES);
    ahead.next();
    stage_barrier();
    if (ahead.more()) copy(ahead, 0, other, other + SA::BYTES);
    read(cur, 0);
    while (ahead.more()) {
      read(cur, 1);
      multiply(0);
      mix();
      stage_barrier();
      ahead.next();
      if (ahead.more()) copy(ahead, 0, cur, cur + SA::BYTES);
      char* t = cur;
      cur = other;
      other = t;
      read(cur, 0);
      multiply(1);
      mix();
    }
    read(cur, 1);
    multiply(0);
    multiply(1);
    stage_barrier();
  }
};

template <typename E>
struct Loop<E, 3> {
  template <typename SA, typename SB>
  static constexpr int bytes() {
    return 3 * (SA::BYTES + SB::BYTES);
  }
  template <bool FLIP, typename SA, typename SB, int TM, int TN, typename Copy>
  __device__ static __forceinline__ void run(f32x4 (&acc)[TM][TN], char* lds, Steps s, int a_row,
                                             int b_row, Copy&& copy) {
    char* to_b = lds + 3 * SA::BYTES;
    for (; s.more(); s.next()) {
#pragma unroll
      for (int q = 0; q < 3; ++q) copy(s, q, lds + q * SA::BYTES, to_b + q * SB::BYTES);
      stage_barrier();
      frag_t<E> a[3][TM], b[3][TN];
#pragma unroll
      for (int q = 2; q >= 0; --q) {
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          a[q][i] = SA::fragment(lds + q * SA::BYTES, a_row + i * 16, 0);
          if (FLIP && i % 2) a[q][i] = negated<E>(a[q][i]);
        }
#pragma unroll
        for (int j = 0; j < TN; ++j) b[q][j] = SB::fragment(to_b + q * SB::BYTES, b_row + j * 16, 0);
      }
      const auto multiply = [&](int pa, int pb) {
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int j = 0; j < TN; ++j) acc[i][j] = mfma32(b[pb][j], a[pa][i], acc[i][j]);
      };
      multiply(2, 0);  // the smallest first
      multiply(0, 2);
      multiply(1, 1);
      multiply(1, 0);
      multiply(0, 1);
      multiply(0, 0);
      stage_barrier();
    }
  }
};
