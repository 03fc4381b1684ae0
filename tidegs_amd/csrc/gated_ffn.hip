// Gated feed-forward block, forward and backward:
//
//   g = x Wg' + bg, u = x Wu' + bu, h = act(g) u, y = h Wd' + bd
//   dh = dy Wd, dg = dh u act'(g), du = dh act(g)
//   dx = dg Wg + du Wu, dWg = dg' x, dWu = du' x, dWd = dy' h, db. = column sums
//
// x [rows, width], Wg and Wu [hidden, width], Wd [out, hidden], row-major (x and dy at
// a pitch).  The backward computes g and u again.
#include "gated_ffn.cuh"

// ---------------------------------------------------------------------------
// The hidden products.  The B rows of a workgroup's tile are runs of 16 of Wg and of Wu in
// turn, so that a lane's accumulators hold g and u of the same row and columns and the gate
// is taken in registers.  The backward adds dh = dy Wd for the same tile before its gate.
//
// h, dg and du of 16-bit tensors are rounded to their type where they are written: they are
// what is stored between the products (200 MB at 8192 rows of 4096), and the matrix cores'
// operands have that type.  y is 0.0023 of itself off in bfloat16 then, 0.0017 from its own
// rounding.
//
// Bound by the matrix cores and what feeds them: at 8192 rows of 1024-4096-1024 bfloat16 the
// forward's hidden products take 124 us (1110 TFLOP/s), y 76 (900), the backward's three
// hidden products 264 (780, with 200 MB of h, dg and du written), dx 143 (960), dWg and dWu 137
// (1000), dWd 145 (470: 256 tiles, one workgroup a CU where two have room); a library product
// of 8192^3 reaches 1307.  g and u are computed again in the backward
// rather than kept: kept in 32 bits they are 268 MB to write and to read, about 120 us,
// for the 137 GFLOP (140 us) that they save.
// ---------------------------------------------------------------------------

// Tiles: 128 x 128 in four wavefronts, two workgroups a CU; 256 x 256 in eight, one a CU, for
// products of operands that both run along k, where there are tiles enough for the CUs.
// A larger tile stages fewer bytes per product and its wavefronts' 128 x 64 read fewer
// fragments: the hidden products of 8192 x 1024 x 2 4096 take 139 us in the large tiles, 161
// in the small. With an operand across k the turning reads, twice as
// many, leave the large tile's lockstep behind two small ones (dW of that block 175 us
// against 154), and so does the backward's third accumulator (343 against 305).  (Pairs of
// variants, here and below, are from runs of a few passes, at lower clocks than the times above.)
typedef Tile<2, 2, 4, 4> TileSmall;
typedef Tile<2, 4, 8, 4> TileLarge;

template <typename E>
struct HiddenArgs {
  Operand<E> x, wg, wu, dy, wd;
  int64_t rows;
  int32_t width8, hidden, hidden8, out, out8, act;
  const void *bg, *bu;
  E* h;     // h, plane by plane; backward: its pitch is hidden8 too
  E* dgu;   // dg | du at a pitch of 2 hidden8
  float* sums;  // of dg and du over a tile's rows: [tiles_m, 2 hidden8], nullable
  int64_t plane;  // values between planes of h; dgu's are 2 * plane
  int32_t add;    // add to sums
  const Lift* lift;  // half's, backward
};

template <typename T, bool BACK, typename Z>
__global__ void __launch_bounds__(Z::THREADS, 2) ffn_hidden_kernel(HiddenArgs<typename Planes<T>::E> a) {
  using E = typename Planes<T>::E;
  constexpr int P = Planes<T>::N, BK = stage_k<T>();
  constexpr int TM = Z::TM, TF = Z::TN / 2, F = Z::N / 2;  // hidden columns of the tile
  using SX = Stage<E, Z::M, ALONG, Z::THREADS, BK>;
  using SW = Stage<E, Z::N, ALONG, Z::THREADS, BK>;
  using SD = Stage<E, F, ACROSS, Z::THREADS, BK>;
  __shared__ __attribute__((aligned(1024))) char lds[Loop<E, P>::template bytes<SX, SW>()];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / Z::WN, wn = wave % Z::WN;
  uint32_t tm, tn;
  tile_of(blockIdx.x, (uint32_t)((a.rows + Z::M - 1) / Z::M), (a.hidden8 + F - 1) / F, tm, tn);
  const int64_t m0 = (int64_t)tm * Z::M;
  const int f0 = tn * F;

  f32x4 gu[TM][2 * TF] = {};
  {
    SX sx;
    SW sw;
    sx.begin(a.x.pitch, m0, a.rows, a.width8);
    sw.begin(a.wg.pitch, f0, a.hidden, a.width8, [](int r) { return (r >> 5) * 16 + (r & 15); });
    const E *x = a.x.p + m0 * a.x.pitch, *wg = a.wg.p + f0 * a.wg.pitch, *wu = a.wu.p + f0 * a.wu.pitch;
    Loop<E, P>::template run<false, SX, SW>(
        gu, lds, Steps(BK, 0, a.width8, 1), wm * TM * 16, wn * TF * 32,
        [&](const Steps& s, int q, char* to_x, char* to_w) {
          sx.copy(to_x, x + q * a.x.plane, s.k);
          sw.copy(to_w, wg + q * a.wg.plane, wu + q * a.wu.plane, s.k,
                  [](int r) { return (r & 16) != 0; });
        });
  }
  f32x4 dh[TM][TF] = {};
  if constexpr (BACK) {
    SX sy;
    SD sd;
    sy.begin(a.dy.pitch, m0, a.rows, a.out8);
    sd.begin(a.wd.pitch, f0, a.hidden8, a.out);
    const E *dy = a.dy.p + m0 * a.dy.pitch, *wd = a.wd.p + f0;
    Loop<E, P>::template run<P == 3, SX, SD>(
        dh, lds, Steps(BK, 0, a.out, 1), wm * TM * 16, wn * TF * 16,
        [&](const Steps& s, int q, char* to_y, char* to_w) {
          sy.copy(to_y, dy + q * a.dy.plane, s.k);
          sd.copy(to_w, wd + q * a.wd.plane, s.k);
        });
  }

  const int group = lane >> 4;
  float sg[TF][4] = {}, su[TF][4] = {};
  Lift lift;
  if constexpr (BACK && LIFTED<T>) lift = *a.lift;
  with_activation(a.act, [&](auto kind) {
#pragma unroll
  for (int j = 0; j < TF; ++j) {
    const int f = f0 + wn * TF * 16 + j * 16 + group * 4;
    float bg[4], bu[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      bg[r] = a.bg && f + r < a.hidden ? to_f32(((const T*)a.bg)[f + r]) : 0.f;
      bu[r] = a.bu && f + r < a.hidden ? to_f32(((const T*)a.bu)[f + r]) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int64_t m = m0 + wm * TM * 16 + i * 16 + (lane & 15);
      const bool live = m < a.rows && f < a.hidden8;
      float vh[4], vg[4], vu[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        // (behind the last hidden column zeros, whatever x holds)
        const bool in = f + r < a.hidden;
        const float g = gu[i][2 * j][r] + bg[r], u = gu[i][2 * j + 1][r] + bu[r];
        const float2 act = activation<kind.value, T>(g);
        vh[r] = in ? act.x * u : 0.f;
        if constexpr (BACK) {
          float d = P == 3 && i % 2 ? -dh[i][j][r] : dh[i][j][r];
          if constexpr (LIFTED<T>) {
            d *= lift.d;
            vh[r] *= lift.h;
          }
          vg[r] = in ? d * u * act.y : 0.f;
          vu[r] = in ? d * act.x : 0.f;
          if (m < a.rows) {
            sg[j][r] += vg[r];
            su[j][r] += vu[r];
          }
        }
      }
      four_t<E> h[P], dg[P], du[P];
      split4<T>(vh, h);
      if constexpr (BACK) {
        split4<T>(vg, dg);
        split4<T>(vu, du);
      }
      if (!live) continue;
#pragma unroll
      for (int q = 0; q < P; ++q) {
        *(four_t<E>*)(a.h + q * a.plane + m * a.hidden8 + f) = h[q];
        if constexpr (BACK) {
          E* at = a.dgu + 2 * (q * a.plane + m * a.hidden8) + f;
          *(four_t<E>*)at = dg[q];
          *(four_t<E>*)(at + a.hidden8) = du[q];
        }
      }
    }
  }
  });
  if constexpr (BACK) {
    if (!a.sums) return;
    float* s = (float*)lds;  // [WM][2][F]; the main loop's last barrier freed it
#pragma unroll
    for (int j = 0; j < TF; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
#pragma unroll
        for (int off = 1; off < 16; off <<= 1) {
          sg[j][r] += __shfl_xor(sg[j][r], off, 64);
          su[j][r] += __shfl_xor(su[j][r], off, 64);
        }
        if ((lane & 15) == 0) {
          const int f = wn * TF * 16 + j * 16 + group * 4 + r;
          s[(wm * 2) * F + f] = sg[j][r];
          s[(wm * 2 + 1) * F + f] = su[j][r];
        }
      }
    __syncthreads();
    if (threadIdx.x < 2 * F) {
      const int which = threadIdx.x / F, f = f0 + threadIdx.x % F;
      if (f < a.hidden8) {
        float* out = a.sums + ((int64_t)tm * 2 + which) * a.hidden8 + f;
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < Z::WM; ++w) v += s[w * 2 * F + threadIdx.x];
        *out = a.add ? *out + v : v;
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Plain products: C = A B' (+ bias), 128 x 128 tiles, either rounded to the call's type
// or, with the sum over k split, as 32-bit partial sums that a second launch joins.
// ---------------------------------------------------------------------------

template <typename E>
struct ProductArgs {
  Operand<E> a, b, a2, b2;  // a2, b2: a second pair (null: none)
  int64_t M, K;             // K: of each pair
  int32_t N;
  int64_t a_limit;          // A's other index runs to this (its columns where k runs across)
  int32_t b_limit;
  int32_t splits;           // of the steps over k
  const void* bias;
  void* c;                  // [M, N] of the call's type, or, of its first and second half of
  void* c2;                 // rows, `each` to c and to c2 (each: 0 or less than M / 2; null: left out)
  int64_t each;
  int32_t wide;             // c is written four values at a time
  float* partial;           // or [splits, M, N]
  int32_t add;              // add to what `partial` holds
  const float* factor;      // of c, half's; nullable
};

template <typename T, Along KA, Along KB, typename Z>
__global__ void __launch_bounds__(Z::THREADS, 2) ffn_product_kernel(ProductArgs<typename Planes<T>::E> g) {
  using E = typename Planes<T>::E;
  constexpr int P = Planes<T>::N, BK = stage_k<T>();
  constexpr int TM = Z::TM, TN = Z::TN;
  using SA = Stage<E, Z::M, KA, Z::THREADS, BK>;
  using SB = Stage<E, Z::N, KB, Z::THREADS, BK>;
  __shared__ __attribute__((aligned(1024))) char lds[Loop<E, P>::template bytes<SA, SB>()];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / Z::WN, wn = wave % Z::WN;
  const uint32_t tiles_m = (uint32_t)((g.M + Z::M - 1) / Z::M);
  const uint32_t tiles_n = (g.N + Z::N - 1) / Z::N;
  uint32_t tm, tn;
  const uint32_t split = blockIdx.x / (tiles_m * tiles_n);
  tile_of(blockIdx.x % (tiles_m * tiles_n), tiles_m, tiles_n, tm, tn);
  const int64_t m0 = (int64_t)tm * Z::M;
  const int n0 = tn * Z::N;
  const int64_t all = (g.K + BK - 1) / BK;
  const int64_t from = all * split / g.splits * BK;
  const int64_t to = min(all * (split + 1) / g.splits * BK, g.K);

  SA sa;
  SB sb;
  sa.begin(g.a.pitch, m0, g.a_limit, g.K);
  sb.begin(g.b.pitch, n0, g.b_limit, g.K);
  const int64_t at_a = KA == ALONG ? m0 * g.a.pitch : m0;
  const int64_t at_b = KB == ALONG ? n0 * g.b.pitch : n0;
  f32x4 acc[TM][TN] = {};
  Loop<E, P>::template run<false, SA, SB>(
      acc, lds, Steps(BK, from, to, g.a2.p ? 2 : 1), wm * TM * 16, wn * TN * 16,
      [&](const Steps& s, int q, char* to_a, char* to_b) {
        sa.copy(to_a, (s.pair ? g.a2.p : g.a.p) + at_a + q * g.a.plane, s.k);
        sb.copy(to_b, (s.pair ? g.b2.p : g.b.p) + at_b + q * g.b.plane, s.k);
      });
  const float factor = LIFTED<T> && g.factor ? *g.factor : 1.f;
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int64_t m = m0 + wm * TM * 16 + i * 16 + (lane & 15);
    if (m >= g.M) continue;
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int n = n0 + wn * TN * 16 + j * 16 + (lane >> 4) * 4;
      if (g.partial) {
        float* at = g.partial + ((int64_t)split * g.M + m) * g.N + n;
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (n + r < g.N) at[r] = g.add ? at[r] + acc[i][j][r] : acc[i][j][r];
      } else {
        const bool upper = g.each && m >= g.M / 2;
        const int64_t row = upper ? m - g.M / 2 : m;
        T* c = (T*)(upper ? g.c2 : g.c);
        if (!c || (g.each && row >= g.each)) continue;
        T* at = c + row * g.N + n;
        four_t<T> v;
#pragma unroll
        for (int r = 0; r < 4; ++r)
          v[r] = from_f32<T>((LIFTED<T> ? acc[i][j][r] * factor : acc[i][j][r]) +
                             (g.bias && n + r < g.N ? to_f32(((const T*)g.bias)[n + r]) : 0.f));
        if (g.wide) {
          if (n < g.N) *(four_t<T>*)at = v;
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (n + r < g.N) at[r] = v[r];
        }
      }
    }
  }
}

// Sums of dy's columns over runs of rows: partial[run, column], 64 columns a workgroup.
template <typename T>
__global__ void __launch_bounds__(256) ffn_column_sum_kernel(int64_t rows, int32_t cols,
                                                             const T* __restrict__ p, int64_t pitch,
                                                             float* __restrict__ partial,
                                                             int32_t add) {
  __shared__ float s[4][64];
  const int c = blockIdx.x * 64 + (threadIdx.x & 63), k = threadIdx.x >> 6;
  const int64_t from = rows * blockIdx.y / gridDim.y, to = rows * (blockIdx.y + 1) / gridDim.y;
  float acc = 0.f;
  if (c < cols)
#pragma unroll 8
    for (int64_t r = from + k; r < to; r += 4) acc += to_f32(p[r * pitch + c]);
  s[k][threadIdx.x & 63] = acc;
  __syncthreads();
  if (k == 0 && c < cols) {
    float* out = partial + (int64_t)blockIdx.y * cols + c;
    const float v = (s[0][threadIdx.x] + s[1][threadIdx.x]) + (s[2][threadIdx.x] + s[3][threadIdx.x]);
    *out = add ? *out + v : v;
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

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

// Rows of one pass: what keeps the hidden tensors of a pass (six bytes a value and plane) and
// the copies of its x and dy within 64M values each; the next rows reuse them.
static int64_t pass_rows(int64_t rows, int64_t width, int64_t hidden, int64_t out) {
  const int64_t cols = round8(std::max(hidden, std::max(width, out)));
  return std::min(rows, std::max<int64_t>((64 << 20) / cols / 256 * 256, 256));
}

template <typename T>
static int splits_of(int64_t tiles_, int64_t k) {
  return split_parts(tiles_, k / stage_k<T>());
}

// Values that the partial sums of a rows x N product over k may take, whatever its splits.
template <typename T>
static int64_t partial_values(int64_t rows, int64_t N, int64_t k) {
  return std::min(rows * N * std::max<int64_t>(1, k / stage_k<T>() / 4), (int64_t)SPLIT_TILES * 128 * 128);
}

// Whether there are enough tiles Z of an M x N product for the CUs.
#define FILLING_TILES 224
template <typename Z>
static bool fills(int64_t M, int64_t N, int64_t times = 1) {
  return tiles(M, Z::M) * tiles(N, Z::N) * times >= FILLING_TILES;
}

#define COLUMN_RUNS 128

// Everything a call keeps in its workspace.
template <typename T>
struct Plan {
  using E = typename Planes<T>::E;
  static constexpr int P = Planes<T>::N;
  int64_t rows, D, F, O, D8, F8, O8, pass;
  E *x, *wg, *wu, *wd, *dy, *h, *dgu;
  float *parts, *gu_sums, *dy_sums, *dwgu, *dwd;  // parts: of y or dx
  Lift* lift = nullptr;  // half's
  float* peaks = nullptr;
  int split_gu = 1, split_d = 1;
  uint64_t bytes;

  Plan(void* ws, int64_t rows_, int64_t D_, int64_t F_, int64_t O_, bool back)
      : rows(rows_), D(D_), F(F_), O(O_), D8(round8(D_)), F8(round8(F_)), O8(round8(O_)) {
    Carver c{(char*)ws};
    pass = pass_rows(rows, D, F, O);
    x = c.take<E>(P * pass * D8);
    wg = c.take<E>(P * F * D8);
    wu = c.take<E>(P * F * D8);
    wd = c.take<E>(P * O * F8);
    h = c.take<E>(P * pass * F8);
    parts = c.take<float>(back ? partial_values<T>(pass, D, F) : partial_values<T>(pass, O, F8));
    if (back) {
      dy = c.take<E>(P * pass * O8);
      dgu = c.take<E>(2 * P * pass * F8);
      gu_sums = c.take<float>(tiles(pass, TileSmall::M) * 2 * F8);
      dy_sums = c.take<float>(COLUMN_RUNS * O);
      split_gu = splits_of<T>(tiles(2 * F8, 128) * tiles(D, 128), pass);
      split_d = splits_of<T>(tiles(O, 128) * tiles(F, 128), pass);
      // (one sum over all rows is rounded where it is taken)
      dwgu = split_gu > 1 || pass < rows ? c.take<float>(split_gu * 2 * F8 * D) : nullptr;
      dwd = split_d > 1 || pass < rows ? c.take<float>(split_d * O * F) : nullptr;
      if (LIFTED<T>) {
        lift = c.take<Lift>(1);
        peaks = c.take<float>(LIFT_PEAKS);
      }
    }
    bytes = c.used;
  }
};

template <typename T, Along KA, Along KB>
static void product(hipStream_t s, ProductArgs<typename Planes<T>::E> g) {
  g.wide = g.N % 4 == 0 && aligned16((const T*)g.c, 0) && aligned16((const T*)g.c2, 0);
  const auto launch = [&](auto tile) {
    using Z = decltype(tile);
    hipLaunchKernelGGL((ffn_product_kernel<T, KA, KB, Z>),
                       dim3((unsigned)(tiles(g.M, Z::M) * tiles(g.N, Z::N) * g.splits)),
                       dim3(Z::THREADS), 0, s, g);
  };
  if constexpr (Planes<T>::N == 1 && KA == ALONG && KB == ALONG)
    if (fills<TileLarge>(g.M, g.N, g.splits)) return launch(TileLarge());
  launch(TileSmall());
}

// A product of rows, its sum over k split where its tiles are few.
template <typename T, Along KA, Along KB>
static void row_product(hipStream_t s, ProductArgs<typename Planes<T>::E> g, float* parts) {
  g.splits = splits_of<T>(tiles(g.M, TileSmall::M) * tiles(g.N, TileSmall::N), g.K);
  if (g.splits == 1) return product<T, KA, KB>(s, g);
  g.partial = parts;
  product<T, KA, KB>(s, g);
  Joiner<T> join;
  join.add(parts, g.M * g.N, g.N, g.splits, g.M, g.N, g.c, g.bias, g.factor);
  join.launch(s);
}

template <typename T, bool BACK>
static void hidden_products(hipStream_t s, const HiddenArgs<typename Planes<T>::E>& a) {
  const auto launch = [&](auto tile) {
    using Z = decltype(tile);
    hipLaunchKernelGGL((ffn_hidden_kernel<T, BACK, Z>),
                       dim3((unsigned)(tiles(a.rows, Z::M) * tiles(a.hidden8, Z::N / 2))),
                       dim3(Z::THREADS), 0, s, a);
  };
  if constexpr (Planes<T>::N == 1 && !BACK)
    if (fills<TileLarge>(a.rows, 2 * a.hidden8)) return launch(TileLarge());
  launch(TileSmall());
}

static uint64_t workspace_size(uint64_t rows, uint32_t width, uint32_t hidden, uint32_t out,
                               int32_t dtype, bool back) {
  uint64_t bytes = 0;
  if (check_sizes("tgs_gated_ffn workspace", rows, width, hidden, out, ACT_SILU)) return 0;
  with_dtype(dtype, "tgs_gated_ffn workspace", [&](auto tag) -> int {
    using T = decltype(tag);
    bytes = Plan<T>(nullptr, rows, width, hidden, out, back).bytes;
    if (RowKernels<T>::takes(width, out))
      bytes = RowKernels<T>::workspace(rows, width, hidden, out, back);
    if (!back) bytes = std::max(bytes, FewKernels<T>::workspace(std::min<int64_t>(rows, FEW_ROWS), hidden));
    return TGS_OK;
  });
  return bytes;
}

extern "C" uint64_t tgs_gated_ffn_fwd_workspace_size(uint64_t rows, uint32_t width, uint32_t hidden,
                                                     uint32_t out, int32_t dtype) {
  return workspace_size(rows, width, hidden, out, dtype, false);
}

extern "C" uint64_t tgs_gated_ffn_bwd_workspace_size(uint64_t rows, uint32_t width, uint32_t hidden,
                                                     uint32_t out, int32_t dtype) {
  return workspace_size(rows, width, hidden, out, dtype, true);
}

extern "C" int tgs_gated_ffn_fwd(uint64_t rows, uint32_t width, uint32_t hidden, uint32_t out,
                                 int32_t dtype, int32_t activation, const void* x, int64_t x_pitch,
                                 const void* w_gate, const void* w_up, const void* w_down,
                                 const void* b_gate, const void* b_up, const void* b_down, void* y,
                                 void* workspace, uint64_t workspace_bytes, hipStream_t stream) {
  return with_dtype(dtype, "tgs_gated_ffn_fwd", [&](auto tag) -> int {
    using T = decltype(tag);
    using E = typename Planes<T>::E;
    if (const int rc = check_sizes("tgs_gated_ffn_fwd", rows, width, hidden, out, activation))
      return rc;
    if (rows == 0) return TGS_OK;
    TGS_CHECK_ARG(x && w_gate && w_up && w_down && y, "tgs_gated_ffn_fwd: null pointer");
    TGS_CHECK_ARG(x_pitch >= (int64_t)width || rows == 1, "tgs_gated_ffn_fwd: pitch below width");
    if (workspace_bytes < tgs_gated_ffn_fwd_workspace_size(rows, width, hidden, out, dtype)) {
      tgs_set_error("tgs_gated_ffn_fwd: workspace too small");
      return TGS_ERR_WORKSPACE;
    }
    TGS_CHECK_ARG(workspace && (uintptr_t)workspace % 16 == 0,
                  "tgs_gated_ffn_fwd: the workspace starts on 16 bytes");
    FfnCall c{};
    c.rows = rows, c.width = width, c.hidden = hidden, c.out = out, c.act = activation;
    c.x = x, c.x_pitch = x_pitch, c.wg = w_gate, c.wu = w_up, c.wd = w_down;
    c.bg = b_gate, c.bu = b_up, c.bd = b_down, c.y = y;
    if (rows <= FEW_ROWS) {
      FewKernels<T>::forward(c, workspace, stream);
      TGS_RETURN_LAUNCH("tgs_gated_ffn_fwd");
    }
    if (RowKernels<T>::takes(width, out)) {
      RowKernels<T>::forward(c, workspace, stream);
      TGS_RETURN_LAUNCH("tgs_gated_ffn_fwd");
    }
    const Plan<T> p(workspace, rows, width, hidden, out, false);
    Layer<T> lay;
    const Operand<E> wg = lay.operand(w_gate, p.F, p.D, p.D, p.wg);
    const Operand<E> wu = lay.operand(w_up, p.F, p.D, p.D, p.wu);
    const Operand<E> wd = lay.operand(w_down, p.O, p.F, p.F, p.wd);
    for (int64_t r = 0; r < p.rows; r += p.pass) {
      const int64_t m = std::min(p.pass, p.rows - r);
      HiddenArgs<E> a{};
      a.x = lay.operand(row_at<T>(x, r, x_pitch), m, p.D, x_pitch, p.x);
      lay.launch(stream);
      a.wg = wg, a.wu = wu;
      a.rows = m, a.width8 = p.D8, a.hidden = p.F, a.hidden8 = p.F8, a.act = activation;
      a.bg = b_gate, a.bu = b_up, a.h = p.h, a.plane = m * p.F8;
      hidden_products<T, false>(stream, a);
      ProductArgs<E> g{};
      g.a = {p.h, a.plane, p.F8}, g.b = wd;
      g.M = m, g.N = p.O, g.K = p.F8, g.a_limit = m, g.b_limit = p.O;
      g.bias = b_down, g.c = (T*)y + r * p.O;
      row_product<T, ALONG, ALONG>(stream, g, p.parts);
    }
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
    using E = typename Planes<T>::E;
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
    TGS_CHECK_ARG(workspace && (uintptr_t)workspace % 16 == 0,
                  "tgs_gated_ffn_bwd: the workspace starts on 16 bytes");
    FfnCall c{};
    c.rows = rows, c.width = width, c.hidden = hidden, c.out = out, c.act = activation;
    c.x = x, c.x_pitch = x_pitch, c.wg = w_gate, c.wu = w_up, c.wd = w_down;
    c.bg = b_gate, c.bu = b_up, c.dy = dy, c.dy_pitch = dy_pitch;
    c.dx = dx, c.dwg = dw_gate, c.dwu = dw_up, c.dwd = dw_down;
    c.dbg = db_gate, c.dbu = db_up, c.dbd = db_down;
    if (rows && RowKernels<T>::takes(width, out)) {
      RowKernels<T>::backward(c, workspace, stream);
      TGS_RETURN_LAUNCH("tgs_gated_ffn_bwd");
    }
    const Plan<T> p(workspace, rows, width, hidden, out, true);
    Layer<T> lay;
    const Operand<E> wg = lay.operand(w_gate, p.F, p.D, p.D, p.wg);
    const Operand<E> wu = lay.operand(w_up, p.F, p.D, p.D, p.wu);
    const Operand<E> wd = lay.operand(w_down, p.O, p.F, p.F, p.wd);
    const bool hidden_sums = db_gate || db_up;
    if (LIFTED<T> && rows) ffn_lift(c, p.lift, p.peaks, stream);
    const float* const back_d = LIFTED<T> && rows ? &p.lift->back_d : nullptr;
    const float* const back_h = LIFTED<T> && rows ? &p.lift->back_h : nullptr;
    for (int64_t r = 0; r < p.rows; r += p.pass) {
      const int64_t m = std::min(p.pass, p.rows - r);
      HiddenArgs<E> a{};
      a.x = lay.operand(row_at<T>(x, r, x_pitch), m, p.D, x_pitch, p.x);
      a.dy = lay.operand(row_at<T>(dy, r, dy_pitch), m, p.O, dy_pitch, p.dy);
      lay.launch(stream);
      a.wg = wg, a.wu = wu, a.wd = wd;
      a.rows = m, a.width8 = p.D8, a.hidden = p.F, a.hidden8 = p.F8, a.out = p.O, a.out8 = p.O8;
      a.act = activation, a.bg = b_gate, a.bu = b_up;
      a.h = p.h, a.dgu = p.dgu, a.plane = m * p.F8;
      a.sums = hidden_sums ? p.gu_sums : nullptr, a.add = r > 0, a.lift = p.lift;
      hidden_products<T, true>(stream, a);
      if (dx) {
        ProductArgs<E> g{};
        g.a = {p.dgu, 2 * a.plane, 2 * p.F8}, g.a2 = {p.dgu + p.F8, 2 * a.plane, 2 * p.F8};
        g.b = wg, g.b2 = wu;
        // (k runs to the weights' last row; behind it dg and du are zero)
        g.M = m, g.N = p.D, g.K = p.F, g.a_limit = m, g.b_limit = p.D8;
        g.c = (T*)dx + r * p.D, g.factor = back_d;
        row_product<T, ALONG, ACROSS>(stream, g, p.parts);
      }
      if (dw_gate || dw_up) {
        ProductArgs<E> g{};
        g.a = {p.dgu, 2 * a.plane, 2 * p.F8}, g.b = a.x;
        g.M = 2 * p.F8, g.N = p.D, g.K = m, g.a_limit = 2 * p.F8, g.b_limit = p.D8;
        g.splits = p.split_gu, g.partial = p.dwgu, g.add = r > 0;
        g.c = dw_gate, g.c2 = dw_up, g.each = p.F, g.factor = back_d;
        product<T, ACROSS, ACROSS>(stream, g);
      }
      if (dw_down) {
        ProductArgs<E> g{};
        g.a = a.dy, g.b = {p.h, a.plane, p.F8};
        g.M = p.O, g.N = p.F, g.K = m, g.a_limit = p.O8, g.b_limit = p.F8;
        g.splits = p.split_d, g.partial = p.dwd, g.add = r > 0, g.c = dw_down;
        g.factor = back_h;
        product<T, ACROSS, ACROSS>(stream, g);
      }
      if (db_down)
        hipLaunchKernelGGL(ffn_column_sum_kernel<T>, dim3((unsigned)tiles(p.O, 64), COLUMN_RUNS),
                           dim3(256), 0, stream, m, (int32_t)p.O,
                           (const T*)row_at<T>(dy, r, dy_pitch), dy_pitch, p.dy_sums, r > 0);
    }
    Joiner<T> join;
    const int64_t some = p.rows > 0;  // no rows: sums of nothing
    if (p.dwgu || !some) {
      join.add(p.dwgu, 2 * p.F8 * p.D, p.D, some * p.split_gu, p.F, p.D, dw_gate,
               nullptr, back_d);
      join.add(p.dwgu + p.F8 * p.D, 2 * p.F8 * p.D, p.D, some * p.split_gu, p.F, p.D, dw_up, nullptr,
               back_d);
    }
    if (p.dwd || !some)
      join.add(p.dwd, p.O * p.F, p.F, some * p.split_d, p.O, p.F, dw_down, nullptr,
               back_h);
    const int64_t row_tiles = tiles(p.pass, TileSmall::M);
    join.add(p.gu_sums, 2 * p.F8, p.F8, some * row_tiles, 1, p.F, db_gate, nullptr,
             back_d);
    join.add(p.gu_sums + p.F8, 2 * p.F8, p.F8, some * row_tiles, 1, p.F, db_up, nullptr,
             back_d);
    join.add(p.dy_sums, p.O, p.O, some * COLUMN_RUNS, 1, p.O, db_down);
    join.launch(stream);
    TGS_RETURN_LAUNCH("tgs_gated_ffn_bwd");
  });
}
