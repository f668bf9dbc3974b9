// A dense layer's parameter gradients on gfx950:
//   w_adj[n][k] = beta w_adj[n][k] + sum over m of g[m][n] x[m][k]
//   b_adj[n]    = beta b_adj[n]    + sum over m of g[m][n]
// over the live rows m, g the output's adjoint and x the layer's input, both
// row-major in fp32, bf16 or fp16.
//
// The contraction runs over the rows, the long axis (up to half a million), and
// the result is small: a workgroup takes a tile of the result over one piece of
// the rows, and the pieces' sums, in the workspace, are added in order by a
// second kernel. Nothing is atomic: results repeat bit for bit.
//
// The products run on the 16-bit matrix instruction 16x16x32, whose lanes want
// eight consecutive m of one column where memory holds consecutive columns of
// one m. So a thread reads 8 rows by V columns, 16 (or 8) bytes a row, and writes
// V chunks of 8 m into LDS, columns as LDS rows of 128 bytes: 16-bit values as
// they are, two rows' halves merged by a byte permute (64 rows a step); fp32 ones
// as fp16 pairs (32 rows a step), whose conversion packs two rows anyway, with
// three products for one:
//   (hi + lo)(hi' + lo') less lo lo', each value held to 2^-23 of itself.
// A column's values share a power of two, so that they fit fp16's range; it
// follows the column: the largest value of its first nonzero step comes to
// [2^11, 2^12), and a later one past 2^15 lowers it, and the sums made before by
// the exact factor. The wave that reads a column's 32 rows of a step holds all of
// them, so it finds the new scale by itself and hands the factor on through LDS
// (rare). A value below 2^-13 of the column's largest is held to 2^-36 of that, an
// absolute error that a sum feels only where the largest meet zeros: one value of
// 1e6 (1e8, 1e12) times the rest whose other factor is 0 leaves 1024 rows' sums off by
// 2.1e-7 (2.5e-5, 4.2e-2) of sum |g| |x|, 40000 rows' by 1.2e-8 (1.4e-6, 2.3e-3). A
// third part would hold it, for six products instead of three.
//
// What bounds it: the matrix unit under the clock that its power leaves. For
// 486946 x 2048 x 512 in bf16 (1.14 to 1.21 ms, 845 to 895 TFLOP/s; a library's
// product of that shape 2.03 ms, of 8192 cubed 1131 TFLOP/s) the products alone take
// 0.73 ms, the rows' way into LDS alone 0.71, the loads alone 0.60; together the clock
// falls from 2.2 to 1.8 GHz, and the matrix unit is busy 42% of the cycles. 122688 x
// 768 x 256 in fp32 takes 187 to 200 us, of which writing and adding the pieces is 25:
// the matrix unit is busy 41% of the cycles, the vector unit 58% (the splits), the
// waves wait 33%. Small results are bound by the pieces: 27318 x 128 x 128 takes 21.5
// to 24 us (5.8 at the copy's rate), and their sums move 82% of the operands' bytes.
//
// The matrix instruction rounds toward minus infinity, an error with a mean that
// half a million rows would add up. So a step is summed from zero, the sums of
// the steps are added in fp32 to nearest, and g's odd steps are negated and
// subtracted.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "../../include/pet_model.h"
#include "attn_common.h"
#include "gemm_common.h"
#include "split_bf16.h"
#include "typed.h"

namespace pet_wgrad {

using pet_attn::max_g;
using pet_gemm::ring_barrier;
using pet_split::f4;
using pet_split::kFltMax;
using pet_split::u4;

// A workgroup of WN x WK waves, each TN x TK tiles of 16 x 16, V columns a thread
// as it reads.
template <class T, int WN, int WK, int TN, int TK, int V>
struct Tile {
  static constexpr bool PAIRS = sizeof(T) == 4;
  static constexpr int STEP = PAIRS ? 32 : 64;        // rows
  static constexpr int BN = 16 * TN * WN, BK = 16 * TK * WK, ROWS = BN + BK;
  static constexpr int WAVES = WN * WK, OQ = STEP / 32;  // a unit of reading: 32 rows by 16 V columns, a wave's
  static constexpr int GA = BN / (16 * V), GB = BK / (16 * V), UNITS = (GA + GB) * OQ;
  static_assert(BN % (16 * V) == 0 && BK % (16 * V) == 0 && UNITS <= WAVES, "a unit a wave");
  static constexpr int W = V * int(sizeof(T)) / 4;  // words a thread reads of a row
  static constexpr int STAGE = ROWS * 8;            // 16-byte chunks
};

// The slot of half h (hi and lo, or a step's first and last 32 rows) of chunk q in
// LDS row r: a read or a write of 16 rows by four chunks runs at the rate of
// consecutive lanes.
__device__ __forceinline__ int slot(int q, int h, int r) {
  return r * 8 + ((2 * q + h) ^ (((r >> 1) & 1) | ((r >> 1) & 4)));
}

// The largest |x| of eight (a NaN is passed over: it makes its column NaN by itself).
__device__ __forceinline__ float amax8(const unsigned (&x)[8]) {
  float m;
  asm("v_max3_f32 %0, |%1|, |%2|, |%3|" : "=v"(m) : "v"(x[0]), "v"(x[1]), "v"(x[2]));
  asm("v_max3_f32 %0, |%1|, |%2|, %0" : "+v"(m) : "v"(x[3]), "v"(x[4]));
  asm("v_max3_f32 %0, |%1|, |%2|, %0" : "+v"(m) : "v"(x[5]), "v"(x[6]));
  asm("v_max3_f32 %0, |%1|, |%1|, %0" : "+v"(m) : "v"(x[7]));
  return m;
}

// Eight floats times s, a power of two, as fp16 pairs to nearest.
__device__ __forceinline__ void split8(const unsigned (&x)[8], float s, u4& hi, u4& lo) {
#pragma clang fp contract(off)
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float a = __uint_as_float(x[2 * j]), b = __uint_as_float(x[2 * j + 1]);
    const pet_split::h2v h = {(_Float16)(a * s), (_Float16)(b * s)};
    const pet_split::h2v l = {(_Float16)fmaf(a, s, -float(h[0])), (_Float16)fmaf(b, s, -float(h[1]))};
    hi[j] = __builtin_bit_cast(unsigned, h);
    lo[j] = __builtin_bit_cast(unsigned, l);
  }
}

template <class T>
__device__ __forceinline__ f4 mfma(const u4& a, const u4& b, const f4& c) {
  if constexpr (std::is_same<T, __bf16>::value) return pet_split::mfma_bf(a, b, c);
  else return pet_split::mfma_h(a, b, c);
}
// c + both halves of x times those of y (ones, of either sign), rounded once.
template <class T>
__device__ __forceinline__ float dot2(unsigned x, unsigned y, float c) {
  typedef T t2 __attribute__((ext_vector_type(2)));
  if constexpr (std::is_same<T, __bf16>::value)
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(t2, x), __builtin_bit_cast(t2, y), c, false);
  else return __builtin_amdgcn_fdot2(__builtin_bit_cast(t2, x), __builtin_bit_cast(t2, y), c, false);
}

typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned u4u __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned u2u __attribute__((ext_vector_type(2), aligned(2)));

struct Args {
  int M, N, K;
  int64_t ldg, ldx;
  int live_base;
  const int* live;
  int64_t chunk;
  int pieces, tiles_n, tiles_k;
  float* out;      // [pieces][N][K], or with one piece w_adj
  int64_t ldo;
  double* bout;    // [pieces][tiles_k][N], with one piece unused
  float* b_adj;    // null: no bias
  float beta;
};

template <class T, int WN, int WK, int TN, int TK, int V>
__global__ void __launch_bounds__(64 * WN * WK, TN * TK >= 16 ? 2 : 4)
    wgrad_kernel(const T* __restrict__ G, const T* __restrict__ X, Args a) {
  using C = Tile<T, WN, WK, TN, TK, V>;
  constexpr bool PAIRS = C::PAIRS;
  constexpr int W = C::W;
  __shared__ u4 stage[2 * C::STAGE];
  __shared__ float factor[PAIRS ? 2 : 1][PAIRS ? C::ROWS : 1];  // a step's factors of the sums before it
  __shared__ int changed[2][C::WAVES];                          // a wave's unit set some
  __shared__ int expo[PAIRS ? C::ROWS : 1];
  __shared__ int special[C::WAVES];
  __shared__ double bsum[4 * C::OQ][C::BN];  // g's sums, a slot a thread and column

  // The pieces go round the XCDs, a piece's tiles to one of them, whose L2 then
  // holds the rows that they share.
  const int tiles = a.tiles_n * a.tiles_k, xcds = a.pieces % 8 == 0 ? 8 : 1;
  const int on = int(blockIdx.x) % xcds, at = int(blockIdx.x) / xcds;
  const int piece = at / tiles * xcds + on, tile = at % tiles;
  const int n0 = tile / a.tiles_k * C::BN, k0 = tile % a.tiles_k * C::BK;
  const int end = pet_typed::live_rows(a.M, a.live_base, a.live);
  const int first = int(min(piece * a.chunk, int64_t(end)));
  const int last = int(min(first + a.chunk, int64_t(end)));
  const int steps = (last - first + C::STEP - 1) / C::STEP;

  const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6)), l = threadIdx.x & 63, c = l & 15, g = l >> 4;

  // ---- this wave's unit of reading
  const bool reads = wave < C::UNITS, is_g = wave < C::GA * C::OQ;
  const int group = (is_g ? wave : wave - C::GA * C::OQ) / C::OQ, oq = wave % C::OQ;  // (GA OQ is a multiple of OQ)
  const int col = (is_g ? n0 : k0) + group * 16 * V + V * c, left = (is_g ? a.N : a.K) - col;
  const int64_t ld = is_g ? a.ldg : a.ldx;
  // (16 consecutive lanes write two octets' chunks, as a read's groups of lanes meet them: no bank twice)
  const int gs = g ^ (((c >> 2) + 1) >> 1 & 1), oct = 4 * oq + gs;  // this thread's eight rows of a step
  const int row0 = (is_g ? 0 : C::BN) + group * 16 * V + c;  // its LDS rows: row0 + 16 j
  // Every load lands in the operand: columns past its last are read as its last V
  // (`mend` moves and drops them), or where it has fewer than V one by one; rows
  // past the piece's last as that one.
  const int cols = is_g ? a.N : a.K;
  const bool narrow = cols < V, whole = col - V * c + 16 * V <= cols;  // of the unit: wave-uniform
  const T* src = (is_g ? G : X) + (int64_t(first) + 8 * oct) * ld + (narrow ? 0 : min(col, cols - V));
  const int64_t ahead = int64_t(C::STEP) * ld;
  unsigned raw[8][W];
  auto load = [&](int s) {
    if (!reads) return;
    const T* p = src;
    src += ahead;
    int rows = 8;
    if ((s + 1) * C::STEP > last - first) {  // the piece's last, partial step
      rows = last - first - s * C::STEP - 8 * oct;
      if (rows < 1) p -= (1 - rows) * ld, rows = 1;
    }
    if (narrow) {
#pragma unroll
      for (int r = 0; r < 8; ++r) {
#pragma unroll
        for (int w = 0; w < W; ++w) {
          if constexpr (PAIRS) raw[r][w] = __float_as_uint(p[min(col + w, cols - 1)]);
          else
            raw[r][w] = unsigned(__builtin_bit_cast(unsigned short, p[min(col + 2 * w, cols - 1)])) |
                        unsigned(__builtin_bit_cast(unsigned short, p[min(col + 2 * w + 1, cols - 1)])) << 16;
        }
        p += r + 1 < rows ? ld : 0;
      }
      return;
    }
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      if constexpr (W == 4) {
        const u4u q = *reinterpret_cast<const u4u*>(p);
        raw[r][0] = q[0], raw[r][1] = q[1], raw[r][2] = q[2], raw[r][3] = q[3];
      } else {
        const u2u q = *reinterpret_cast<const u2u*>(p);
        raw[r][0] = q[0], raw[r][1] = q[1];
      }
      p += r + 1 < rows ? ld : 0;
    }
  };
  // Zeros for the rows and columns that are not the piece's.
  auto mend = [&](int s) {
    const int rows = last - first - s * C::STEP - 8 * oct;
    constexpr int PER = V / W;  // elements a word
    if (!whole) {
      const int up = narrow ? 0 : min(max(V - left, 0), V - 1);  // elements to move down
#pragma unroll
      for (int r = 0; r < 8; ++r)
#pragma unroll
        for (int w = 0; w < W; ++w) {
          unsigned x[W + 1];
#pragma unroll
          for (int i = 0; i <= W; ++i) x[i] = w + i < W ? raw[r][w + i] : 0u;
          unsigned lo = 0, hi = 0;
#pragma unroll
          for (int i = 0; i < W; ++i)
            if (up / PER == i) lo = x[i], hi = x[i + 1];
          unsigned v = PER == 2 && (up & 1) ? lo >> 16 | hi << 16 : lo;
          const int n = left - w * PER;  // elements of the word that are the operand's
          raw[r][w] = n >= PER ? v : PER == 2 && n == 1 ? v & 0xffffu : 0u;
        }
    }
#pragma unroll
    for (int r = 0; r < 8; ++r)
#pragma unroll
      for (int w = 0; w < W; ++w) raw[r][w] = r < rows ? raw[r][w] : 0u;
  };

  float scale[PAIRS ? V : 1];  // of each column, 2^126 until a value is too large for that
#pragma unroll
  for (int j = 0; j < (PAIRS ? V : 1); ++j) scale[j] = 0x1p126f;
  // A column's tiles share out the steps whose g they sum; with one piece the first
  // takes all, and the bias is done (one launch a call).
  const bool direct = a.pieces == 1;
  const int kt = tile % a.tiles_k;
  const bool bias = a.b_adj && is_g && reads && (!direct || kt == 0);
  int turn = 0;
  double* mine = &bsum[oct][(is_g ? group : 0) * 16 * V + c];  // LDS rows' order, as row0
  float few[V];  // of sixteen steps, then added there (every step: a tenth of the whole time)
#pragma unroll
  for (int j = 0; j < V; ++j) few[j] = 0.f;
  if (bias)
#pragma unroll
    for (int j = 0; j < V; ++j) mine[16 * j] = 0.0;
  int inf = 0;

  // the step that `load` read, into LDS
  auto put = [&](int s) {
    if (!reads) return;
    if (!whole || (s + 1) * C::STEP > last - first) mend(s);
    u4* to = stage + (s & 1) * C::STAGE;
    const bool sums = bias && (direct || turn == kt);
    turn = turn + 1 == a.tiles_k ? 0 : turn + 1;
    if constexpr (PAIRS) {
      unsigned x[V][8];
#pragma unroll
      for (int j = 0; j < V; ++j)
#pragma unroll
        for (int r = 0; r < 8; ++r) x[j][r] = raw[r][j];
      float m[V];
      bool grew = false;
#pragma unroll
      for (int j = 0; j < V; ++j) m[j] = amax8(x[j]), grew |= m[j] * scale[j] > 32768.f;
      const bool any = __builtin_amdgcn_ballot_w64(grew) != 0;
      if (any) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float top = max_g(m[j]);
          float f = 1.f;
          if (top * scale[j] > 32768.f) {
            const int k = 12 - __builtin_amdgcn_frexp_expf(fminf(top, kFltMax));
            f = __builtin_amdgcn_ldexpf(1.f, k + 1 - __builtin_amdgcn_frexp_expf(scale[j]));
            scale[j] = __builtin_amdgcn_ldexpf(1.f, k);
          }
          inf |= top > kFltMax;
          if (g == 0) factor[s & 1][row0 + 16 * j] = f;
        }
      }
      if (l == 0) changed[s & 1][wave] = any;
      const bool neg = is_g && (s & 1);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        u4 hi, lo;
        split8(x[j], neg ? -scale[j] : scale[j], hi, lo);
        to[slot(gs, 0, row0 + 16 * j)] = hi;
        to[slot(gs, 1, row0 + 16 * j)] = lo;
        if (sums) {
          float t[8];
#pragma unroll
          for (int r = 0; r < 8; ++r) t[r] = __uint_as_float(x[j][r]);
          few[j] += ((t[0] + t[1]) + (t[2] + t[3])) + ((t[4] + t[5]) + (t[6] + t[7]));
        }
      }
    } else {
      const unsigned flip = is_g && (s & 1) ? 0x80008000u : 0u;
      const unsigned one = (std::is_same<T, __bf16>::value ? 0x3f803f80u : 0x3c003c00u) ^ flip;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        u4 even, odd;
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          even[d] = __builtin_amdgcn_perm(raw[2 * d + 1][w], raw[2 * d][w], 0x05040100u) ^ flip;
          odd[d] = __builtin_amdgcn_perm(raw[2 * d + 1][w], raw[2 * d][w], 0x07060302u) ^ flip;
        }
        if (sums)
#pragma unroll
          for (int d = 0; d < 4; ++d) {
            few[2 * w] = dot2<T>(even[d], one, few[2 * w]);
            few[2 * w + 1] = dot2<T>(odd[d], one, few[2 * w + 1]);
          }
        to[slot(gs, oq, row0 + 32 * w)] = even;
        to[slot(gs, oq, row0 + 32 * w + 16)] = odd;
      }
    }
    if (bias && ((s & 15) == 15 || (s + 1) * C::STEP >= last - first))
#pragma unroll
      for (int j = 0; j < V; ++j) mine[16 * j] += double(few[j]), few[j] = 0.f;
  };

  // ---- this wave's products
  const int rn = wave / WK * 16 * TN, rk = C::BN + wave % WK * 16 * TK;  // its LDS rows
  f4 acc[TN][TK];
#pragma unroll
  for (int i = 0; i < TN; ++i)
#pragma unroll
    for (int j = 0; j < TK; ++j) acc[i][j] = f4{0.f, 0.f, 0.f, 0.f};

  // (a wave past the result's edge has no products to make: 6% of 62001 x 500 x 333)
  auto first_column = [](int r) { return r / (16 * V) * 16 * V + r / 16 % V; };
  const bool works = n0 + first_column(rn) < a.N && k0 + first_column(rk - C::BN) < a.K;
  auto products = [&](int s) {
    if (!works) return;
    const u4* from = stage + (s & 1) * C::STAGE;
    if constexpr (PAIRS) {
      if (__builtin_amdgcn_ballot_w64(l < C::UNITS && changed[s & 1][l < C::UNITS ? l : 0]) != 0) {
        float fk[TK];
#pragma unroll
        for (int j = 0; j < TK; ++j) {
          const int r = rk + 16 * j + c, u = C::GA * C::OQ + (r - C::BN) / (16 * V);
          fk[j] = changed[s & 1][u] ? factor[s & 1][r] : 1.f;
        }
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = rn + 16 * i + 4 * g + e;
            const float fn = changed[s & 1][r / (16 * V)] ? factor[s & 1][r] : 1.f;
#pragma unroll
            for (int j = 0; j < TK; ++j) acc[i][j][e] *= fn * fk[j];
          }
      }
    }
    __builtin_amdgcn_s_setprio(1);
    u4 b[TK][2];
#pragma unroll
    for (int j = 0; j < TK; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) b[j][h] = from[slot(g, h, rk + 16 * j + c)];
    const float sg = s & 1 ? -1.f : 1.f;
    u4 x = from[slot(g, 0, rn + c)], y = from[slot(g, 1, rn + c)];
#pragma unroll
    for (int i = 0; i < TN; ++i) {
      const int ahead = rn + 16 * (i + 1 < TN ? i + 1 : i) + c;
      const u4 nx = from[slot(g, 0, ahead)], ny = from[slot(g, 1, ahead)];
#pragma unroll
      for (int j = 0; j < TK; ++j) {
        f4 t = {0.f, 0.f, 0.f, 0.f};
        if constexpr (PAIRS) {  // (hi, lo) parts, the small products first
          t = pet_split::mfma_h(y, b[j][0], t);
          t = pet_split::mfma_h(x, b[j][1], t);
          t = pet_split::mfma_h(x, b[j][0], t);
        } else {
          t = mfma<T>(x, b[j][0], t);
          t = mfma<T>(y, b[j][1], t);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(t[e], sg, acc[i][j][e]);
      }
      x = nx, y = ny;
    }
    __builtin_amdgcn_s_setprio(0);
  };

  if (steps > 0) {
    load(0);
    if constexpr (C::WAVES == 8) {
      // Two waves a SIMD, half a step apart: while one of them splits its rows
      // into LDS the other has the matrix unit. (All in step: 1289 us against 1227
      // for 486946 x 2048 x 512 in bf16, 1197 with the products' priority raised.)
      const bool late = wave >= 4;
      if (late) ring_barrier();
      for (int i = 0; i < steps + !late; ++i) {
        if (i < steps) put(i);
        if (i + 1 < steps) load(i + 1);
        ring_barrier();
        const int p = late ? i : i - 1;
        if (p >= 0) products(p);
        ring_barrier();
      }
      if (late) ring_barrier();
    } else {
      put(0);
      if (steps > 1) load(1);
      ring_barrier();
      for (int s = 0; s < steps; ++s) {
        if (s + 1 < steps) put(s + 1);
        if (s + 2 < steps) load(s + 2);
        products(s);
        ring_barrier();
      }
    }
  }

  // ---- the scales' exponents, whether an infinity came by, the bias
  if constexpr (PAIRS) {
    if (l == 0) special[wave] = 0;
    if (reads && g == 0)
#pragma unroll
      for (int j = 0; j < V; ++j) expo[row0 + 16 * j] = 1 - __builtin_amdgcn_frexp_expf(scale[j]);
    if (__builtin_amdgcn_ballot_w64(inf) != 0 && l == 0) special[wave] = 1;
  }
  __syncthreads();
  if (a.b_adj && (!direct || kt == 0))
    for (int r = threadIdx.x; r < C::BN; r += 64 * C::WAVES) {
      const int n = n0 + r / (16 * V) * 16 * V + r % 16 * V + r / 16 % V;
      if (n < a.N) {
        double v = 0.0;
        for (int q = 0; q < 4 * C::OQ; ++q) v += bsum[q][r];
        if (!direct) a.bout[(int64_t(piece) * a.tiles_k + kt) * a.N + n] = v;
        else a.b_adj[n] = a.beta != 0.f ? float(double(a.beta) * a.b_adj[n] + v) : float(v);
      }
    }

  // columns of LDS rows: row 16 j + i of a group is column V i + j
  auto n_of = [&](int i, int e) {
    const int r = rn + 16 * i;
    return n0 + r / (16 * V) * 16 * V + V * (4 * g + e) + r / 16 % V;
  };
  auto k_of = [&](int j) {
    const int r = rk - C::BN + 16 * j;
    return k0 + r / (16 * V) * 16 * V + V * c + r / 16 % V;
  };

  bool scaled = PAIRS;
  if constexpr (PAIRS) {
    int seen = 0;
#pragma unroll
    for (int w = 0; w < C::WAVES; ++w) seen |= special[w];
    if (seen) {
      // An infinity's low part is NaN, and spoils more than fp32 products would:
      // the piece again on the fp32 matrix instruction, from memory.
      scaled = false;
#pragma unroll
      for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int j = 0; j < TK; ++j) acc[i][j] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
      for (int m = first; m < last; m += 4) {
        float x[TN], y[TK];
        const bool in = m + g < last;
        const T* gr = G + int64_t(in ? m + g : first) * a.ldg;
        const T* xr = X + int64_t(in ? m + g : first) * a.ldx;
#pragma unroll
        for (int i = 0; i < TN; ++i) {
          const int r = rn + 16 * i, n = n0 + r / (16 * V) * 16 * V + V * c + r / 16 % V;
          x[i] = in && n < a.N ? float(gr[n]) : 0.f;
        }
#pragma unroll
        for (int j = 0; j < TK; ++j) y[j] = in && k_of(j) < a.K ? float(xr[k_of(j)]) : 0.f;
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
          for (int j = 0; j < TK; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[i], y[j], acc[i][j], 0, 0, 0);
      }
    }
  }

  float* out = a.out + (direct ? 0 : int64_t(piece) * a.N * a.K);
#pragma unroll
  for (int i = 0; i < TN; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int n = n_of(i, e);
      if (n >= a.N) continue;
      int en = 0;
      if constexpr (PAIRS) en = expo[rn + 16 * i + 4 * g + e];
#pragma unroll
      for (int j = 0; j < TK; j += 4) {
        const int k = k_of(j);
        if (k >= a.K) continue;
        float v[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          v[q] = acc[i][j + q][e];
          if constexpr (PAIRS)
            if (scaled) v[q] = __builtin_amdgcn_ldexpf(v[q], en + expo[rk + 16 * (j + q) + c]);
        }
        float* o = out + int64_t(n) * a.ldo + k;
        if (k + 4 <= a.K) {
          f4u old = {0.f, 0.f, 0.f, 0.f};
          if (direct && a.beta != 0.f) old = *reinterpret_cast<const f4u*>(o);
          f4u w;
#pragma unroll
          for (int q = 0; q < 4; ++q) w[q] = direct && a.beta != 0.f ? fmaf(a.beta, old[q], v[q]) : v[q];
          *reinterpret_cast<f4u*>(o) = w;
        } else {
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (k + q < a.K) o[q] = direct && a.beta != 0.f ? fmaf(a.beta, o[q], v[q]) : v[q];
        }
      }
    }
}

// adj = beta adj + the pieces' sums in double: a thread sums every eighth piece of
// four elements, or every 64th of one column's biases, eight loads at a time, and
// the strips are joined in order. MI355X: 80 pieces of 768 x 256 11 us (24 with a
// thread an element, its loads one after the other); 26670 x 128 x 512, whose 512
// pieces of the bias eight strips summed as they do the rest, 66 us a call and 40 now.
constexpr int kStrips = 8, kSumElements = 4 * 256 / kStrips;
__global__ void __launch_bounds__(256) wgrad_sum_kernel(int N, int K, int pieces, int bpieces,
                                                        const float* __restrict__ part,
                                                        const double* __restrict__ bpart, float* __restrict__ w_adj,
                                                        int64_t ldw, float* __restrict__ b_adj, float beta) {
  constexpr int Q = 256 / kStrips, E = kSumElements;  // threads a strip, elements a workgroup
  __shared__ double sums[256][4];             // [strip][thread][element]; a bias's [strip][column]
  const int64_t nk = int64_t(N) * K, wblocks = (nk + E - 1) / E;
  const bool bias = int64_t(blockIdx.x) >= wblocks;
  double v[4] = {0.0, 0.0, 0.0, 0.0};
  if (bias) {
    const int64_t n = (int64_t(blockIdx.x) - wblocks) * 4 + (threadIdx.x & 3);
    if (n < N)
      for (int s = threadIdx.x >> 2; s < bpieces; s += 8 * 64) {
        double x[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) x[u] = s + 64 * u < bpieces ? bpart[int64_t(s + 64 * u) * N + n] : 0.0;
#pragma unroll
        for (int u = 0; u < 8; ++u) v[0] += x[u];
      }
    sums[threadIdx.x >> 2][threadIdx.x & 3] = v[0];
    __syncthreads();
    if (threadIdx.x < 4 && n < N) {
      double r = 0.0;
#pragma unroll
      for (int s = 0; s < 64; ++s) r += sums[s][threadIdx.x];
      b_adj[n] = beta != 0.f ? float(double(beta) * b_adj[n] + r) : float(r);
    }
    return;
  }
  const int strip = threadIdx.x / Q;
  const int64_t first = int64_t(blockIdx.x) * E, i = first + 4 * (threadIdx.x % Q);
  if (i + 4 <= nk) {
    int s = strip;
    for (; s + 7 * kStrips < pieces; s += 8 * kStrips) {
      f4u x[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) x[u] = *reinterpret_cast<const f4u*>(part + int64_t(s + u * kStrips) * nk + i);
#pragma unroll
      for (int u = 0; u < 8; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += x[u][e];
    }
#pragma unroll 2
    for (; s < pieces; s += kStrips) {
      const f4u x = *reinterpret_cast<const f4u*>(part + int64_t(s) * nk + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += x[e];
    }
  } else {
    for (int s = strip; s < pieces; s += kStrips)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i + e < nk) v[e] += part[int64_t(s) * nk + i + e];
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) sums[threadIdx.x][e] = v[e];
  __syncthreads();
  const int t = threadIdx.x;
  if (t >= E || first + t >= nk) return;
  double r = 0.0;
#pragma unroll
  for (int s = 0; s < kStrips; ++s) r += sums[s * Q + (t >> 2)][t & 3];
  const int64_t j = first + t;
  float* o = w_adj + j / K * ldw + j % K;
  *o = beta != 0.f ? float(double(beta) * *o + r) : float(r);
}

// How a product is cut: the tile and the pieces.
struct Plan {
  int64_t chunk;
  int tile, pieces, tiles_n, tiles_k;
};
constexpr int kEdge[3] = {256, 128, 64};
constexpr int kResident[3] = {256, 512, 1024};  // workgroups that the chip holds at once

// The largest tile that the result fills and the work feeds. MI355X, us a call in
// fp32:
//   256 against 128 wide: 122688 x 768 x 256 197 and 250, 8192 x 1024 x 1024 89 and 98, 62001 x 500 x 333 (1.0e10
//     products) 139 and 151, 20011 x 1000 x 330 in fp16 (6.6e9) 57 and 64, but 27318 x 384 x 256 (2.7e9) 56 and 48;
//   128 against 64 wide: 26670 x 1024 x 128 (3.5e9) 59 and 69, 27318 x 384 x 256 48 and 58, 5000 x 512 x 512 (1.3e9)
//     36.5 and 36.7, but 27318 x 128 x 128 (4.5e8) 26 and 24, 8000 x 384 x 128 27 and 24, 648 x 1024 x 256 (1.7e8) 23
//     and 20: few steps wait on memory, not on the tile.
// Pieces fill the chip, in whole eights (an XCD each in turn), of at least four steps (27318 x 128 x 128 in 128 wide
// tiles 26.5 us, 28 with two and 31 with eight).
Plan plan_of(int dtype, int M, int N, int K) {
  const int step = dtype == PET_DTYPE_F32 ? 32 : 64;
  const double work = double(M) * N * K;
  Plan p{};
  p.tile = N > 128 && K > 128 && work >= 4e9 ? 0 : N > 64 && K > 64 && work >= 1e9 ? 1 : 2;
  const int64_t edge = kEdge[p.tile], tn = (int64_t(N) + edge - 1) / edge, tk = (int64_t(K) + edge - 1) / edge;
  const int64_t steps = std::max<int64_t>(1, (int64_t(M) + step - 1) / step);
  int64_t pieces = std::max<int64_t>(1, std::min<int64_t>(kResident[p.tile] / (tn * tk), (steps + 3) / 4));
  if (pieces > 8) pieces &= ~int64_t(7);
  p.chunk = (steps + pieces - 1) / pieces * step;
  p.pieces = int(std::max<int64_t>(1, (int64_t(M) + p.chunk - 1) / p.chunk));
  if (p.pieces > 8) p.pieces = (p.pieces + 7) & ~7;
  p.tiles_n = int(tn), p.tiles_k = int(tk);
  return p;
}
size_t bias_bytes(const Plan& p, int N) {
  return p.pieces == 1 ? 16 : (size_t(p.pieces) * p.tiles_k * N * sizeof(double) + 15) & ~size_t(15);
}

}  // namespace pet_wgrad

using namespace pet_wgrad;

size_t pet_linear_grads_bytes(int dtype, int M, int N, int K) {
  const Plan p = plan_of(dtype, M, N, K);
  return bias_bytes(p, N) + (p.pieces > 1 ? size_t(p.pieces) * N * K * sizeof(float) : 0);
}

// pet_linear_grads past its checks; rows at or past live_base + *live (all with no live) are not read.
int pet_linear_grads_run(int dtype, int M, int N, int K, const void* out_adj, int64_t ldo, const void* in, int64_t ldi,
                         int live_base, const int* live, float* w_adj, int64_t ldw, float* b_adj, float beta, void* ws,
                         hipStream_t st) {
  const Plan p = plan_of(dtype, M, N, K);
  double* bpart = static_cast<double*>(ws);
  float* part = reinterpret_cast<float*>(static_cast<char*>(ws) + bias_bytes(p, N));
  Args a{M, N, K, ldo, ldi, live_base, live, p.chunk, p.pieces, p.tiles_n, p.tiles_k,
         p.pieces > 1 ? part : w_adj, p.pieces > 1 ? K : ldw, bpart, b_adj, beta};
  const dim3 grid(unsigned(int64_t(p.tiles_n) * p.tiles_k * p.pieces));
  const int e = pet_typed::with_dtype(dtype, [&](auto tv) {
    using T = decltype(tv);
    constexpr int V = sizeof(T) == 4 ? 4 : 8;
    const T *g = static_cast<const T*>(out_adj), *x = static_cast<const T*>(in);
    if (p.tile == 0) hipLaunchKernelGGL((wgrad_kernel<T, 2, 4, 8, 4, V>), grid, dim3(512), 0, st, g, x, a);
    else if (p.tile == 1) hipLaunchKernelGGL((wgrad_kernel<T, 2, 2, 4, 4, V>), grid, dim3(256), 0, st, g, x, a);
    else hipLaunchKernelGGL((wgrad_kernel<T, 4, 1, 1, 4, 4>), grid, dim3(256), 0, st, g, x, a);
    return hipGetLastError() == hipSuccess ? int(PET_ATTN_OK) : int(PET_ATTN_ELAUNCH);
  });
  if (e) return e;
  if (p.pieces == 1) return PET_ATTN_OK;
  const int64_t blocks = (int64_t(N) * K + kSumElements - 1) / kSumElements + (b_adj ? (int64_t(N) + 3) / 4 : 0);
  hipLaunchKernelGGL(wgrad_sum_kernel, dim3(unsigned(blocks)), dim3(256), 0, st, N, K, p.pieces, p.pieces * p.tiles_k,
                     part, bpart, w_adj, ldw, b_adj, beta);
  return hipGetLastError() == hipSuccess ? int(PET_ATTN_OK) : int(PET_ATTN_ELAUNCH);
}

extern "C" {

size_t pet_linear_grads_workspace(int dtype, int M, int N, int K) {
  if (!pet_typed::dtype_ok(dtype) || M < 0 || N < 1 || K < 1) return 0;
  return pet_linear_grads_bytes(dtype, M, N, K);
}

int pet_linear_grads(int dtype, int M, int N, int K, const void* out_adj, int64_t ldo, const void* in, int64_t ldi,
                     const int* live, float* w_adj, int64_t ldw, float* b_adj, float beta, void* workspace,
                     size_t workspace_bytes, void* stream) {
  if (!pet_typed::dtype_ok(dtype) || M < 0 || N < 1 || K < 1) return PET_ATTN_EINVAL;
  if (!w_adj || b_adj == w_adj || ldo < N || ldi < K || ldw < K || (M > 0 && (!out_adj || !in))) return PET_ATTN_EINVAL;
  if (int64_t(N) > (int64_t(1) << 30) / K) return PET_ATTN_EINDEX;
  // (2^24 workgroups of 256 threads would come out as none: HIP takes them modulo 2^32)
  if ((int64_t(N) + 63) / 64 * ((int64_t(K) + 63) / 64) >> 24) return PET_ATTN_EINDEX;
  if (!pet_typed::element_aligned(out_adj, dtype) || !pet_typed::element_aligned(in, dtype) ||
      !pet_typed::element_aligned(w_adj, PET_DTYPE_F32) || !pet_typed::element_aligned(b_adj, PET_DTYPE_F32))
    return PET_ATTN_EALIGN;
  if (!workspace || workspace_bytes < pet_linear_grads_bytes(dtype, M, N, K)) return PET_ATTN_EWORKSPACE;
  if ((reinterpret_cast<uintptr_t>(workspace) & 15u) != 0) return PET_ATTN_EALIGN;
  return pet_linear_grads_run(dtype, M, N, K, out_adj, ldo, in, ldi, 0, live, w_adj, ldw, b_adj, beta, workspace,
                              reinterpret_cast<hipStream_t>(stream));
}

}  // extern "C"
