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
// (rare). A value below 2^-14 of the column's largest is held to 2^-36 of that.
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
template <class T>
__device__ __forceinline__ float half_of(unsigned w, int h) {
  if constexpr (std::is_same<T, __bf16>::value) return __uint_as_float(h ? w & 0xffff0000u : w << 16);
  const unsigned short s = static_cast<unsigned short>(h ? w >> 16 : w);
  return float(__builtin_bit_cast(_Float16, s));
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
  double* bout;    // [pieces][N], null: no bias
  float beta;      // with one piece
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
  const int oct = 4 * oq + g;  // this thread's eight rows of a step
  const int row0 = (is_g ? 0 : C::BN) + group * 16 * V + c;  // its LDS rows: row0 + 16 j
  const T* src = (is_g ? G : X) + (int64_t(first) + 8 * oct) * ld + col;
  unsigned raw[8][W];
  auto load = [&](int s) {
    const int rows = last - first - s * C::STEP - 8 * oct;
    const T* p = src + int64_t(s) * C::STEP * ld;
#pragma unroll
    for (int r = 0; r < 8; ++r) {
#pragma unroll
      for (int w = 0; w < W; ++w) raw[r][w] = 0;
      if (reads && r < rows) {
        if (left >= V) {
          if constexpr (W == 4) {
            const u4u q = *reinterpret_cast<const u4u*>(p + r * ld);
            raw[r][0] = q[0], raw[r][1] = q[1], raw[r][2] = q[2], raw[r][3] = q[3];
          } else {
            const u2u q = *reinterpret_cast<const u2u*>(p + r * ld);
            raw[r][0] = q[0], raw[r][1] = q[1];
          }
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j)
            if (j < left) {
              if constexpr (PAIRS) raw[r][j] = __float_as_uint(p[r * ld + j]);
              else raw[r][j / 2] |= unsigned(__builtin_bit_cast(unsigned short, p[r * ld + j])) << (16 * (j & 1));
            }
        }
      }
    }
  };

  float scale[PAIRS ? V : 1], limit[PAIRS ? V : 1];
#pragma unroll
  for (int j = 0; j < (PAIRS ? V : 1); ++j) scale[j] = 1.f, limit[j] = 0.f;
  double bsum[V];
#pragma unroll
  for (int j = 0; j < V; ++j) bsum[j] = 0.0;
  const bool bias = a.bout && is_g && k0 == 0 && reads;
  int inf = 0;

  // the step that `load` read, into LDS
  auto put = [&](int s) {
    if (!reads) return;
    u4* to = stage + (s & 1) * C::STAGE;
    if constexpr (PAIRS) {
      unsigned x[V][8];
#pragma unroll
      for (int j = 0; j < V; ++j)
#pragma unroll
        for (int r = 0; r < 8; ++r) x[j][r] = raw[r][j];
      float m[V];
      bool grew = false;
#pragma unroll
      for (int j = 0; j < V; ++j) m[j] = amax8(x[j]), grew |= m[j] > limit[j];
      const bool any = __builtin_amdgcn_ballot_w64(grew) != 0;
      if (any) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float top = max_g(m[j]);
          float f = 1.f;
          if (top > limit[j]) {
            const int k = min(12 - __builtin_amdgcn_frexp_expf(fminf(top, kFltMax)), 126);
            f = limit[j] > 0.f ? __builtin_amdgcn_ldexpf(limit[j], k - 15) : 0.f;
            scale[j] = __builtin_amdgcn_ldexpf(1.f, k);
            limit[j] = fminf(__builtin_amdgcn_ldexpf(1.f, 15 - k), kFltMax);
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
        to[slot(g, 0, row0 + 16 * j)] = hi;
        to[slot(g, 1, row0 + 16 * j)] = lo;
        if (bias) {
          float t[8];
#pragma unroll
          for (int r = 0; r < 8; ++r) t[r] = __uint_as_float(x[j][r]);
          bsum[j] += ((t[0] + t[1]) + (t[2] + t[3])) + ((t[4] + t[5]) + (t[6] + t[7]));
        }
      }
    } else {
      const unsigned flip = is_g && (s & 1) ? 0x80008000u : 0u;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        u4 even, odd;
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          even[d] = __builtin_amdgcn_perm(raw[2 * d + 1][w], raw[2 * d][w], 0x05040100u) ^ flip;
          odd[d] = __builtin_amdgcn_perm(raw[2 * d + 1][w], raw[2 * d][w], 0x07060302u) ^ flip;
        }
        to[slot(g, oq, row0 + 32 * w)] = even;
        to[slot(g, oq, row0 + 32 * w + 16)] = odd;
        if (bias) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float t[8];
#pragma unroll
            for (int r = 0; r < 8; ++r) t[r] = half_of<T>(raw[r][w], h);
            bsum[2 * w + h] += ((t[0] + t[1]) + (t[2] + t[3])) + ((t[4] + t[5]) + (t[6] + t[7]));
          }
        }
      }
    }
  };

  // ---- this wave's products
  const int rn = wave / WK * 16 * TN, rk = C::BN + wave % WK * 16 * TK;  // its LDS rows
  f4 acc[TN][TK];
#pragma unroll
  for (int i = 0; i < TN; ++i)
#pragma unroll
    for (int j = 0; j < TK; ++j) acc[i][j] = f4{0.f, 0.f, 0.f, 0.f};

  auto products = [&](int s) {
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
    u4 b[TK][2];
#pragma unroll
    for (int j = 0; j < TK; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) b[j][h] = from[slot(g, h, rk + 16 * j + c)];
    const float sg = s & 1 ? -1.f : 1.f;
#pragma unroll
    for (int i = 0; i < TN; ++i) {
      const u4 x = from[slot(g, 0, rn + 16 * i + c)], y = from[slot(g, 1, rn + 16 * i + c)];
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
    }
  };

  if (steps > 0) {
    load(0);
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

  // ---- the scales' exponents, whether an infinity came by, the bias
  if constexpr (PAIRS) {
    if (l == 0) special[wave] = 0;
    if (reads && g == 0)
#pragma unroll
      for (int j = 0; j < V; ++j) expo[row0 + 16 * j] = 1 - __builtin_amdgcn_frexp_expf(scale[j]);
    if (__builtin_amdgcn_ballot_w64(inf) != 0 && l == 0) special[wave] = 1;
  }
  double* bs = reinterpret_cast<double*>(stage);  // [8 rows' groups][BN]
  if (bias)
#pragma unroll
    for (int j = 0; j < V; ++j) bs[oct * C::BN + group * 16 * V + V * c + j] = bsum[j];
  __syncthreads();
  if (a.bout && k0 == 0)
    for (int i = threadIdx.x; i < C::BN; i += 64 * C::WAVES)
      if (n0 + i < a.N) {
        double v = 0.0;
        for (int q = 0; q < 4 * C::OQ; ++q) v += bs[q * C::BN + i];
        a.bout[int64_t(piece) * a.N + n0 + i] = v;
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

  const bool direct = a.pieces == 1;
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

// adj = beta adj + the pieces' sums in double: a thread sums every STRIPS-th
// piece of four elements, eight loads at a time, the strips are joined in order.
// (One thread an element, its loads one after the other: 24 us for 80 pieces of
// 768 x 256 against 8.)
constexpr int kStrips = 8;
__global__ void __launch_bounds__(256) wgrad_sum_kernel(int N, int K, int pieces, const float* __restrict__ part,
                                                        const double* __restrict__ bpart, float* __restrict__ w_adj,
                                                        int64_t ldw, float* __restrict__ b_adj, float beta) {
  __shared__ double sums[kStrips][32][4];
  const int64_t nk = part ? int64_t(N) * K : 0, wblocks = (nk + 127) / 128;
  const int q = threadIdx.x & 31, strip = threadIdx.x >> 5;
  const bool bias = int64_t(blockIdx.x) >= wblocks;
  const int64_t i = (int64_t(blockIdx.x) - (bias ? wblocks : 0)) * 128 + 4 * q, n = bias ? N : nk;
  double v[4] = {0.0, 0.0, 0.0, 0.0};
  if (bias) {
    for (int s = strip; s < pieces; s += kStrips)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i + e < n) v[e] += bpart[int64_t(s) * N + i + e];
  } else if (i + 4 <= n) {
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
        if (i + e < n) v[e] += part[int64_t(s) * nk + i + e];
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) sums[strip][q][e] = v[e];
  __syncthreads();
  const int t = threadIdx.x;
  const int64_t j = i - 4 * q + t;
  if (t >= 128 || j >= n) return;
  double r = 0.0;
#pragma unroll
  for (int s = 0; s < kStrips; ++s) r += sums[s][t >> 2][t & 3];
  float* o = bias ? b_adj + j : w_adj + j / K * ldw + j % K;
  *o = beta != 0.f ? float(double(beta) * *o + r) : float(r);
}

// How a product is cut: the tile and the pieces.
struct Plan {
  int64_t chunk;
  int tile, pieces, tiles_n, tiles_k;
};
constexpr int kEdge[3] = {256, 128, 64};
constexpr int kResident[3] = {256, 512, 1024};  // workgroups that the chip holds at once

Plan plan_of(int dtype, int M, int N, int K) {
  const int step = dtype == PET_DTYPE_F32 ? 32 : 64;
  Plan p{};
  auto tiles = [&](int t) {
    return ((int64_t(N) + kEdge[t] - 1) / kEdge[t]) * ((int64_t(K) + kEdge[t] - 1) / kEdge[t]);
  };
  p.tile = 2;
  if (N > 64 && K > 64) p.tile = 1;
  if (N > 128 && K > 128 && double(M) * N * K >= 4e9) p.tile = 0;
  const int64_t t = tiles(p.tile), steps = std::max<int64_t>(1, (int64_t(M) + step - 1) / step);
  int64_t pieces = std::max<int64_t>(1, std::min<int64_t>(kResident[p.tile] / t, (steps + 3) / 4));
  if (pieces > 8) pieces &= ~int64_t(7);
  p.chunk = (steps + pieces - 1) / pieces * step;
  p.pieces = int(std::max<int64_t>(1, (int64_t(M) + p.chunk - 1) / p.chunk));
  if (p.pieces > 8) p.pieces = int(std::min<int64_t>(pieces, (p.pieces + 7) & ~7));
  p.tiles_n = (N + kEdge[p.tile] - 1) / kEdge[p.tile], p.tiles_k = (K + kEdge[p.tile] - 1) / kEdge[p.tile];
  return p;
}
size_t bias_bytes(const Plan& p, int N) { return (size_t(p.pieces) * N * sizeof(double) + 15) & ~size_t(15); }

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
         p.pieces > 1 ? part : w_adj, p.pieces > 1 ? K : ldw, b_adj ? bpart : nullptr, beta};
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
  const int64_t blocks = (p.pieces > 1 ? (int64_t(N) * K + 127) / 128 : 0) + (b_adj ? (int64_t(N) + 127) / 128 : 0);
  if (blocks == 0) return PET_ATTN_OK;
  hipLaunchKernelGGL(wgrad_sum_kernel, dim3(unsigned(blocks)), dim3(256), 0, st, N, K, p.pieces,
                     p.pieces > 1 ? part : nullptr, bpart, w_adj, ldw, b_adj, beta);
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
  if (!w_adj || ldo < N || ldi < K || ldw < K || (M > 0 && (!out_adj || !in))) return PET_ATTN_EINVAL;
  if (int64_t(N) > (int64_t(1) << 30) / K) return PET_ATTN_EINDEX;
  if (!pet_typed::element_aligned(out_adj, dtype) || !pet_typed::element_aligned(in, dtype) ||
      !pet_typed::element_aligned(w_adj, PET_DTYPE_F32) || !pet_typed::element_aligned(b_adj, PET_DTYPE_F32))
    return PET_ATTN_EALIGN;
  if (!workspace || workspace_bytes < pet_linear_grads_bytes(dtype, M, N, K)) return PET_ATTN_EWORKSPACE;
  if ((reinterpret_cast<uintptr_t>(workspace) & 15u) != 0) return PET_ATTN_EALIGN;
  return pet_linear_grads_run(dtype, M, N, K, out_adj, ldo, in, ldi, 0, live, w_adj, ldw, b_adj, beta, workspace,
                              reinterpret_cast<hipStream_t>(stream));
}

}  // extern "C"
