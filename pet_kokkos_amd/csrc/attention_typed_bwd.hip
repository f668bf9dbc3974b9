// The backward of attention_typed.h, the probabilities recomputed from the saved
// (max, 1/sum): with D_i = dO_i.O_i,
//   dP_ij = M_ij dO_i.v_j,   dS_ij = P_ij (dP_ij - D_i),
//   dQ_i = scale sum_j dS_ij k_j,   dK_j = scale sum_i dS_ij q_i,   dV_j = sum_i P_ij M_ij dO_i,
//   dcf_j = sum over heads and i of dS_ij / cf_j,   dtable[b][h] = sum over pairs in bucket b of dS_ij.
// Keys and values shared by a group of heads sum over it.
//
// Results repeat bit for bit. Sums of floats have one owner and a fixed order. The bias
// table's gradient is summed in LDS by the workgroup's waves at once, 32 columns a bucket,
// with 64-bit atomic additions of whole numbers, which give one sum in any order
// (Columns); the columns and then the workgroups' sums are added in order, in float64.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "../../include/pet_attn.h"
#include "attention_typed.h"

namespace pet_tattn {
namespace {

constexpr int kMaxSlots = 1024;    // workgroups a head at most (a partial sum of the table each)
constexpr int kColumns = 32;       // columns of a bucket's sum

// What the backward's kernels are given beside Args.
struct Grads {
  const void *out_adj, *out;
  int64_t ldg, ldm;
  const float* ml;
  void* adj;
  int64_t lda;
  float* delta;   // [T, H]: dO.O
  float* norms;   // [T, H] |dO|, then [T, Hk] |v|: fp16, or a table's gradient
  float* bounds;  // [N, H], where norms are, past 128 slots: of an atom's and head's |dS|
  float* cfh;     // [queries_in, N, H, S], or null
  double* part;   // [slots, H, nb], with a table's gradient
  // the pass over the keys in parts, of a group's heads by `heads_in`, of the queries by `queries_in`
  int heads_in, queries_in;
  float* kv;      // [parts, T, 2 Hk hd]: dK and dV of a part, where there is more than one
};

__device__ __forceinline__ float power_of_two(int e) { return ldexpf(1.f, e); }

// Over groups of `n` lanes (4, 8, 16) within a row of 16.
template <int n, class Join>
__device__ __forceinline__ float row_join(float x, const Join& join) {
  const auto swap = [](float v, auto ctrl) {
    return __uint_as_float(__builtin_amdgcn_update_dpp(0u, __float_as_uint(v), decltype(ctrl)::value, 0xf, 0xf, true));
  };
  x = join(x, swap(x, std::integral_constant<int, 0xB1>{}));                        // lane ^ 1
  x = join(x, swap(x, std::integral_constant<int, 0x4E>{}));                        // lane ^ 2
  if constexpr (n >= 8) x = join(x, swap(x, std::integral_constant<int, 0x141>{}));  // 7 - lane of eight
  if constexpr (n >= 16) x = join(x, swap(x, std::integral_constant<int, 0x140>{}));  // 15 - lane
  return x;
}
template <int n>
__device__ __forceinline__ float row_sum(float x) {
  return row_join<n>(x, [](float a, float b) { return a + b; });
}
template <int n>
__device__ __forceinline__ float row_max(float x) {
  return row_join<n>(x, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float wave_max(float x) {
  const auto swap = [](float v, auto ctrl) {
    return __uint_as_float(__builtin_amdgcn_update_dpp(0u, __float_as_uint(v), decltype(ctrl)::value, 0xf, 0xf, true));
  };
  x = fmaxf(x, swap(x, std::integral_constant<int, 0xB1>{}));
  x = fmaxf(x, swap(x, std::integral_constant<int, 0x4E>{}));
  x = fmaxf(x, swap(x, std::integral_constant<int, 0x141>{}));
  x = fmaxf(x, swap(x, std::integral_constant<int, 0x140>{}));
  return pet_attn::max_g(x);
}

// The power of two that brings a bound to 2^to .. 2^(to + 1); 1 for 0 and for what is not finite.
__device__ __forceinline__ float scale_to(float bound, int to) {
  if (!(bound > 0.f) || !(bound < kInf)) return 1.f;
  const int e = to - ilogbf(bound);
  return power_of_two(e > 126 ? 126 : e);
}

// Elements of one register in two sums: in one, the compiler takes fp16's dot instruction for
// them, which drops bits to one side as the matrix instruction does.
__device__ __forceinline__ float dot8(const float (&x)[8], const float (&y)[8]) {
  float even = 0.f, odd = 0.f;
#pragma unroll
  for (int e = 0; e < 8; e += 2) even = fmaf(x[e], y[e], even), odd = fmaf(x[e + 1], y[e + 1], odd);
  return even + odd;
}

// dO.O of each row and head (and |dO| and |v| where b.norms is there): a group of lanes
// takes a head's slice, eight elements each.
template <class T, int LG>
__global__ __launch_bounds__(256) void delta_kernel(Args a, Grads b) {
  const int64_t heads = int64_t(a.T) * a.H, all = heads + (b.norms ? int64_t(a.T) * a.Hk : 0);
  const int l = threadIdx.x % LG;
  for (int64_t i = (int64_t(blockIdx.x) * 256 + threadIdx.x) / LG; i < all; i += int64_t(gridDim.x) * (256 / LG)) {
    const bool q = i < heads;
    const int64_t j = q ? i : i - heads, per = q ? a.H : a.Hk, row = j / per;
    const int h = int(j - row * per);
    float x[8], y[8] = {}, most = 0.f, sq = 0.f;
    const T* p = q ? static_cast<const T*>(b.out_adj) + row * b.ldg + h * a.hd
                   : static_cast<const T*>(a.qkv) + row * a.ldq + (a.H + a.Hk + h) * a.hd;
    pet_typed::unpack<T>(__builtin_bit_cast(u4e, row_chunk(p, 8 * l, a.hd)), x);
    if (q)
      pet_typed::unpack<T>(__builtin_bit_cast(u4e, row_chunk(static_cast<const T*>(b.out) + row * b.ldm + h * a.hd, 8 * l, a.hd)), y);
#pragma unroll
    for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(x[e]));
    const float dot = row_sum<LG>(dot8(x, y));
    if (b.norms) {
      const float to_one = scale_to(row_max<LG>(most), 1);  // (a square's exponent is twice its number's)
#pragma unroll
      for (int e = 0; e < 8; ++e) sq = fmaf(x[e] * to_one, x[e] * to_one, sq);
      sq = sqrtf(row_sum<LG>(sq)) / to_one;
    }
    if (l == 0) {
      if (q) b.delta[i] = dot;
      if (b.norms) b.norms[i] = sq;
    }
  }
}

// One for the wave, and known to be.
__device__ __forceinline__ float uniform(float x) {
  return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(x)));
}

// Three maxima over the workgroup: m of every thread of every wave. room: 3 floats a wave.
__device__ __forceinline__ void block_max(float (&m)[3], float* room) {
  const int waves = int(blockDim.x >> 6), wave = wave_of();
#pragma unroll
  for (int i = 0; i < 3; ++i) m[i] = wave_max(m[i]);
  __syncthreads();
  if ((threadIdx.x & 63) == 0)
#pragma unroll
    for (int i = 0; i < 3; ++i) room[3 * wave + i] = m[i];
  __syncthreads();
  for (int w = 0; w < waves; ++w)
#pragma unroll
    for (int i = 0; i < 3; ++i) m[i] = fmaxf(m[i], room[3 * w + i]);
}

// A magnitude onto a maximum; a NaN is infinite.
__device__ __forceinline__ void onto(float& at, float x) { at = fmaxf(at, x == x ? fabsf(x) : kInf); }

// A bound of the dS of an atom and head, max |dO| max |v| / (1 - p) + max |dO.O|: a workgroup an
// atom and head. Infinite or NaN where something of them is.
__global__ __launch_bounds__(1024) void bounds_kernel(Args a, Grads b) {
  __shared__ float room[48];
  const int G = a.H / a.Hk;
  const int64_t items = int64_t(a.N) * a.H;
  for (int64_t i = blockIdx.x; i < items; i += gridDim.x) {
    const int64_t n = i / a.H;
    const int h = int(i - n * a.H);
    const Segment seg(a, int(n));
    float m[3] = {0.f, 0.f, 0.f};
    for (int s = threadIdx.x; s < seg.count; s += blockDim.x) {
      if (!seg.query(a, s)) continue;
      const int64_t row = seg.row(s);
      onto(m[0], b.norms[row * a.H + h]);
      onto(m[2], b.delta[row * a.H + h]);
      if (seg.key(a, s)) onto(m[1], b.norms[int64_t(a.T) * a.H + row * a.Hk + h / G]);
    }
    block_max(m, room);
    if (threadIdx.x == 0) b.bounds[i] = m[0] * m[1] * a.drop.scale + m[2];
  }
}

// fp16 holds down to 2^-14 at full precision, and a long row's dS lie far under the
// adjoints that they come from: those of `heads` heads from h on are scaled by the power of
// two that brings their bound to 2^14 .. 2^15. bf16 has fp32's range, and takes 1.
template <class T>
__device__ __forceinline__ float adjoint_scale(const Args& a, const Grads& b, int n, int h, int heads) {
  if constexpr (!std::is_same<T, _Float16>::value) return 1.f;
  float bound = 0.f;
  for (int i = 0; i < heads; ++i) onto(bound, b.bounds[int64_t(n) * a.H + h + i]);
  return scale_to(uniform(bound), 14);
}

// And a long row's probabilities, or a key's near the cutoff, lie as far under 1: for their
// product with dO they are scaled by the power of two that brings 1 / (1 - p), the most that
// P M is, to 2^13 .. 2^14 (P of large logits can be off to past 1), and dV is scaled back.
// Unscaled, keys of cf 1e-5 among 2500 had no dV at all.
template <class T>
__device__ __forceinline__ float probability_scale(const Args& a) {
  return std::is_same<T, _Float16>::value ? scale_to(a.drop.scale, 13) : 1.f;
}

// The matrix instruction drops what lies some bits under a sum's last, towards minus infinity:
// 2^-31 of a dP on the mean, which the sum of 10^7 pairs' dS by bucket shows (fp16, 955 atoms up
// to 202 tokens: the table's adjoint was 1.2e-6 from float64, and is 3.6e-7). So every other
// dP is formed of negated operands. Up to 128 slots every other query's dO is negated in LDS,
// and its P for their product, signs that the instructions take for nothing; past them, where
// dO comes into LDS as it is, the V of every other key, and with it the key's dS, in a lane's
// own column, whose sums take the sign at their end.
__device__ __forceinline__ bool negated(int c, int n) { return (c + n) & 1; }
// dO.O of n queries, and their negatives at + negative(n) (4 further: other banks).
__device__ __forceinline__ constexpr int negative(int n) { return n + 4; }
__device__ __forceinline__ void put_delta(float* at, int n, int q, float x) { at[q] = x, at[negative(n) + q] = -x; }

// A query's exponent: P = 2^(s - this), +inf (P = 0) for one that attends to nothing.
__device__ __forceinline__ float exponent(const Args& a, const Grads& b, int n, int h, int s, bool live) {
  if (!live) return kInf;
  const float2 v = *reinterpret_cast<const float2*>(b.ml + ((int64_t(n) * a.H + h) * a.S + s) * 2);
  return v.y == 0.f ? kInf : v.x * kLog2e - log2f(v.y);
}

// The mask of 16 keys (slots key0 ..) by 32 queries (query_row: that of query l % 32), as
// lane (c, g)'s eight queries 8g .. 8g + 7 of its key c: bit 8 r of word t is query 8g +
// 4t + r's. A block of numbers is a query's four keys, so a lane makes two of its query
// (keys 8j + 4 (l / 32) + r), eight bits, and the bytes of eight lanes are what a lane
// of the key reads. exchange: 64 bytes of LDS of the wave's own.
__device__ __forceinline__ u2 keys_mask(const Args& a, const Words& key, uint32_t query_row, int key0, int h, int lane,
                                        unsigned char* exchange) {
  unsigned byte = 0;
  Words w[2];
#pragma unroll
  for (int j = 0; j < 2; ++j)
    w[j] = a.drop.block(key, query_row, uint32_t((key0 >> 2) + 2 * j + (lane >> 5)) * uint32_t(a.H) + uint32_t(h));
#pragma unroll
  for (int i = 7; i >= 0; --i) byte = byte + byte + unsigned(Drop::number(w[i >> 2], i & 3) >= a.drop.least);
  const int c = lane & 15, g = lane >> 4;
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
  exchange[lane] = static_cast<unsigned char>(byte);
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
  __builtin_amdgcn_wave_barrier();
  const u2 got = *reinterpret_cast<const u2*>(exchange + 8 * (c & 4) + 8 * g);
  __builtin_amdgcn_wave_barrier();
  return got >> unsigned((c >> 3) * 4 + (c & 3));
}
__device__ __forceinline__ float masked(float x, const u2& bits, int t, int r) {
  return __uint_as_float(__float_as_uint(x) & unsigned(int(bits[t] << (31 - 8 * r)) >> 31));
}

struct BiasEntry {
  float value;  // table[bucket][h] log2 e
  int column;   // the bucket's first column, in bytes
};

// The bias table's gradient, sums of dS by bucket, in whole numbers of a power of two
// that brings a bound of the atom's and head's dS to 2^33 .. 2^34 (past 128 slots, where
// probabilities are small, to 2^36 .. 2^37): additions in any order give one result, so a
// bucket's 32 columns are shared by the workgroup's waves, and the LDS adds 64-bit integers to
// them at 8 cycles a wave where its fp32 addition takes 194 (a CU, measured: a lane at a time). A
// query's |dS| sum to at most about the bound, so a column holds 2^25 queries and more. The
// unit stays while bounds are within 2^-6 and 2 of it, and the columns are summed in float64
// before another is taken. A bound past fp32's range, or of what is not finite, has no unit:
// there every dS is added in float64, a column by one lane of a wave at a time (Columns::real).
//
// Four of a lane's dS at a time: under 2^30, as nearly all are, one conversion to 32 bits each.
// floor(x + 1/2): halves go up. All of them up would shift the sum of 10^7 pairs by 10^-5 of
// it, so every other one is taken as less floor(1/2 - x), whose halves go down (rounding them
// to even by an instruction of its own cost a tenth of the whole kernel: 2040 -> 2240 us).
__device__ __forceinline__ int nearest(float x) {
  int q;
  asm("v_cvt_rpi_i32_f32 %0, %1" : "=v"(q) : "v"(x));
  return q;
}
__device__ __forceinline__ int less_nearest(float x) {
  int q;
  asm("v_cvt_rpi_i32_f32 %0, -%1" : "=v"(q) : "v"(x));
  return q;
}
struct Columns {
  int64_t* at;        // [nb, kColumns]
  float units = 0.f;  // a dS of 1 counts so much (0: nothing is counted)
  bool real = false;  // the columns are float64

  __device__ __forceinline__ void clear(int nb) {
    for (int i = threadIdx.x; i < nb * kColumns; i += blockDim.x) at[i] = 0;
  }
  // For dS under a bound (one for the workgroup), brought to 2^TO .. ; sums: what a flush adds to.
  template <int TO>
  __device__ __forceinline__ void fit(float bound, int nb, double* sums) {
    constexpr float most = float(uint64_t(1) << (TO + 2)), least = float(uint64_t(1) << (TO - 6));
    const float counted = bound * units;
    if (!real && counted >= least && counted < most) return;
    const bool over = !(bound < kInf);
    if (!over && !(bound > 0.f)) return;  // (every dS is 0)
    const float one = over ? 1.f : scale_to(bound, TO);
    if (one == units && real == over) return;
    if (units > 0.f) flush(nb, sums);
    units = one, real = over;
  }
  // x: four of a lane's dS in units, onto the buckets whose first columns are at column (bytes).
  __device__ __forceinline__ void count(const int (&column)[4], const float (&x)[4]) const {
    char* const columns = reinterpret_cast<char*>(at + (threadIdx.x & (kColumns - 1)));
    const auto add = [&](int i, int64_t q) {
      __hip_atomic_fetch_add(reinterpret_cast<unsigned long long*>(columns + column[i]), static_cast<unsigned long long>(q),
                             __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    };
    const auto take = [&](int i, int64_t q) {
      __hip_atomic_fetch_sub(reinterpret_cast<unsigned long long*>(columns + column[i]), static_cast<unsigned long long>(q),
                             __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    };
    const float m = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
    if (__builtin_expect(__any(!(m < (real ? -1.f : 0x1p30f))), 0)) {
      if (real) {
        count_real(column, x);
        return;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int high = nearest(x[i] * 0x1p-16f);
        const float low = fmaf(float(high), -0x1p16f, x[i]);
        add(i, int64_t(high) << 16);
        if (i & 1) take(i, less_nearest(low)); else add(i, nearest(low));
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i & 1) take(i, less_nearest(x[i])); else add(i, nearest(x[i]));
  }
  // Eight columns a wave, eight lanes at a time: one lane to a column, in one order.
  __device__ __forceinline__ void count_real(const int (&column)[4], const float (&x)[4]) const {
    const int lane = threadIdx.x & 63;
    char* const columns = reinterpret_cast<char*>(at + 8 * wave_of() + (lane & 7));
#pragma unroll 1
    for (int turn = 0; turn < 8; ++turn) {
      if (lane >> 3 == turn)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          double* const to = reinterpret_cast<double*>(columns + column[i]);
          const double was = __hip_atomic_load(to, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
          __hip_atomic_store(to, was + double(x[i]), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
      __builtin_amdgcn_wave_barrier();
    }
  }
  // The columns summed onto a head's row of the workgroup's own sums, and cleared.
  __device__ __forceinline__ void flush(int nb, double* sums) {
    __syncthreads();
    for (int k = threadIdx.x; k < nb && units > 0.f; k += blockDim.x) {
      int64_t whole = 0;
      double sum = 0.0;
#pragma unroll 4
      for (int l = 0; l < kColumns; ++l) {
        int64_t* const column = at + k * kColumns + ((l + k) & (kColumns - 1));
        const int64_t x = *column;
        *column = 0;
        if (real) sum += __builtin_bit_cast(double, x); else whole += x;
      }
      if (!real) sum = double(whole) * double(1.f / units);
      sums[k] += sum;
    }
    __syncthreads();
  }
};
__device__ __forceinline__ void bias_entries(const Args& a, BiasEntry* lut, int h) {
  for (int i = threadIdx.x; i <= 2 * a.reach; i += blockDim.x) {
    const int bucket = bucket_of(a, i);
    lut[i] = BiasEntry{a.table[int64_t(bucket) * a.H + h] * kLog2e, bucket * kColumns * 8};
  }
}

// ---- up to 128 slots: an atom's whole backward in one workgroup ------------------------

template <int HD>
struct ShortLds {
  int rows;       // R: slots to a whole 32
  size_t stats, more, bytes;
  ShortLds(const Args& a, bool hist) : rows(round_up(a.S, 32)) {
    stats = size_t(2) * rows * HD * 2 + size_t(rows) * size_t(rows + 8) * 2;
    more = stats + size_t(rows) * 12;
    bytes = more + 4 * (64 + 16) + (a.table ? size_t(2 * a.reach + 1) * 8 : 0) + (hist ? size_t(a.nb) * kColumns * 8 : 0);
  }
};

// The larger of m and the magnitudes of a piece's elements, as 16-bit patterns (a NaN's is past infinity's).
__device__ __forceinline__ void onto_magnitude(unsigned& m, const u4& x) {
  typedef unsigned short us2 __attribute__((ext_vector_type(2)));
  us2 v = __builtin_bit_cast(us2, m);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned bits = x[i] & 0x7fff7fffu;
    v = __builtin_elementwise_max(v, __builtin_bit_cast(us2, bits));
  }
  m = __builtin_bit_cast(unsigned, v);
}
template <class T>
__device__ __forceinline__ float magnitude(unsigned m) {
  const unsigned short bits = static_cast<unsigned short>(std::max(m & 0xffffu, m >> 16));
  const float x = float(__builtin_bit_cast(T, bits));
  return x == x ? x : kInf;
}

// A wave has KT tiles of 16 keys as B operands and dK^T, dV^T in registers; a head's
// queries and adjoints are staged in LDS whole (dO.O made of the pieces as they pass),
// S = Q K^T and dP = dO V^T come with a lane's key in its column, and P and dS are the B
// operands of dV^T += dO^T P and dK^T += Q^T dS as they lie. dS goes to LDS, a key's
// queries a row, and once every wave is done with Q's rows and K's lie there, it is read
// transposed for dQ^T += K^T dS^T, a tile of queries a wave: every product is formed once,
// where the two passes past 128 slots form S, dP and their exponentials twice. dS is rounded
// to the row type for its products with Q and K, as P is for its with dO: the operands'
// type. 1728 atoms of 71 tokens, 8 heads of 32, bf16: 137 us (209 in two passes' kernels with
// all sums kept), 3.8 TB/s of what is moved once, the vector unit busy two thirds of it; 11392
// of 32 to 71, 8 heads of 64, with bias, its gradient and dropout: 2030 us, the vector unit half
// busy, waves waiting half of their time at two a SIMD, which registers bound.
// Two waves a SIMD, or three where that takes little or no scratch: with dropout 64 dims take 72
// to 108 bytes a lane at three, 32 dims in groups 72 to 104. At 128 dims, and in groups at 64,
// two take scratch as well: 156 to 356 bytes, in groups past 64 slots 84 to 200 at 64 dims and
// 1116 to 1516 at 128, some of it in the pairs' loop.
template <int HD, int KT, bool GROUP, bool BIAS>
constexpr int kShortWaves =
    HD == 128 || (KT == 2 && GROUP && (HD == 64 || BIAS)) || (HD == 64 && (BIAS || KT == 1)) ? 2 : 3;
template <class T, int HD, int KT, bool GROUP, bool WHOLE, bool BIAS, bool DROP>
__global__ __launch_bounds__(256, (kShortWaves<HD, KT, GROUP, BIAS>)) void typed_bwd_short_kernel(Args a, Grads b, int R,
                                                                                           unsigned stats, unsigned more) {
  extern __shared__ __align__(16) char lds[];
  constexpr int DS = HD / 32, DT = HD / 16, CH = HD / 8;
  constexpr int AT = GROUP ? KT : 1;  // tiles whose sums are kept: over a group's heads, or one at a time
  constexpr bool HALF = std::is_same<T, _Float16>::value;
  const int lane = threadIdx.x & 63, wave = wave_of(), waves = int(blockDim.x >> 6), c = lane & 15, g = lane >> 4;
  T* const qs = reinterpret_cast<T*>(lds);  // Q's rows, then K's
  T* const gs = qs + R * HD;                // dO's rows, every other one negated
  T* const dss = gs + R * HD;               // dS, a key's queries a row
  const int pitch = R + 8;
  float* const expo = reinterpret_cast<float*>(lds + stats);
  float* const delta = expo + R;
  int* const qpos = reinterpret_cast<int*>(delta + R);
  unsigned char* const exchange = reinterpret_cast<unsigned char*>(lds + more) + 64 * wave;
  float* const room = reinterpret_cast<float*>(lds + more + 256);
  BiasEntry* const lut = reinterpret_cast<BiasEntry*>(room + 16);
  int64_t* const columns = reinterpret_cast<int64_t*>(lut + (BIAS ? 2 * a.reach + 1 : 0));
  const int G = GROUP ? a.H / a.Hk : 1;
  const Share share(a.Hk);
  const int hk = share.head;
  const bool hist = BIAS && b.part;
  const float up = probability_scale<T>(a);
  const T* const qkv = static_cast<const T*>(a.qkv);
  const T* const kcols = qkv + (a.H + hk) * a.hd;
  const T* const vcols = qkv + (a.H + a.Hk + hk) * a.hd;
  Words key{};
  if constexpr (DROP) key = a.drop.key();
  Columns cols{columns};
  double* const sums = hist ? b.part + (int64_t(share.slot) * a.H + hk * G) * a.nb : nullptr;
  if (hist) {
    cols.clear(a.nb);
    for (int k = threadIdx.x; k < a.nb; k += blockDim.x)
      for (int i = 0; i < G; ++i) sums[i * a.nb + k] = 0.0;
  }
  if (BIAS && G == 1) bias_entries(a, lut, hk);

  for (int n = share.slot; n < a.N; n += share.step) {
    const Segment seg(a, n);
    const int rows = round_up(seg.count, 32), first = (wave + n) & (waves - 1);
    u4 kf[KT][DS], vf[KT][DS];
    f4 dk[AT][DT], dv[AT][DT];
    float weight[KT];
    int kpos[KT];
    bool klive[KT];
    unsigned vmax = 0;
    // everything that the atom is read from goes out before any of it is waited for
    float kcf[KT];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      const int s = 16 * (first + waves * kt) + c, at = s < seg.count ? s : 0;
      kcf[kt] = seg.cf(a, at);
      if constexpr (BIAS) kpos[kt] = a.pos[seg.row(at)];
      own_pieces<T, WHOLE>(a, kcols, a.ldq, seg, s, lane, kf[kt]);
      own_pieces<T, WHOLE>(a, vcols, a.ldq, seg, s, lane, vf[kt]);
    }
    const auto clear = [&](int at) {
#pragma unroll
      for (int j = 0; j < DT; ++j) dk[at][j] = dv[at][j] = f4{0.f, 0.f, 0.f, 0.f};
    };
    float sc = 1.f;
    // a tile's dK and dV to their rows
    const auto store = [&](int kt, int at) {
      const int s = 16 * (first + waves * kt) + c;
      if (s >= seg.count) return;
      T* const row = static_cast<T*>(b.adj) + seg.row(s) * b.lda;
#pragma unroll
      for (int j = 0; j < DT; ++j) {
        if (!klive[kt]) dk[at][j] = dv[at][j] = f4{0.f, 0.f, 0.f, 0.f};
        put4<WHOLE>(row + (a.H + hk) * a.hd, dk[at][j], a.scale / sc, 16 * j + 4 * g, a.hd);
        put4<WHOLE>(row + (a.H + a.Hk + hk) * a.hd, dv[at][j], 1.f / up, 16 * j + 4 * g, a.hd);
      }
    };
    if constexpr (GROUP)
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) clear(kt);
    for (int i = 0; i < G; ++i) {
      const int h = hk * G + i;
      const T* const qcols = qkv + h * a.hd;
      const T* const gcols = static_cast<const T*>(b.out_adj) + h * a.hd;
      const T* const ocols = static_cast<const T*>(b.out) + h * a.hd;
      Staged<T, HD, KT * CH / 4, WHOLE, true, true> staged;
      staged.load(a, qcols, a.ldq, gcols, b.ldg, ocols, b.ldm, seg, threadIdx.x);
      const int q = threadIdx.x, q_at = min(q, seg.count - 1);  // (threads are more than rows)
      const float q_cf = seg.cf(a, q_at);
      const float2 q_ml = *reinterpret_cast<const float2*>(b.ml + ((int64_t(n) * a.H + h) * a.S + q_at) * 2);
      int q_pos = 0;
      if constexpr (BIAS) q_pos = a.pos[seg.row(q_at)];
      stage_barrier();  // (the last head's or atom's rows are done with)
      if (i == 0) {
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
          klive[kt] = (16 * (first + waves * kt) + c < seg.count) & (kcf[kt] > 0.f);
          own_live(a, klive[kt], lane, kf[kt]);
          own_live(a, klive[kt], lane, vf[kt]);
          weight[kt] = klive[kt] ? log_weight(kcf[kt]) : -kInf;
          if (HALF || hist)
#pragma unroll
            for (int d = 0; d < DS; ++d) onto_magnitude(vmax, vf[kt][d]);
        }
      }
      if (BIAS && G > 1) bias_entries(a, lut, h);
      if (q < rows) {
        const bool on = (q < seg.count) & ((q == 0) | (q_cf > 0.f)) & (q_ml.y != 0.f);
        const float e = on ? q_ml.x * kLog2e - log2f(q_ml.y) : kInf;
        expo[q] = (DROP ? log2f(a.drop.scale) - e : -e) * a.inv2;  // P is scaled by 1 / (1 - p) with its exponent
        if constexpr (BIAS) qpos[q] = q_pos;
      }
      unsigned gmax = 0;
      float dmax = 0.f;
      staged.put(a, qs, qcols, a.ldq, gs, gcols, b.ldg, ocols, b.ldm, seg, rows,
                 [&](int k, int ch, const u4& y, const u4& o) {
                   float u[8], v[8];
                   pet_typed::unpack<T>(__builtin_bit_cast(u4e, y), u);
                   pet_typed::unpack<T>(__builtin_bit_cast(u4e, o), v);
                   const float dot = row_sum<CH>(dot8(u, v));
                   if (ch == 0) delta[k] = DROP ? dot / a.drop.scale : dot;
                   if (HALF || hist) onto_magnitude(gmax, y), dmax = fmaxf(dmax, dot == dot ? fabsf(dot) : kInf);
                 });
      if (HALF || hist) {
        const float m[3] = {wave_max(magnitude<T>(gmax)), wave_max(magnitude<T>(vmax)), wave_max(dmax)};
        if (lane == 0)
#pragma unroll
          for (int k = 0; k < 3; ++k) room[3 * wave + k] = m[k];
      }
      stage_barrier();
      // what brings dS into the range of fp16, and into whole numbers (adjoint_scale, Columns)
      float counts = 0.f;
      if (HALF || hist) {
        float m[3] = {0.f, 0.f, 0.f};
        for (int w = 0; w < waves; ++w)
#pragma unroll
          for (int k = 0; k < 3; ++k) m[k] = fmaxf(m[k], room[3 * w + k]);
        const float bound = uniform(float(a.hd) * m[0] * m[1] * a.drop.scale + m[2]);
        if (hist) cols.fit<33>(bound, a.nb, sums + i * a.nb);
        if constexpr (HALF) {
          const float was = sc;
          sc = scale_to(bound, 14);
          if (GROUP && i > 0 && sc != was)
#pragma unroll
            for (int at = 0; at < AT; ++at)
#pragma unroll
              for (int j = 0; j < DT; ++j) dk[at][j] *= sc / was;
        }
        counts = cols.units / sc;
      }
      const float back = 1.f / sc, down = sc / up;
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        const int tile = first + waves * kt;
        if (16 * tile >= seg.count) continue;
        const int at_tile = GROUP ? kt : 0;
        if constexpr (!GROUP) clear(0);
        float cf_sum = 0.f;
#pragma unroll 1
        for (int qb = 0; qb < rows; qb += 32) {
          u2 bits{};
          if constexpr (DROP) {
            const int s = qb + (lane & 31);
            bits = keys_mask(a, key, uint32_t(s < seg.count ? seg.row(s) : 0), 16 * tile, h, lane, exchange);
          }
          float p[8], ds[8];
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const int at = qb + 8 * g + 4 * t;
            f4 s = *reinterpret_cast<const f4*>(expo + at), dp = {0.f, 0.f, 0.f, 0.f};
            const f4 d4 = *reinterpret_cast<const f4*>(delta + at);
#pragma unroll
            for (int d = 0; d < DS; ++d) {
              s = mfma<T>(straight<T, HD>(qs, qb, t, d, lane), kf[kt][d], s);
              dp = mfma<T>(straight<T, HD>(gs, qb, t, d, lane), vf[kt][d], dp);
            }
            i4 qp{};
            int column[4] = {};
            float counted[4];
            if constexpr (BIAS) qp = *reinterpret_cast<const i4*>(qpos + at);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              float w = weight[kt];
              if constexpr (BIAS) {
                const BiasEntry be = lut[pair_index(kpos[kt], qp[r], a.reach)];
                w += be.value;
                column[r] = be.column;
              }
              float e = exp2_fast(fmaf(s[r], a.scale2, w));
              if constexpr (HALF) e *= up;
              float kept = e;
              if constexpr (DROP) kept = masked(e, bits, t, r);
              p[4 * t + r] = r & 1 ? -kept : kept;
              float x = fmaf(kept, r & 1 ? -dp[r] : dp[r], -e * d4[r]);
              if constexpr (HALF) x *= down;
              ds[4 * t + r] = x;
              cf_sum += x;
              counted[r] = x * counts;
            }
            if (hist) cols.count(column, counted);
          }
          const u4 pf = pack8<T>(p), df = pack8<T>(ds);
          *reinterpret_cast<u4*>(dss + (16 * tile + c) * pitch + qb + 8 * g) = df;
#pragma unroll
          for (int j = 0; j < DT; ++j) {
            dv[at_tile][j] = mfma<T>(transposed<T, HD>(gs, qb, j, lane), pf, dv[at_tile][j]);
            dk[at_tile][j] = mfma<T>(transposed<T, HD>(qs, qb, j, lane), df, dk[at_tile][j]);
          }
        }
        if (b.cfh) {
          const float sum = pet_attn::sum_g(cf_sum) * back;
          const int s = 16 * tile + c;
          if (g == 0 && s < seg.count) b.cfh[(int64_t(n) * a.H + h) * a.S + s] = sum;
        }
        if constexpr (!GROUP) store(kt, 0);
      }
      stage_barrier();
      // K's rows in the place of Q's; zeros for the tiles behind the last token's
      const u4 none = {0u, 0u, 0u, 0u};
      const auto put_keys = [&](int tile, const u4 (&k)[DS]) {
#pragma unroll
        for (int d = 0; d < DS; ++d) put_piece<T, HD>(qs, lds_row(16 * tile + c), 4 * d + g, k[d]);
        if (16 * tile >= seg.count)
          for (int qb = 0; qb < rows; qb += 32) *reinterpret_cast<u4*>(dss + (16 * tile + c) * pitch + qb + 8 * g) = none;
      };
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
        if (16 * (first + waves * kt) < rows) put_keys(first + waves * kt, kf[kt]);
      if (waves == 1) {  // (one tile of two)
        const u4 zeros[DS] = {};
        put_keys(1, zeros);
      }
      stage_barrier();
      for (int tile = first; 16 * tile < seg.count; tile += waves) {
        f4 dq[DT];
#pragma unroll
        for (int j = 0; j < DT; ++j) dq[j] = f4{0.f, 0.f, 0.f, 0.f};
        for (int kb = 0; kb < rows; kb += 32) {
          const T* const at = dss + (kb + 8 * g + (c >> 2)) * pitch + 16 * tile + 4 * (c & 3);
          const u2 lo = lds_tr(at), hi = lds_tr(at + 4 * pitch);
          const u4 df = {lo[0], lo[1], hi[0], hi[1]};
#pragma unroll
          for (int j = 0; j < DT; ++j) dq[j] = mfma<T>(transposed<T, HD>(qs, kb, j, lane), df, dq[j]);
        }
        const int s = 16 * tile + c;
        if (s < seg.count) {
          T* const row = static_cast<T*>(b.adj) + seg.row(s) * b.lda + h * a.hd;
#pragma unroll
          for (int j = 0; j < DT; ++j) put4<WHOLE>(row, dq[j], a.scale * back, 16 * j + 4 * g, a.hd);
        }
      }
      if (hist && G > 1) cols.flush(a.nb, sums + i * a.nb);
    }
    if constexpr (GROUP)
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) store(kt, kt);
  }
  if (hist && G == 1) cols.flush(a.nb, sums);
}

// ---- past 128 slots: a pass over the keys and one over the queries --------------------

template <int HD>
struct KvLds {
  static constexpr size_t rows = size_t(4) * kStage * HD * 2, queries = rows + size_t(2 * kStage) * 8 + size_t(4) * negative(kStage) * 4,
                          waves = queries + 4 * 64;  // masks
  // + the bias's entries, the buckets' columns
  static size_t bytes(const Args& a, bool hist) {
    return waves + (a.table ? size_t(2 * a.reach + 1) * 8 : 0) + (hist ? size_t(a.nb) * kColumns * 8 : 0);
  }
};

// dK, dV, the cutoff factors' and the table's adjoints: a wave has KT tiles of 16 keys
// as B operands, dK^T and dV^T in registers, and goes over all queries of the group's
// heads, staged in LDS: S = Q K^T and dP = dO V^T with a lane's key in its column, so P
// and dS are the B operands of dV^T += dO^T P and dK^T += Q^T dS as they lie. Two atoms
// of 3500 to 4096 tokens, 8 heads of 128 over 2, with a bias and its gradient: 535 us, 460
// TFLOP/s of its four products. LDS is busy 44% of that (each wave reads Q and dO twice for
// 16 keys), the vector unit 42%. Two tiles of keys a wave there halve the reads and leave one
// wave a SIMD: 647 us against 551.
template <class T, int HD, int KT, bool WHOLE, bool BIAS, bool DROP>
__global__ __launch_bounds__(256, 2) void typed_bwd_kv_kernel(Args a, Grads b, int kblocks) {
  extern __shared__ __align__(16) char lds[];
  constexpr int DS = HD / 32, DT = HD / 16, per = 4 * KT * 16;
  constexpr bool HALF = std::is_same<T, _Float16>::value;
  const int lane = threadIdx.x & 63, wave = wave_of(), c = lane & 15, g = lane >> 4;
  T* const staged = reinterpret_cast<T*>(lds);  // two stages, each Q's rows and dO's
  float* const expos = reinterpret_cast<float*>(staged + 4 * kStage * HD);
  float* const deltas = expos + 2 * kStage;
  int* const positions = reinterpret_cast<int*>(deltas + 4 * negative(kStage));
  unsigned char* const exchange = reinterpret_cast<unsigned char*>(positions + 2 * kStage) + 64 * wave;
  BiasEntry* const lut = reinterpret_cast<BiasEntry*>(positions + 2 * kStage + 64);
  int64_t* const columns = reinterpret_cast<int64_t*>(lut + (BIAS ? 2 * a.reach + 1 : 0));
  const int G = a.H / a.Hk;
  const Share share(a.Hk);
  const int hk = share.head;
  const bool hist = BIAS && b.part;
  const float up = probability_scale<T>(a);
  const T* const qkv = static_cast<const T*>(a.qkv);
  const T* const kcols = qkv + (a.H + hk) * a.hd;
  const T* const vcols = qkv + (a.H + a.Hk + hk) * a.hd;
  Words key{};
  if constexpr (DROP) key = a.drop.key();
  Columns cols{columns};
  double* const sums = hist ? b.part + (int64_t(share.slot) * a.H + hk * G) * a.nb : nullptr;
  if (hist) {
    cols.clear(a.nb);
    for (int k = threadIdx.x; k < a.nb; k += 256)
      for (int i = 0; i < G; ++i) sums[i * a.nb + k] = 0.0;
  }
  if (BIAS && G == 1) bias_entries(a, lut, hk);

  const int parts = b.heads_in * b.queries_in, items = a.N * kblocks * parts;
  for (int item = share.slot; item < items; item += share.step) {
    const int n = item / (kblocks * parts), kb = item / parts - n * kblocks, part = item % parts;
    const Segment seg(a, n);
    if (kb * per >= seg.count) continue;
    const int hi = part % b.heads_in, qi = part / b.heads_in;
    const int first_head = hi * (G / b.heads_in), last_head = first_head + G / b.heads_in;
    const int q_each = round_up((seg.count + b.queries_in - 1) / b.queries_in, kStage);
    const int q_first = min(qi * q_each, seg.count), q_last = min(q_first + q_each, seg.count);
    const float sc = adjoint_scale<T>(a, b, n, hk * G, G), back = 1.f / sc, down = sc / up;
    const bool minus = negated(c, n);
    const float sign = minus ? -1.f : 1.f;
    const int k0 = kb * per + wave * KT * 16;
    u4 kf[KT][DS], vf[KT][DS];
    f4 dk[KT][DT], dv[KT][DT];
    float weight[KT];
    int kpos[KT];
    bool klive[KT];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      const int s = k0 + 16 * kt + c;
      klive[kt] = seg.key(a, s);
      const int64_t row = klive[kt] ? seg.row(s) : 0;
      own_pieces<T, WHOLE>(a, kcols, a.ldq, seg, s, lane, kf[kt]);
      own_pieces<T, WHOLE>(a, vcols, a.ldq, seg, s, lane, vf[kt]);
      own_live(a, klive[kt], lane, kf[kt]);
      own_live(a, klive[kt], lane, vf[kt]);
#pragma unroll
      for (int d = 0; d < DS; ++d) vf[kt][d] = negate_if(minus, vf[kt][d]);
      weight[kt] = klive[kt] ? log_weight(seg.cf(a, s)) : -kInf;
      if constexpr (BIAS) kpos[kt] = a.pos[row];
#pragma unroll
      for (int j = 0; j < DT; ++j) dk[kt][j] = dv[kt][j] = f4{0.f, 0.f, 0.f, 0.f};
    }
    for (int i = first_head; i < last_head; ++i) {
      const int h = hk * G + i;
      float cf_sum[KT] = {};
      const T* const qcols = qkv + h * a.hd;
      const T* const gcols = static_cast<const T*>(b.out_adj) + h * a.hd;
      Ahead<T, HD, WHOLE, true> ahead;
      float next_expo = 0.f, next_delta = 0.f;
      int next_pos = 0;
      const auto start = [&](int q0, int to) {
        T* const qs = staged + to * 2 * kStage * HD;
        ahead.start(a, qs, qcols, a.ldq, qs + kStage * HD, gcols, b.ldg, seg, q0);
        if (threadIdx.x < kStage) {
          const int s = q0 + int(threadIdx.x);
          const bool on = seg.query(a, s);
          const int64_t row = on ? seg.row(s) : 0;
          next_expo = exponent(a, b, n, h, s, on);
          next_delta = on ? b.delta[row * a.H + h] : 0.f;
          if constexpr (BIAS) next_pos = a.pos[row];
        }
      };
      const auto land = [&](int q0, int to) {
        T* const qs = staged + to * 2 * kStage * HD;
        ahead.land(a, qs, qcols, a.ldq, qs + kStage * HD, gcols, b.ldg, seg, q0);
        if (threadIdx.x < kStage) {
          const int q = to * kStage + int(threadIdx.x);
          // P is scaled by 1 / (1 - p) with its exponent
          expos[q] = DROP ? log2f(a.drop.scale) - next_expo : -next_expo;
          put_delta(deltas + to * 2 * negative(kStage), kStage, int(threadIdx.x), DROP ? next_delta / a.drop.scale : next_delta);
          if constexpr (BIAS) positions[q] = next_pos;
        }
        stage_barrier();
      };
      stage_barrier();  // (the stages and the bias of the head before are done with)
      if (hist) cols.fit<36>(uniform(b.bounds[int64_t(n) * a.H + h]), a.nb, sums + i * a.nb);
      const float counts = sign * cols.units * back;
      if (BIAS && G > 1) bias_entries(a, lut, h);
      if (q_first < q_last) start(q_first, 0), land(q_first, 0);
      int at_stage = 0;
      for (int q0 = q_first; q0 < q_last; q0 += kStage, at_stage ^= 1) {
        const int n_queries = min(kStage, round_up(seg.count - q0, 32));
        const bool more = q0 + kStage < q_last;
        if (more) start(q0 + kStage, at_stage ^ 1);
        const T *const qs = staged + at_stage * 2 * kStage * HD, *const gs = qs + kStage * HD;
        const float *const expo = expos + at_stage * kStage, *const delta = deltas + at_stage * 2 * negative(kStage) + (minus ? negative(kStage) : 0);
        const int* const qpos = positions + at_stage * kStage;
        float part_sum[KT] = {};
        for (int qb = 0; qb < n_queries && k0 < seg.count; qb += 32) {
          u2 bits[KT];
          if constexpr (DROP) {
            const int s = q0 + qb + (lane & 31);
            const uint32_t row = uint32_t(s < seg.count ? seg.row(s) : 0);
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) bits[kt] = keys_mask(a, key, row, k0 + 16 * kt, h, lane, exchange);
          }
          u4 pf[KT], df[KT];
          float p[KT][8], ds[KT][8];
          f4 s2[2][KT], dp2[2][KT], d2[2];
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const int at = qb + 8 * g + 4 * t;
            u4 qf[DS], gf[DS];
            d2[t] = *reinterpret_cast<const f4*>(delta + at);
#pragma unroll
            for (int d = 0; d < DS; ++d) {
              qf[d] = straight<T, HD>(qs, qb, t, d, lane);
              gf[d] = straight<T, HD>(gs, qb, t, d, lane);
            }
            reads_first();
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) s2[t][kt] = dp2[t][kt] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int d = 0; d < DS; ++d)
#pragma unroll
              for (int kt = 0; kt < KT; ++kt) {
                s2[t][kt] = mfma<T>(qf[d], kf[kt][d], s2[t][kt]);
                dp2[t][kt] = mfma<T>(gf[d], vf[kt][d], dp2[t][kt]);
              }
          }
          u4 gt[DT];
#pragma unroll
          for (int j = 0; j < DT; ++j) gt[j] = transposed<T, HD>(gs, qb, j, lane);
          reads_first();
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            // (added here: in the products' sums it would round each of them at its own size)
            const f4 d4 = d2[t], e4 = *reinterpret_cast<const f4*>(expo + qb + 8 * g + 4 * t);
            i4 qp{};
            if constexpr (BIAS) qp = *reinterpret_cast<const i4*>(qpos + qb + 8 * g + 4 * t);
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) {
              int column[4] = {};
              float counted[4];
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                float w = weight[kt] + e4[r];
                BiasEntry be{};
                if constexpr (BIAS) {
                  be = lut[pair_index(kpos[kt], qp[r], a.reach)];
                  w += be.value;
                  column[r] = be.column;
                }
                float e = exp2_fast(fmaf(s2[t][kt][r], a.scale2, w));
                if constexpr (HALF) e *= up;
                float kept = e;
                if constexpr (DROP) kept = masked(e, bits[kt], t, r);
                p[kt][4 * t + r] = kept;
                float x = fmaf(kept, dp2[t][kt][r], -e * d4[r]);
                if constexpr (HALF) x *= down;
                ds[kt][4 * t + r] = x;
                part_sum[kt] += x;
                counted[r] = x * counts;
              }
              if (hist) cols.count(column, counted);
            }
          }
#pragma unroll
          for (int kt = 0; kt < KT; ++kt) pf[kt] = pack8<T>(p[kt]), df[kt] = pack8<T>(ds[kt]);
#pragma unroll
          for (int j = 0; j < DT; ++j)
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) dv[kt][j] = mfma<T>(gt[j], pf[kt], dv[kt][j]);
          u4 qt[DT];
#pragma unroll
          for (int j = 0; j < DT; ++j) qt[j] = transposed<T, HD>(qs, qb, j, lane);
          reads_first();
#pragma unroll
          for (int j = 0; j < DT; ++j)
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) dk[kt][j] = mfma<T>(qt[j], df[kt], dk[kt][j]);
        }
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) cf_sum[kt] += part_sum[kt];  // (a stage's sum at a time, for its roundings)
        if (more) land(q0 + kStage, at_stage ^ 1);
      }
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        const float sum = pet_attn::sum_g(cf_sum[kt]) * sign * back;
        const int s = k0 + 16 * kt + c;
        if (b.cfh && g == 0 && s < seg.count) b.cfh[((int64_t(qi) * a.N + n) * a.H + h) * a.S + s] = sum;
      }
      if (hist && G > 1) cols.flush(a.nb, sums + i * a.nb);
    }
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      const int s = k0 + 16 * kt + c;
      if (s >= seg.count) continue;
      T* const row = static_cast<T*>(b.adj) + seg.row(s) * b.lda;
      float* const sums_row = b.kv + ((int64_t(part) * a.T + seg.row(s)) * 2 * a.Hk + hk) * a.hd;
#pragma unroll
      for (int j = 0; j < DT; ++j) {
        if (!klive[kt]) dk[kt][j] = dv[kt][j] = f4{0.f, 0.f, 0.f, 0.f};
        const int d = 16 * j + 4 * g;
        if (parts > 1) {
          put4<WHOLE>(sums_row, dk[kt][j], sign * a.scale * back, d, a.hd);
          put4<WHOLE>(sums_row + a.Hk * a.hd, dv[kt][j], 1.f / up, d, a.hd);
        } else {
          put4<WHOLE>(row + (a.H + hk) * a.hd, dk[kt][j], sign * a.scale * back, d, a.hd);
          put4<WHOLE>(row + (a.H + a.Hk + hk) * a.hd, dv[kt][j], 1.f / up, d, a.hd);
        }
      }
    }
  }
  if (hist && G == 1) cols.flush(a.nb, sums);
}

// dQ: a wave has QT tiles of 16 queries as B operands and goes over the keys: S^T and
// dP^T with a lane's query in its column, dS^T the B operand of dQ^T += K^T dS^T. The same
// case: 285 us, 650 TFLOP/s of its three products, the exponentials between them (the vector
// unit is busy 45% of it, the matrix unit 30%).
template <class T, int HD, int QT, bool WHOLE, bool BIAS, bool DROP>
__global__ __launch_bounds__(256, 2) void typed_bwd_q_kernel(Args a, Grads b, int qblocks) {
  extern __shared__ __align__(16) char lds[];
  constexpr int DS = HD / 32, DT = HD / 16, per = 4 * QT * 16;
  constexpr bool HALF = std::is_same<T, _Float16>::value;
  const int lane = threadIdx.x & 63, wave = wave_of(), c = lane & 15, g = lane >> 4;
  T* const staged = reinterpret_cast<T*>(lds);  // two stages, each K's rows and V's
  float* const weights = reinterpret_cast<float*>(staged + 4 * kStage * HD);
  int* const positions = reinterpret_cast<int*>(weights + 2 * kStage);
  float* const lut = reinterpret_cast<float*>(positions + 2 * kStage);
  const Share share(a.H);
  const int h = share.head, hk = h / (a.H / a.Hk);
  const T* const qkv = static_cast<const T*>(a.qkv);
  const T* const qcols = qkv + h * a.hd;
  const T* const gcols = static_cast<const T*>(b.out_adj) + h * a.hd;
  const T* const kcols = qkv + (a.H + hk) * a.hd;
  const T* const vcols = qkv + (a.H + a.Hk + hk) * a.hd;
  Words key{};
  if constexpr (DROP) key = a.drop.key();
  if constexpr (BIAS)
    for (int i = threadIdx.x; i <= 2 * a.reach; i += 256)
      lut[i] = a.table[int64_t(bucket_of(a, i)) * a.H + h] * kLog2e;

  const int items = a.N * qblocks;
  for (int item = share.slot; item < items; item += share.step) {
    const int n = item / qblocks, qb = item - n * qblocks;
    const Segment seg(a, n);
    if (qb * per >= seg.count) continue;
    const float sc = adjoint_scale<T>(a, b, n, h, 1), back = 1.f / sc;
    const int q0 = qb * per + wave * QT * 16;
    u4 qf[QT][DS], gf[QT][DS];
    f4 dq[QT][DT];
    float expo[QT], delta[QT];
    int qpos[QT];
    int64_t qrow[QT];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      const int s = q0 + 16 * qt + c;
      const bool on = seg.query(a, s);
      qrow[qt] = on ? seg.row(s) : 0;
      own_pieces<T, WHOLE>(a, qcols, a.ldq, seg, s, lane, qf[qt]);
      own_pieces<T, WHOLE>(a, gcols, b.ldg, seg, s, lane, gf[qt]);
      own_live(a, on, lane, qf[qt]);
      own_live(a, on, lane, gf[qt]);
      expo[qt] = exponent(a, b, n, h, s, on);
      if constexpr (DROP) expo[qt] -= log2f(a.drop.scale);
      delta[qt] = on ? b.delta[qrow[qt] * a.H + h] / a.drop.scale : 0.f;
      if constexpr (BIAS) qpos[qt] = a.pos[qrow[qt]];
#pragma unroll
      for (int j = 0; j < DT; ++j) dq[qt][j] = f4{0.f, 0.f, 0.f, 0.f};
    }
    Ahead<T, HD, WHOLE, false> ahead;
    float next_weight = 0.f;
    int next_pos = 0;
    const auto start = [&](int k0, int to) {
      T* const ks = staged + to * 2 * kStage * HD;
      ahead.start(a, ks, kcols, a.ldq, ks + kStage * HD, vcols, a.ldq, seg, k0);
      if (threadIdx.x < kStage) {
        const int s = k0 + int(threadIdx.x);
        next_weight = s < seg.count ? seg.cf(a, s) : 0.f;
        if constexpr (BIAS) next_pos = s < seg.count ? a.pos[seg.row(s)] : 0;
      }
    };
    const auto land = [&](int k0, int to) {
      T* const ks = staged + to * 2 * kStage * HD;
      ahead.land(a, ks, kcols, a.ldq, ks + kStage * HD, vcols, a.ldq, seg, k0);
      if (threadIdx.x < kStage) {
        weights[to * kStage + threadIdx.x] = next_weight > 0.f ? log_weight(next_weight) * a.inv2 : -kInf;
        if constexpr (BIAS) positions[to * kStage + threadIdx.x] = next_pos;
      }
      stage_barrier();
    };
    stage_barrier();  // (the last item's stages are done with)
    start(0, 0);
    land(0, 0);
    int at_stage = 0;
    for (int k0 = 0; k0 < seg.count; k0 += kStage, at_stage ^= 1) {
      const int n_keys = min(kStage, round_up(seg.count - k0, 32));
      const bool more = k0 + kStage < seg.count;
      if (more) start(k0 + kStage, at_stage ^ 1);
      const T *const ks = staged + at_stage * 2 * kStage * HD, *const vs = ks + kStage * HD;
      const float* const weight = weights + at_stage * kStage;
      const int* const kpos = positions + at_stage * kStage;
      for (int kb = 0; kb < n_keys && q0 < seg.count; kb += 32) {
        float ds[QT][8];
        f4 s2[2][QT], dp2[2][QT];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          u4 kf[DS], vf[DS];
          const f4 w4 = *reinterpret_cast<const f4*>(weight + kb + 8 * g + 4 * t);
#pragma unroll
          for (int d = 0; d < DS; ++d) kf[d] = straight<T, HD>(ks, kb, t, d, lane), vf[d] = straight<T, HD>(vs, kb, t, d, lane);
          reads_first();
#pragma unroll
          for (int qt = 0; qt < QT; ++qt) s2[t][qt] = w4, dp2[t][qt] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int d = 0; d < DS; ++d)
#pragma unroll
            for (int qt = 0; qt < QT; ++qt) {
              s2[t][qt] = mfma<T>(kf[d], qf[qt][d], s2[t][qt]);
              dp2[t][qt] = mfma<T>(vf[d], gf[qt][d], dp2[t][qt]);
            }
        }
        u4 ktr[DT];
#pragma unroll
        for (int j = 0; j < DT; ++j) ktr[j] = transposed<T, HD>(ks, kb, j, lane);
        reads_first();
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int at = kb + 8 * g + 4 * t;
          i4 kp{};
          if constexpr (BIAS) kp = *reinterpret_cast<const i4*>(kpos + at);
#pragma unroll
          for (int qt = 0; qt < QT; ++qt) {
            Words w{};
            if constexpr (DROP)
              w = a.drop.block(key, uint32_t(qrow[qt]), uint32_t((k0 + at) >> 2) * uint32_t(a.H) + uint32_t(h));
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              float x = -expo[qt];
              if constexpr (BIAS) x += lut[pair_index(kp[r], qpos[qt], a.reach)];
              float e = exp2_fast(fmaf(s2[t][qt][r], a.scale2, x));
              if constexpr (HALF) e *= sc;
              float kept = e;
              if constexpr (DROP) kept = Drop::number(w, r) >= a.drop.least ? e : 0.f;
              ds[qt][4 * t + r] = fmaf(kept, dp2[t][qt][r], -e * delta[qt]);
            }
          }
        }
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) {
          const u4 df = pack8<T>(ds[qt]);
#pragma unroll
          for (int j = 0; j < DT; ++j)
            dq[qt][j] = mfma<T>(ktr[j], df, dq[qt][j]);
        }
      }
      if (more) land(k0 + kStage, at_stage ^ 1);
    }
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      const int s = q0 + 16 * qt + c;
      if (s >= seg.count) continue;
      T* const row = static_cast<T*>(b.adj) + seg.row(s) * b.lda + h * a.hd;
#pragma unroll
      for (int j = 0; j < DT; ++j) put4<WHOLE>(row, dq[qt][j], a.scale * back, 16 * j + 4 * g, a.hd);
    }
  }
}

// dK and dV of the parts, summed in order and rounded once: a wave has a token's row, a lane four
// columns of it. It goes by atoms and slots as the pass does, so that rows which are no atom's stay.
template <class T>
__global__ __launch_bounds__(256) void typed_kv_sum_kernel(Args a, Grads b) {
  const int width = 2 * a.Hk * a.hd, parts = b.heads_in * b.queries_in, lane = threadIdx.x & 63;
  const int slots = a.N * a.S;  // (parts are of fewer than 512 blocks of slots)
  for (int slot = int(blockIdx.x) * 4 + wave_of(); slot < slots; slot += int(gridDim.x) * 4) {
    const int n = slot / a.S, s = slot - n * a.S;
    const Segment seg(a, n);
    if (s >= seg.count) continue;
    const int64_t row = seg.row(s);
    T* const to = static_cast<T*>(b.adj) + row * b.lda + a.H * a.hd;
    for (int c = 4 * lane; c < width; c += 256) {
      const int count = min(4, width - c);
      float sum[4] = {};
      for (int p = 0; p < parts; ++p) {
        const float* const from = b.kv + (int64_t(p) * a.T + row) * width + c;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (e < count) sum[e] += from[e];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < count) to[c + e] = T(sum[e]);
    }
  }
}

// What is left to sum, one launch of both: workgroups h < tables take a head's table adjoint,
// table_adj[b][h] = beta table_adj[b][h] + the passes' workgroups' sums, 16 strips of them in
// order, in double (1024 threads); the rest the cutoff factors' adjoints, the heads' sums over
// cf. (Two launches: 4 us more a call.)
__global__ __launch_bounds__(1024) void typed_sums_kernel(Args a, Grads b, int slots, int tables, float* table_adj,
                                                          float* cf_adj, int64_t ldc, float beta) {
  __shared__ double strips[16][64];
  if (int(blockIdx.x) < tables) {
    const int h = blockIdx.x, k = threadIdx.x & 63, strip = threadIdx.x >> 6;
    double sum = 0.0;
    if (k < a.nb)
      for (int s = strip; s < slots; s += 16) sum += b.part[(int64_t(s) * a.H + h) * a.nb + k];
    strips[strip][k] = sum;
    __syncthreads();
    if (strip || k >= a.nb) return;
    sum = 0.0;
    for (int i = 0; i < 16; ++i) sum += strips[i][k];
    float* const to = table_adj + int64_t(k) * a.H + h;
    *to = float(beta == 0.f ? sum : double(beta) * *to + sum);
    return;
  }
  const int64_t all = int64_t(a.N) * a.S, step = int64_t(int(gridDim.x) - tables) * blockDim.x;
  for (int64_t i = int64_t(int(blockIdx.x) - tables) * blockDim.x + threadIdx.x; i < all; i += step) {
    const int64_t n = i / a.S;
    const int s = int(i - n * a.S);
    const Segment seg(a, int(n));
    float sum = 0.f;
    if (seg.key(a, s)) {
      for (int h = 0; h < a.H; ++h)
        for (int p = 0; p < b.queries_in; ++p) sum += b.cfh[((int64_t(p) * a.N + n) * a.H + h) * a.S + s];
      sum /= seg.cf(a, s);
    }
    float* const to = cf_adj + n * ldc + s;
    *to = beta == 0.f ? sum : fmaf(beta, *to, sum);
  }
}

constexpr size_t aligned(size_t n) { return (n + 255) & ~size_t(255); }

// Tiles of 16 keys a wave of the pass over the keys, by head_dim: two share each read of
// the staged queries, where their dK and dV leave registers for the rest.
template <int HD>
constexpr int kKeyTiles = HD == 128 ? 1 : 2;

// The parts of the pass over the keys: a chip holds two workgroups a CU of it, so with
// fewer than 512 of them a group's heads, then the queries, are shared out, at the cost of
// writing and reading fp32 sums.
struct Parts {
  int heads = 1, queries = 1;
  Parts(int N, int S, int H, int Hk, int hd) {
    if (S <= kShort) return;
    const int tile = 64 * (hd > 64 ? kKeyTiles<128> : kKeyTiles<64>), G = H / Hk;
    const int64_t have = std::max<int64_t>(1, int64_t(N) * ((int64_t(S) + tile - 1) / tile) * Hk);
    const int64_t want = (512 + have - 1) / have;
    while (heads < G && (heads < want || G % heads != 0)) ++heads;
    queries = int(std::min<int64_t>((want + heads - 1) / heads, (int64_t(S) + 511) / 512));
  }
};

struct Workspace {
  size_t delta, norms, bounds, cfh, part, kv, bytes;
  Workspace(int dtype, const pet_attn_shape& s, int kv_heads, int nb) {
    const size_t T = size_t(s.n_rows), H = size_t(s.heads);
    const Parts parts(s.n_atoms, s.slots, s.heads, kv_heads, s.head_dim);
    delta = 0;
    norms = delta + aligned(T * H * 4);
    bounds = norms + (dtype == PET_DTYPE_F16 || nb ? aligned(T * (H + size_t(kv_heads)) * 4) : 0);
    cfh = bounds + aligned((dtype == PET_DTYPE_F16 || nb) && s.slots > kShort ? size_t(s.n_atoms) * H * 4 : 0);
    part = cfh + aligned(size_t(parts.queries) * size_t(s.n_atoms) * H * size_t(s.slots) * 4);
    kv = part + aligned(size_t(kMaxSlots) * H * size_t(nb) * 8);
    const size_t all = size_t(parts.heads) * size_t(parts.queries);
    bytes = kv + (all > 1 ? aligned(all * T * 2 * size_t(kv_heads) * size_t(s.head_dim) * 4) : 0);
  }
};

}  // namespace
}  // namespace pet_tattn

using namespace pet_tattn;

extern "C" size_t pet_attn_bwd_typed_workspace(int dtype, const pet_attn_shape* shape, int kv_heads, int n_buckets) {
  if (!shape || (dtype != PET_DTYPE_BF16 && dtype != PET_DTYPE_F16) || kv_heads < 1 || shape->heads < 1 ||
      shape->heads % kv_heads != 0 || shape->n_atoms < 0 || shape->n_rows < 0 || shape->slots < 1 || shape->head_dim < 1 ||
      shape->head_dim > 128 || n_buckets < 0 || n_buckets > PET_BIAS_MAX_BUCKETS)
    return 0;
  return Workspace(dtype, *shape, kv_heads, n_buckets).bytes;
}

extern "C" int pet_attn_bwd_typed(int dtype, const pet_attn_shape* shape, int kv_heads, const void* qkv, int64_t ldq,
                                  const int* off, const void* dmerged, int64_t ldg, const void* merged, int64_t ldm,
                                  const float* ml, const float* cf_seq, int64_t ldc, const pet_attn_bias* bias,
                                  const pet_dropout* dropout, void* qkv_adj, int64_t lda, float* cf_seq_adj,
                                  int64_t ldca, float* table_adj, float beta, void* workspace, size_t workspace_bytes,
                                  void* stream) {
  Args a;
  if (const int e = check_args(dtype, shape, kv_heads, qkv, ldq, off, cf_seq, ldc, bias, dropout, a)) return e;
  const int D = a.H * a.hd, W = (a.H + 2 * a.Hk) * a.hd;
  if ((a.T > 0 && (!dmerged || !merged || !qkv_adj)) || (a.N > 0 && !ml) || ldg < D || ldm < D || lda < W)
    return PET_ATTN_EINVAL;
  if ((cf_seq_adj && ldca < a.S) || (table_adj && !bias)) return PET_ATTN_EINVAL;
  const auto in_place = [](const void* to, std::initializer_list<const void*> from) {
    return to && std::find(from.begin(), from.end(), to) != from.end();
  };
  if ((a.T > 0 && in_place(qkv_adj, {qkv, dmerged, merged})) || in_place(cf_seq_adj, {cf_seq, ml}) ||
      in_place(table_adj, {a.table, cf_seq, ml}))
    return PET_ATTN_EINVAL;
  if (table_adj && a.H > 1 << 20) return PET_ATTN_EINDEX;  // (threads of typed_sums_kernel)
  for (const void* p : {dmerged, merged, static_cast<const void*>(qkv_adj)})
    if (!pet_typed::element_aligned(p, dtype)) return PET_ATTN_EALIGN;
  if ((reinterpret_cast<uintptr_t>(ml) & 7u) != 0 || !pet_typed::element_aligned(cf_seq_adj, PET_DTYPE_F32) ||
      !pet_typed::element_aligned(table_adj, PET_DTYPE_F32))
    return PET_ATTN_EALIGN;
  const Workspace ws(dtype, *shape, kv_heads, a.nb);
  if (!workspace || workspace_bytes < ws.bytes) return PET_ATTN_EWORKSPACE;
  if ((reinterpret_cast<uintptr_t>(workspace) & 15u) != 0) return PET_ATTN_EALIGN;
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  char* const base = static_cast<char*>(workspace);
  a.whole = a.whole && narrow(a, ldg) && narrow(a, ldm);
  const bool half = dtype == PET_DTYPE_F16;
  const Parts parts(a.N, a.S, a.H, a.Hk, a.hd);
  const auto at = [&](size_t offset) { return reinterpret_cast<float*>(base + offset); };
  const Grads b{dmerged, merged, ldg, ldm, ml, qkv_adj, lda, at(ws.delta), half || table_adj ? at(ws.norms) : nullptr,
                half || table_adj ? at(ws.bounds) : nullptr, cf_seq_adj ? at(ws.cfh) : nullptr,
                table_adj ? reinterpret_cast<double*>(base + ws.part) : nullptr, parts.heads, parts.queries, at(ws.kv)};
  if (shape->dead && a.T > 0)
    if (const int e = zero_dead(a, qkv_adj, lda, W, st)) return e;
  int slots = 0;
  const auto launched = [] { return hipGetLastError() == hipSuccess ? int(PET_ATTN_OK) : int(PET_ATTN_ELAUNCH); };
  const int err = a.N == 0 ? int(PET_ATTN_OK) : with_row_type(dtype, [&](auto tv) {
    using T = decltype(tv);
    return with_head_dim(a, [&](auto hc, auto wc) {
      constexpr int HD = decltype(hc)::value;
      constexpr bool WHOLE = decltype(wc)::value;
      const auto run = [&](auto bc, auto dc) {
        constexpr bool BIAS = decltype(bc)::value, DROP = decltype(dc)::value;
        if (a.S <= kShort) {
          const ShortLds<HD> l(a, b.part != nullptr);
          const auto kernel = a.S <= 64     ? typed_bwd_short_kernel<T, HD, 1, true, WHOLE, BIAS, DROP>
                              : a.H > a.Hk ? typed_bwd_short_kernel<T, HD, 2, true, WHOLE, BIAS, DROP>
                                           : typed_bwd_short_kernel<T, HD, 2, false, WHOLE, BIAS, DROP>;
          if (const int e = pet_attn::raise_lds(reinterpret_cast<const void*>(kernel), l.bytes)) return e;
          slots = grid_slots(a.N, b.part ? std::clamp(4096 / a.Hk / 8 * 8, 8, kMaxSlots) : 4096, a.Hk);
          if (slots == 0) return int(PET_ATTN_EINDEX);
          hipLaunchKernelGGL(kernel, dim3(unsigned(slots * a.Hk)), dim3(a.S <= 16 ? 64 : a.S <= 32 ? 128 : 256), l.bytes, st, a, b,
                             l.rows, unsigned(l.stats), unsigned(l.more));
          return launched();
        }
        {
          const int64_t groups = int64_t(a.T) * (a.H + (b.norms ? a.Hk : 0));
          const unsigned blocks = unsigned(std::min<int64_t>((groups * (HD / 8) + 255) / 256, 16384));
          hipLaunchKernelGGL((delta_kernel<T, HD / 8>), dim3(blocks), dim3(256), 0, st, a, b);
          if (const int e = launched()) return e;
          if (b.norms) {
            const int64_t items = int64_t(a.N) * a.H;
            hipLaunchKernelGGL(bounds_kernel, dim3(unsigned(std::min<int64_t>(items, 16384))), dim3(a.S > 512 ? 1024 : 256), 0, st,
                               a, b);
            if (const int e = launched()) return e;
          }
        }
        {
          constexpr int KT = kKeyTiles<HD>;
          const auto kernel = typed_bwd_kv_kernel<T, HD, KT, WHOLE, BIAS, DROP>;
          const int blocks = (a.S + KT * 64 - 1) / (KT * 64);
          const int64_t items = int64_t(a.N) * blocks * parts.heads * parts.queries;
          const size_t bytes = KvLds<HD>::bytes(a, b.part != nullptr);
          if (const int e = pet_attn::raise_lds(reinterpret_cast<const void*>(kernel), bytes)) return e;
          slots = grid_slots(items, b.part ? std::clamp(2048 / a.Hk / 8 * 8, 8, kMaxSlots) : kMaxSlots, a.Hk);
          if (slots == 0) return int(PET_ATTN_EINDEX);
          hipLaunchKernelGGL(kernel, dim3(unsigned(slots * a.Hk)), dim3(256), bytes, st, a, b, blocks);
          if (const int e = launched()) return e;
          if (parts.heads * parts.queries > 1) {
            const int64_t token_slots = int64_t(a.N) * a.S;
            hipLaunchKernelGGL(typed_kv_sum_kernel<T>, dim3(unsigned(std::min<int64_t>((token_slots + 3) / 4, 8192))), dim3(256), 0,
                               st, a, b);
            if (const int e = launched()) return e;
          }
        }
        {
          constexpr int QT = 2;
          const auto kernel = typed_bwd_q_kernel<T, HD, QT, WHOLE, BIAS, DROP>;
          const int blocks = (a.S + QT * 64 - 1) / (QT * 64);
          const size_t bytes = size_t(2 * kStage) * (2 * HD * 2 + 8) + (a.table ? size_t(2 * a.reach + 1) * 4 : 0);
          if (const int e = pet_attn::raise_lds(reinterpret_cast<const void*>(kernel), bytes)) return e;
          const int q_slots = grid_slots(int64_t(a.N) * blocks, 2048, a.H);
          if (q_slots == 0) return int(PET_ATTN_EINDEX);
          hipLaunchKernelGGL(kernel, dim3(unsigned(q_slots * a.H)), dim3(256), bytes, st, a, b, blocks);
          return launched();
        }
      };
      if (a.table) return dropout ? run(std::true_type{}, std::true_type{}) : run(std::true_type{}, std::false_type{});
      return dropout ? run(std::false_type{}, std::true_type{}) : run(std::false_type{}, std::false_type{});
    });
  });
  if (err) return err;
  const int tables = table_adj ? a.H : 0, threads = table_adj ? 1024 : 256;
  const int64_t cfs = cf_seq_adj && a.N > 0
                          ? std::min<int64_t>((int64_t(a.N) * a.S + threads - 1) / threads, (1 << 22) / threads) : 0;
  if (tables + cfs > 0) {
    hipLaunchKernelGGL(typed_sums_kernel, dim3(unsigned(tables + cfs)), dim3(threads), 0, st, a, b, slots, tables, table_adj,
                       cf_seq_adj, ldca, beta);
    if (hipGetLastError() != hipSuccess) return PET_ATTN_ELAUNCH;
  }
  return PET_ATTN_OK;
}
