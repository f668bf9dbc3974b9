// Attention of 16-bit rows for training (attention_typed.hip, the forward;
// attention_typed_bwd.hip): what the kernels share.
//
// For query i and key j of atom n (slots of its CSR segment) and head h,
//   s_ij = scale q_i.k_j + log cf_j + b_ij,   b_ij = table[bucket(pos_j - pos_i)][h],
//   P_ij = exp(s_ij - max_j s_ij) / sum_j,    O_i = sum_j P_ij M_ij v_j,
// M the dropout mask (0 or 1 / (1 - p)), keys with cf <= 0 left out, queries on
// edges with cf <= 0 zero. All in base 2 inside: exp(s) = 2^(s log2 e).
//
// The 16x16x32 matrix instruction of the row type: lane l = (c, g) = (l % 16, l / 16)
// holds row (A) or column (B) c at k = 8g .. 8g + 7, and of the result column c at
// rows 4g .. 4g + 3. Products that contract over tokens take the result of one
// product as the B operand of the next without an exchange: of 32 tokens,
// instruction t (0, 1) computes those 8a + 4t + r (a, r = 0 .. 3) as its rows 4a + r,
// so a lane ends with tokens 8g .. 8g + 7, which is what B wants of it. LDS rows lie
// in that order (lds_row).
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include "../../include/pet_attn.h"
#include "attn_common.h"
#include "counter_rng.h"
#include "typed.h"

namespace pet_tattn {

using pet_attn::f4;
using pet_rng::Drop;
using pet_rng::Words;
using pet_typed::u4e;

typedef unsigned u4 __attribute__((ext_vector_type(4)));
typedef unsigned u2 __attribute__((ext_vector_type(2)));
typedef int i4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr float kInf = __builtin_huge_valf();

template <class T>
__device__ __forceinline__ f4 mfma(const u4& a, const u4& b, const f4& c) {
  typedef T t8 __attribute__((ext_vector_type(8)));
  if constexpr (std::is_same<T, __bf16>::value)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(t8, a), __builtin_bit_cast(t8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(t8, a), __builtin_bit_cast(t8, b), c, 0, 0, 0);
}

// The transposing LDS read (ds_read_b64_tr_b16) on the 16 lanes of a row: lane j's
// element m is element j % 4 of what lane 4m + j / 4 addressed.
template <class T>
__device__ __forceinline__ u2 lds_tr(const T* p) {
  typedef short s4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) s4 lds_s4;
  return __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(p)));
}

// An LDS row is a token's HD dims in 16-byte pieces, piece p at p ^ row_key(row): the
// pieces that a wave reads at once, one of each of 16 rows or two of each of 16, lie in
// different banks without padding, and rows can be loaded into LDS straight from memory,
// a wave's 64 pieces in a line.
template <int HD>
__device__ __forceinline__ int row_key(int row) {
  return HD == 128 ? row & 15 : HD == 64 ? row >> 1 & 7 : row >> 2 & 3;
}

// The most slots whose atoms a workgroup holds whole.
constexpr int kShort = 128;

// Tokens a stage past that, two stages in LDS.
constexpr int kStage = 64;

// Where token k of a stage lies: of each 32, tokens 8a + 4t + r at row 16t + 4a + r; and the token of a row.
__device__ __forceinline__ int lds_row(int k) {
  return (k & ~31) | (k & 4) << 2 | (k & 24) >> 1 | (k & 3);
}
__device__ __forceinline__ int row_token(int row) {
  return (row & ~31) | (row & 12) << 1 | (row & 16) >> 2 | (row & 3);
}

// The A operand of a product over 32 staged tokens (rows base .. base + 31): row m of
// it is dim 16 j + m.
template <class T, int HD>
__device__ __forceinline__ u4 transposed(const T* rows, int base, int j, int lane) {
  const int i = lane & 15, row = 4 * (lane >> 4) + (i >> 2);
  const T* p = rows + base * HD + row * HD + ((8 * ((i & 3) >> 1 ^ row_key<HD>(row)) + 4 * (i & 1)) ^ 16 * j);
  const u2 lo = lds_tr(p), hi = lds_tr(p + 16 * HD);
  return u4{lo[0], lo[1], hi[0], hi[1]};
}
// Its plain A operand: rows 16t .. 16t + 15 of the 32 at base, dims 32 step .. + 31.
template <class T, int HD>
__device__ __forceinline__ u4 straight(const T* rows, int base, int t, int step, int lane) {
  const int c = lane & 15;
  return *reinterpret_cast<const u4*>(rows + (base + 16 * t) * HD + c * HD + (8 * (lane >> 4 ^ row_key<HD>(c)) ^ 32 * step));
}
// Dims 8 ch .. + 7 of a row into its place.
template <class T, int HD>
__device__ __forceinline__ void put_piece(T* rows, int row, int ch, const u4& x) {
  *reinterpret_cast<u4*>(rows + row * HD + 8 * (ch ^ row_key<HD>(row))) = x;
}

// Reads ahead of this are sent before what follows, which waits for them one by one: left
// to itself the compiler reads an operand, waits and multiplies, one after the other.
__device__ __forceinline__ void reads_first() { __builtin_amdgcn_sched_barrier(0); }

template <class T>
__device__ __forceinline__ u4 pack8(const float (&x)[8]) {
  return __builtin_bit_cast(u4, pet_typed::pack<T>(x));
}

__host__ __device__ inline int round_up(int64_t x, int to) { return int((x + to - 1) / to * to); }

// What every kernel of a call is given.
struct Args {
  const void* qkv;
  int64_t ldq;
  const int* off;
  const float* cf;
  int64_t ldc;
  int N, T, S, H, Hk, hd;
  float scale, scale2, inv2;  // scale, scale log2 e, and its reciprocal
  const float* table;         // [nb, H], or null
  const int* buckets;         // [2 reach + 1]
  const int* pos;             // [T]
  int nb, reach;
  Drop drop;
  bool whole;  // head_dim in pieces of 8, and a segment's offsets in 32 bits
};


// Atom n's tokens. Counts past S or past the rows would be the caller's error; they
// are cut, so that no row outside 0 .. T - 1 is touched whatever off holds.
struct Segment {
  int n, count;
  int64_t edge;  // slot s >= 1 is row edge + s
  __device__ __forceinline__ Segment(const Args& a, int n_) : n(n_) {
    const int64_t o0 = a.off[n], o1 = a.off[n + 1];
    int64_t c = o1 - o0, room = int64_t(a.T) - a.N - o0;
    c = c < a.S - 1 ? c : a.S - 1;
    c = c < room ? c : room;
    count = o0 < 0 || c < 0 ? 1 : int(c) + 1;
    edge = int64_t(a.N) + o0 - 1;
  }
  __device__ __forceinline__ int64_t row(int s) const { return s == 0 ? int64_t(n) : edge + s; }
  __device__ __forceinline__ float cf(const Args& a, int s) const { return a.cf[int64_t(n) * a.ldc + s]; }
  __device__ __forceinline__ bool key(const Args& a, int s) const { return s < count && cf(a, s) > 0.f; }
  __device__ __forceinline__ bool query(const Args& a, int s) const {
    return s < count && (s == 0 || cf(a, s) > 0.f);
  }
};

// The wave's number, known to be one for all of its lanes.
__device__ __forceinline__ int wave_of() { return __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6); }

// Dims d .. d + 7 of a row of hd, zeros past its end.
template <class T>
__device__ __forceinline__ u4 row_chunk(const T* row, int d, int hd) {
  return __builtin_bit_cast(u4, pet_typed::load_raw<T>(row, d, hd));
}

// A column of a matrix over an atom's tokens: the row of slot 0, that of slot 1 (less a
// row), and the rows' distance in bytes.
struct Column {
  const char *own, *edges;
  uint32_t ld;
  template <class T>
  __device__ __forceinline__ Column(const T* src, int64_t ld_, const Segment& seg)
      : own(reinterpret_cast<const char*>(src + int64_t(seg.n) * ld_)),
        edges(reinterpret_cast<const char*>(src + seg.edge * ld_)), ld(uint32_t(ld_ * sizeof(T))) {}
  // dims d .. of slot s (both there), where Args::whole
  __device__ __forceinline__ const char* at(int s, int d) const {
    const char* const p = s == 0 ? own : edges;
    return p + uint32_t(__umul24(uint32_t(s), ld) + 2u * uint32_t(d));
  }
};
typedef unsigned u2e __attribute__((ext_vector_type(2), aligned(2)));

__device__ __forceinline__ u4 where(bool on, const u4& x) {
  return u4{on ? x[0] : 0u, on ? x[1] : 0u, on ? x[2] : 0u, on ? x[3] : 0u};
}

__device__ __forceinline__ u4 negate_if(bool on, const u4& x) {
  const unsigned flip = on ? 0x80008000u : 0u;
  return x ^ u4{flip, flip, flip, flip};
}

// Columns of slots 0 .. n - 1 (n a multiple of 32), keys and values or queries and
// adjoints, into LDS rows, zeros where the slot's weight says that it is left out: nothing
// that a masked row holds is ever multiplied. load() sends a thread's first EACH pieces of
// both (and of a third column, where there is one), without a branch (a piece that is not
// wanted is of a place that is there), put() stores them and goes on with the rest.
// take(row k, chunk, y, z): what else is made of a piece. QUERY: queries and adjoints, the
// adjoints of odd slots negated.
template <class T, int HD, int EACH, bool WHOLE, bool QUERY, bool THIRD>
struct Staged {
  static constexpr int CH = HD / 8;
  u4 x[EACH], y[EACH], z[THIRD ? EACH : 1];
  float w[EACH];

  __device__ __forceinline__ void load(const Args& a, const T* xsrc, int64_t ldx, const T* ysrc, int64_t ldy,
                                       const T* zsrc, int64_t ldz, const Segment& seg, int i0) {
    if constexpr (!WHOLE) return;
    const int last = seg.count - 1;
    const Column xc(xsrc, ldx, seg), yc(ysrc, ldy, seg), zc(THIRD ? zsrc : xsrc, ldz, seg);
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
      const int i = i0 + j * int(blockDim.x), s = i / CH, ch = 8 * (i % CH), at = s < last ? s : last, d = ch < a.hd ? ch : 0;
      w[j] = seg.cf(a, at);
      x[j] = __builtin_bit_cast(u4, *reinterpret_cast<const u4e*>(xc.at(at, d)));
      y[j] = __builtin_bit_cast(u4, *reinterpret_cast<const u4e*>(yc.at(at, d)));
      if constexpr (THIRD) z[j] = __builtin_bit_cast(u4, *reinterpret_cast<const u4e*>(zc.at(at, d)));
    }
  }
  template <class Take>
  __device__ __forceinline__ void put(const Args& a, T* xs, const T* xsrc, int64_t ldx, T* ys, const T* ysrc, int64_t ldy,
                                      const T* zsrc, int64_t ldz, const Segment& seg, int n, const Take& take) {
    const int total = n * CH, step = int(blockDim.x);
    if constexpr (WHOLE) {
      for (int i0 = threadIdx.x;;) {
#pragma unroll
        for (int j = 0; j < EACH; ++j) {
          const int i = i0 + j * step, k = i / CH, ch = i % CH;
          if (i < total) {
            const bool on = (k < seg.count) & (8 * ch < a.hd) & ((w[j] > 0.f) | (QUERY && k == 0));
            const u4 u = where(on, x[j]), v = where(on, y[j]);
            put_piece<T, HD>(xs, lds_row(k), ch, u);
            put_piece<T, HD>(ys, lds_row(k), ch, negate_if(QUERY && (k & 1), v));
            take(k, ch, v, where(on, z[THIRD ? j : 0]));
          }
        }
        i0 += EACH * step;
        if (i0 - int(threadIdx.x) >= total) break;  // (the same for the workgroup)
        load(a, xsrc, ldx, ysrc, ldy, zsrc, ldz, seg, i0);
      }
    } else {
#pragma unroll 1
      for (int i = threadIdx.x; i < total; i += step) {
        const int k = i / CH, ch = i % CH;
        u4 u = {0u, 0u, 0u, 0u}, v = u, q = u;
        if (QUERY ? seg.query(a, k) : seg.key(a, k)) {
          const int64_t row = seg.row(k);
          u = row_chunk(xsrc + row * ldx, 8 * ch, a.hd), v = row_chunk(ysrc + row * ldy, 8 * ch, a.hd);
          if constexpr (THIRD) q = row_chunk(zsrc + row * ldz, 8 * ch, a.hd);
        }
        put_piece<T, HD>(xs, lds_row(k), ch, u);
        put_piece<T, HD>(ys, lds_row(k), ch, negate_if(QUERY && (k & 1), v));
        take(k, ch, v, q);
      }
    }
  }
};

// 16 bytes a lane from memory into LDS, a wave's 64 lanes to dst .. dst + 1 KB in their
// order (dst one for the wave).
__device__ __forceinline__ void to_lds(const void* src, void* dst) {
  __builtin_amdgcn_global_load_lds(src, reinterpret_cast<u4*>(dst), 16, 0, 0);
}
// Every load of this wave has landed.
__device__ __forceinline__ void wait_loads() {
  __builtin_amdgcn_s_waitcnt(7 << 4 | 15 << 8);  // vmcnt(0) alone
  asm volatile("" ::: "memory");
}
// The workgroup's barrier with this wave's LDS accesses done and its loads still on their
// way: a fence would wait for those too.
__device__ __forceinline__ void stage_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(15 | 3 << 14 | 7 << 4);  // lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Stages of kStage slots of two columns for kernels of 256 threads, loaded into LDS past
// the registers while the stage before is used: start() sends the loads, land() waits
// for this thread's and puts zeros over what is left out, and a stage_barrier makes the
// stage everyone's. (Not WHOLE: land() loads and stores.)
template <class T, int HD, bool WHOLE, bool QUERY>
struct Ahead {
  static constexpr int CH = HD / 8, EACH = kStage * CH / 256;
  float w[EACH];
  __device__ __forceinline__ void start(const Args& a, T* xs, const T* xsrc, int64_t ldx, T* ys, const T* ysrc,
                                        int64_t ldy, const Segment& seg, int s0) {
    if constexpr (!WHOLE) return;
    const int last = seg.count - 1, wave = wave_of();
    const Column xc(xsrc, ldx, seg), yc(ysrc, ldy, seg);
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
      const int i = threadIdx.x + 256 * j, row = i / CH, ch = 8 * (i % CH ^ row_key<HD>(row));
      const int s = s0 + row_token(row), at = s < last ? s : last, d = ch < a.hd ? ch : 0, to = (64 * wave + 256 * j) * 8;
      to_lds(xc.at(at, d), xs + to);
      to_lds(yc.at(at, d), ys + to);
      w[j] = seg.cf(a, at);
    }
  }
  __device__ __forceinline__ void land(const Args& a, T* xs, const T* xsrc, int64_t ldx, T* ys, const T* ysrc,
                                       int64_t ldy, const Segment& seg, int s0) const {
    const u4 none = {0u, 0u, 0u, 0u};
    if constexpr (WHOLE) {
      wait_loads();
#pragma unroll
      for (int j = 0; j < EACH; ++j) {
        const int i = threadIdx.x + 256 * j, row = i / CH, ch = 8 * (i % CH ^ row_key<HD>(row)), s = s0 + row_token(row);
        const bool on = (s < seg.count) & (ch < a.hd) & ((w[j] > 0.f) | (QUERY && s == 0));
        if (!on) {
          *reinterpret_cast<u4*>(xs + 8 * i) = none;
          *reinterpret_cast<u4*>(ys + 8 * i) = none;
        }
      }
    } else {
#pragma unroll 1
      for (int i = threadIdx.x; i < kStage * CH; i += 256) {
        const int s = s0 + i / CH, d = 8 * (i % CH), row = lds_row(i / CH);
        u4 u = none, v = none;
        if (QUERY ? seg.query(a, s) : seg.key(a, s)) {
          u = row_chunk(xsrc + seg.row(s) * ldx, d, a.hd);
          v = row_chunk(ysrc + seg.row(s) * ldy, d, a.hd);
        }
        put_piece<T, HD>(xs, row, i % CH, u);
        put_piece<T, HD>(ys, row, i % CH, v);
      }
    }
  }
};

// A lane's B operands of a token's own columns: dims 32 step + 8g .. + 7 of slot s, as they
// lie (own_pieces), and with zeros unless live (own_live). What comes between them is not
// waited for.
template <class T, bool WHOLE, int DS>
__device__ __forceinline__ void own_pieces(const Args& a, const T* src, int64_t ld, const Segment& seg, int s, int lane,
                                           u4 (&out)[DS]) {
  const int d0 = 8 * (lane >> 4), at = s < seg.count ? s : 0;
  if constexpr (WHOLE) {
    const Column col(src, ld, seg);
#pragma unroll
    for (int step = 0; step < DS; ++step) {
      const int d = 32 * step + d0;
      out[step] = __builtin_bit_cast(u4, *reinterpret_cast<const u4e*>(col.at(at, d < a.hd ? d : 0)));
    }
  } else {
#pragma unroll
    for (int step = 0; step < DS; ++step) out[step] = row_chunk(src + seg.row(at) * ld, 32 * step + d0, a.hd);
  }
}
template <int DS>
__device__ __forceinline__ void own_live(const Args& a, bool live, int lane, u4 (&out)[DS]) {
#pragma unroll
  for (int step = 0; step < DS; ++step) out[step] = where(live && 32 * step + 8 * (lane >> 4) < a.hd, out[step]);
}

// A row's dims d = 16 j + 4g .. + 3 of a result's tile, times f. (WHOLE: all of them or none
// are there: the way for parts of them, present if never taken, costs a store its branches.)
template <bool WHOLE, class T>
__device__ __forceinline__ void put4(T* row, const f4& x, float f, int d, int hd) {
  if (WHOLE ? d < hd : d + 4 <= hd) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int r = 0; r < 4; ++r) row[d + r] = x[r] * f;
    } else {
      typedef T t4 __attribute__((ext_vector_type(4)));
      const t4 y = {T(x[0] * f), T(x[1] * f), T(x[2] * f), T(x[3] * f)};
      *reinterpret_cast<u2e*>(row + d) = __builtin_bit_cast(u2e, y);
    }
  } else if constexpr (!WHOLE) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (d + r < hd) row[d + r] = T(x[r] * f);
  }
}

// The offset of a pair in positions as an index 0 .. 2 reach (the difference does not wrap).
__device__ __forceinline__ int pair_index(int pos_key, int pos_query, int reach) {
  int d = __builtin_elementwise_sub_sat(pos_key, pos_query);
  asm("v_med3_i32 %0, %1, %2, %3" : "=v"(d) : "v"(d), "v"(-reach), "v"(reach));
  return d + reach;
}
__device__ __forceinline__ int bucket_of(const Args& a, int i) {
  const int b = a.buckets[i];
  return b < 0 ? 0 : b >= a.nb ? a.nb - 1 : b;
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// A key's part of the exponent in base 2.
__device__ __forceinline__ float log_weight(float cf) { return log2f(cf); }

// Workgroups go round the XCDs, and so do the items of a head: block b has head
// (b / 8) % heads and items slot, slot + step, ... of it, so the heads of an atom
// run on one XCD close in time and its rows' lines meet in one L2.
struct Share {
  int head, slot, step;
  __device__ __forceinline__ explicit Share(int heads) {
    const int b = blockIdx.x;
    head = (b >> 3) % heads;
    slot = (b >> 3) / heads * 8 + (b & 7);
    step = int(gridDim.x) / heads;
  }
};

// ---- the host's half --------------------------------------------------------------

// Slots of items of a grid (Share): `items` to a whole 8, `most` at most, and no more than
// 2^31 threads hold of `heads` heads; 0 where not 8 fit.
inline int grid_slots(int64_t items, int64_t most, int heads) {
  const int64_t room = INT32_MAX / 256 / heads / 8 * 8;
  return int(std::min({(items + 7) / 8 * 8, most, room}));
}

// Arguments that forward and backward share; fills `a`.
int check_args(int dtype, const pet_attn_shape* sh, int kv_heads, const void* qkv, int64_t ldq, const int* off,
               const float* cf_seq, int64_t ldc, const pet_attn_bias* bias, const pet_dropout* dropout, Args& a);

bool narrow(const Args& a, int64_t ld);

// Rows N + off[N] .. T - 1 of x set to zero.
int zero_dead(const Args& a, void* x, int64_t ld, int width, hipStream_t st);

// f(HD, WHOLE): heads of whole pieces at the next of 32, 64 and 128 dims; the rest (a
// head_dim that is no multiple of 8, strides past 2^23) at 128, by loads of any address
// that keep few pieces on their way: with both in one kernel their registers cost the
// main path a third of its waves.
template <class F>
int with_head_dim(const Args& a, F&& f) {
  if (!a.whole) return f(std::integral_constant<int, 128>{}, std::false_type{});
  if (a.hd <= 32) return f(std::integral_constant<int, 32>{}, std::true_type{});
  if (a.hd <= 64) return f(std::integral_constant<int, 64>{}, std::true_type{});
  return f(std::integral_constant<int, 128>{}, std::true_type{});
}
template <class F>
int with_row_type(int dtype, F&& f) {
  return dtype == PET_DTYPE_BF16 ? f(__bf16{}) : f(_Float16{});
}

}  // namespace pet_tattn
