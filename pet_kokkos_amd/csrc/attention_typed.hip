// The forward of attention_typed.h: one pass over an atom's keys with each query's
// running maximum and sum.
//
// A workgroup has a head and goes through its items, (atom, block of queries): its
// waves hold QT tiles of 16 queries each as B operands in registers; keys and values
// are staged in LDS, masked ones as zeros with a weight of -inf, and S^T = K Q^T
// comes with a lane's query in its column, so maxima and sums are the lane's own but
// for two lane swaps, and P^T is the B operand of O^T += V^T P^T as it lies. log cf
// is the product's first summand, the bias a gather from LDS by the pair's offset. The
// probabilities are rounded to the row type for their product with V, whose operands are
// of that type; their sum is of the unrounded ones.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "../../include/pet_attn.h"
#include "attention_typed.h"

namespace pet_tattn {
namespace {

template <int HD>
constexpr int fwd_stage_bytes(int keys) { return keys * (2 * HD * 2 + 8); }

// The tiles of 16 queries at q[], QT of them, against staged keys kb .. kb + 32 U - 1
// (slots k0 + kb ..; those past n_keys do not count): scores, the running maximum and sum,
// and the products with the values onto o.
template <class T, int HD, int QT, int U, bool WHOLE, bool BIAS, bool DROP>
struct Tiles {
  static constexpr int DS = HD / 32, DT = HD / 16;
  // Operands read ahead of their products: two waves a SIMD need it, and have the registers.
  static constexpr bool EAGER = QT > 1;
  u4 qf[QT][DS];
  f4 o[QT][DT];
  float top[QT], base[QT], sum[QT];  // the largest logit, what exponents are taken from, their sum (log2 units)
  int64_t row[QT];
  float cf[QT];
  int pos[QT];
  bool live[QT];

  __device__ __forceinline__ void load(const Args& a, const T* qcols, const Segment& seg, int q0, int lane) {
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      const int s = q0 + 16 * qt + (lane & 15), at = s < seg.count ? s : 0;
      row[qt] = seg.row(at);
      cf[qt] = seg.cf(a, at);
      if constexpr (BIAS) pos[qt] = a.pos[row[qt]];
      own_pieces<T, WHOLE>(a, qcols, a.ldq, seg, s, lane, qf[qt]);
    }
  }
  __device__ __forceinline__ void start(const Args& a, const Segment& seg, int q0, int lane) {
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      const int s = q0 + 16 * qt + (lane & 15);
      live[qt] = (s < seg.count) & ((s == 0) | (cf[qt] > 0.f));
      own_live(a, live[qt], lane, qf[qt]);
#pragma unroll
      for (int j = 0; j < DT; ++j) o[qt][j] = f4{0.f, 0.f, 0.f, 0.f};
      top[qt] = base[qt] = -kInf, sum[qt] = 0.f;
    }
  }

  // the biases of four keys
  __device__ __forceinline__ void gather(const Args& a, float (&b)[QT][2][4], int t, const int* kpos, const float* lut) {
    const i4 kp = *reinterpret_cast<const i4*>(kpos);
#pragma unroll
    for (int qt = 0; qt < QT; ++qt)
#pragma unroll
      for (int r = 0; r < 4; ++r) b[qt][t][r] = lut[pair_index(kp[r], pos[qt], a.reach)];
  }

  __device__ __forceinline__ void keys(const Args& a, const Words& key, int h, const T* ks, const T* vs,
                                       const float* weight, const int* kpos, const float* lut, int k0, int kb, int n_keys,
                                       int lane) {
    const int g = lane >> 4;
    f4 s[QT][U][2];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (kb + 32 * u >= n_keys) {
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) s[qt][u][0] = s[qt][u][1] = f4{-kInf, -kInf, -kInf, -kInf};
        continue;
      }
      u4 kf[2][DS];
      float b[QT][2][4];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int at = kb + 32 * u + 8 * g + 4 * t;
        const f4 w = *reinterpret_cast<const f4*>(weight + at);
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) s[qt][u][t] = w;
        if constexpr (EAGER) {
#pragma unroll
          for (int d = 0; d < DS; ++d) kf[t][d] = straight<T, HD>(ks, kb + 32 * u, t, d, lane);
          if constexpr (BIAS) gather(a, b, t, kpos + at, lut);
        }
      }
      if constexpr (EAGER) reads_first();
#pragma unroll
      for (int d = 0; d < DS; ++d)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const u4 k = EAGER ? kf[t][d] : straight<T, HD>(ks, kb + 32 * u, t, d, lane);
#pragma unroll
          for (int qt = 0; qt < QT; ++qt) s[qt][u][t] = mfma<T>(k, qf[qt][d], s[qt][u][t]);
        }
      if constexpr (BIAS)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if constexpr (!EAGER) gather(a, b, t, kpos + kb + 32 * u + 8 * g + 4 * t, lut);
#pragma unroll
          for (int qt = 0; qt < QT; ++qt)
#pragma unroll
            for (int r = 0; r < 4; ++r) s[qt][u][t][r] = fmaf(s[qt][u][t][r], a.scale2, b[qt][t][r]);
        }
    }
    // the values' operands, on their way while the probabilities are made
    u4 vt[U][DT];
    if constexpr (EAGER) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (u == 0 || kb + 32 * u < n_keys)
#pragma unroll
          for (int j = 0; j < DT; ++j) vt[u][j] = transposed<T, HD>(vs, kb + 32 * u, j, lane);
      reads_first();
    }
    const float f = BIAS ? 1.f : a.scale2;
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      float m = -kInf;
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) m = fmaxf(m, s[qt][u][t][r]);
      top[qt] = fmaxf(top[qt], pet_attn::max_g(m) * f);
      // The sums move to a larger base only where the maximum has passed it by 2^8 (or is
      // the first): their 4 HD / 16 products a tile were a fifth of a step's instructions.
      if (__any(top[qt] > base[qt] + 8.f)) {
        const float now = top[qt] == -kInf ? 0.f : top[qt];
        if (k0 + kb > 0) {
          const float fade = exp2_fast(base[qt] - now);
          sum[qt] *= fade;
#pragma unroll
          for (int j = 0; j < DT; ++j) o[qt][j] *= fade;
        }
        base[qt] = top[qt];
      }
      const float from = base[qt] == -kInf ? 0.f : base[qt];
      u4 pf[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (u > 0 && kb + 32 * u >= n_keys) continue;
        float p[8];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          Words w{};
          if constexpr (DROP)
            w = a.drop.block(key, uint32_t(row[qt]),
                             uint32_t((k0 + kb + 32 * u + 8 * g + 4 * t) >> 2) * uint32_t(a.H) + uint32_t(h));
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float x = s[qt][u][t][r];
            float e = exp2_fast(BIAS ? x - from : fmaf(x, f, -from));
            sum[qt] += e;
            if constexpr (DROP) e = Drop::number(w, r) >= a.drop.least ? e : 0.f;
            p[4 * t + r] = e;
          }
        }
        pf[u] = pack8<T>(p);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (u > 0 && kb + 32 * u >= n_keys) continue;
#pragma unroll
        for (int j = 0; j < DT; ++j)
          o[qt][j] = mfma<T>(EAGER ? vt[u][j] : transposed<T, HD>(vs, kb + 32 * u, j, lane), pf[u], o[qt][j]);
      }
    }
  }

  __device__ __forceinline__ void finish(const Args& a, const Segment& seg, int h, int q0, int lane, T* merged,
                                         int64_t ldm, float* ml) {
    const int c = lane & 15, g = lane >> 4;
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
      const int s = q0 + 16 * qt + c;
      const float l = pet_attn::sum_g(sum[qt]);
      const bool some = live[qt] && l != 0.f;
      const float inv = some ? 1.f / l : 0.f;
      if (ml && g == 0 && s < a.S)
        *reinterpret_cast<float2*>(ml + ((int64_t(seg.n) * a.H + h) * a.S + s) * 2) =
            make_float2(some ? top[qt] * kLn2 : 0.f, inv * exp2_fast(some ? top[qt] - base[qt] : 0.f));
      if (s < seg.count) {
        T* const to = merged + seg.row(s) * ldm + h * a.hd;
        const float f = DROP ? inv * a.drop.scale : inv;
#pragma unroll
        for (int j = 0; j < DT; ++j) {
          if (!some) o[qt][j] = f4{0.f, 0.f, 0.f, 0.f};
          // (at 64 dims with a bias and dropout the short way moved the stores, 711 -> 787 us; at 32 dims it
          // took 69 -> 66; past 128 slots at 128 it made no difference)
          put4<WHOLE && HD == 32>(to, o[qt][j], f, 16 * j + 4 * g, a.hd);
        }
      }
    }
  }
};

__device__ __forceinline__ void fill_lut(const Args& a, float* lut, int h) {
  for (int i = threadIdx.x; i <= 2 * a.reach; i += blockDim.x)
    lut[i] = a.table[int64_t(bucket_of(a, i)) * a.H + h] * kLog2e;
}

// Up to 128 slots: an item is an atom, all of its keys staged at once, its tiles of
// queries dealt to the workgroup's waves (4 from 33 slots on: a workgroup's waves start
// at one SIMD, and 5 of them, one a tile of 71 slots, left room for no third workgroup
// on the CU; which wave has the odd tile goes round by the atom). 1728 atoms of 71
// tokens, 8 heads of 32, bf16: 66 us, 3.9 TB/s of Q, K, V and the result, each moved once
// (a copy reaches 5.0), the vector unit issuing 98% of the time; 11392 of 32 to 71, 8 heads of
// 64, with bias and dropout: 712 us, 3.4 TB/s, the vector unit (exponentials, the bias, the
// random numbers) 77%.
// Four waves a SIMD up to 64 dims (with dropout 64 take 24 bytes of scratch a lane); with bias
// and dropout 64 are compiled for three, which runs the batch in 712 us where four takes 724.
template <int HD, bool BIAS, bool DROP>
constexpr int kFwdWaves = HD == 128 ? 2 : HD == 64 && BIAS && DROP ? 3 : 4;
template <class T, int HD, bool WHOLE, bool BIAS, bool DROP>
__global__ __launch_bounds__(256, (kFwdWaves<HD, BIAS, DROP>)) void typed_fwd_short_kernel(Args a, int keys, T* merged,
                                                                                           int64_t ldm, float* ml) {
  extern __shared__ __align__(16) char lds[];
  T* const ks = reinterpret_cast<T*>(lds);
  T* const vs = ks + keys * HD;
  float* const weight = reinterpret_cast<float*>(vs + keys * HD);
  int* const kpos = reinterpret_cast<int*>(weight + keys);
  float* const lut = reinterpret_cast<float*>(kpos + keys);
  const int lane = threadIdx.x & 63, wave = wave_of(), waves = int(blockDim.x >> 6);
  const Share share(a.H);
  const int h = share.head, hk = h / (a.H / a.Hk);
  const T* const qkv = static_cast<const T*>(a.qkv);
  const T* const qcols = qkv + h * a.hd;
  const T* const kcols = qkv + (a.H + hk) * a.hd;
  const T* const vcols = qkv + (a.H + a.Hk + hk) * a.hd;
  Words key{};
  if constexpr (DROP) key = a.drop.key();
  if constexpr (BIAS) fill_lut(a, lut, h);
  const int slots = (a.S + 15) >> 4;
  for (int n = share.slot; n < a.N; n += share.step) {
    const Segment seg(a, n);
    const int n_keys = round_up(seg.count, 32), tiles = (seg.count + 15) >> 4;
    // everything that the atom is read from goes out before any of it is waited for
    int tile = (wave + n) & (waves - 1);
    Tiles<T, HD, 1, 2, WHOLE, BIAS, DROP> q;
    Staged<T, HD, HD == 32 ? 2 : 4, WHOLE, false, false> staged;
    staged.load(a, kcols, a.ldq, vcols, a.ldq, kcols, a.ldq, seg, threadIdx.x);
    q.load(a, qcols, seg, 16 * tile, lane);
    const int k_at = min(int(threadIdx.x), seg.count - 1);  // (threads are more than n_keys)
    const float w = seg.cf(a, k_at);
    int p = 0;
    if constexpr (BIAS) p = a.pos[seg.row(k_at)];
    stage_barrier();  // (the last atom's rows are done with)
    if (int(threadIdx.x) < n_keys) {
      weight[threadIdx.x] = int(threadIdx.x) < seg.count && w > 0.f ? log_weight(w) * a.inv2 : -kInf;
      if constexpr (BIAS) kpos[threadIdx.x] = p;
    }
    staged.put(a, ks, kcols, a.ldq, vs, vcols, a.ldq, kcols, a.ldq, seg, n_keys,
               [](int, int, const u4&, const u4&) {});
    stage_barrier();
    while (tile < slots) {
      q.start(a, seg, 16 * tile, lane);
      if (tile < tiles)
        for (int kb = 0; kb < n_keys; kb += 64) q.keys(a, key, h, ks, vs, weight, kpos, lut, 0, kb, n_keys, lane);
      q.finish(a, seg, h, 16 * tile, lane, merged, ldm, ml);
      tile += waves;
      if (tile < slots) q.load(a, qcols, seg, 16 * tile, lane);
    }
  }
}

// Past 128 slots: an item is an atom's 128 queries, two tiles a wave, and the keys come in
// stages, the next one's loads on their way into LDS while the present one is used. Two
// atoms of 3500 to 4096 tokens, 8 heads of 128 over 2, with a bias: 190 us, 650 TFLOP/s
// (a library's large product: 1143); the exponentials and the bias' gathers stand between
// the products (vector unit 61%, matrix unit 27% of the time). Two tiles a wave share each read of K and V.
template <class T, int HD, bool WHOLE, bool BIAS, bool DROP>
__global__ __launch_bounds__(256, 2) void typed_fwd_long_kernel(Args a, int qblocks, T* merged, int64_t ldm, float* ml) {
  extern __shared__ __align__(16) char lds[];
  constexpr int QT = 2, per = 4 * QT * 16, U = HD == 128 ? 1 : 2;
  T* const rows = reinterpret_cast<T*>(lds);  // two stages, each K's rows and V's
  float* const weights = reinterpret_cast<float*>(rows + 4 * kStage * HD);
  int* const positions = reinterpret_cast<int*>(weights + 2 * kStage);
  float* const lut = reinterpret_cast<float*>(positions + 2 * kStage);
  const int lane = threadIdx.x & 63, wave = wave_of();
  const Share share(a.H);
  const int h = share.head, hk = h / (a.H / a.Hk);
  const T* const qkv = static_cast<const T*>(a.qkv);
  const T* const qcols = qkv + h * a.hd;
  const T* const kcols = qkv + (a.H + hk) * a.hd;
  const T* const vcols = qkv + (a.H + a.Hk + hk) * a.hd;
  Words key{};
  if constexpr (DROP) key = a.drop.key();
  if constexpr (BIAS) fill_lut(a, lut, h);
  const int items = a.N * qblocks;
  for (int item = share.slot; item < items; item += share.step) {
    const int n = item / qblocks, qb = item - n * qblocks;
    const Segment seg(a, n);
    const int q0 = qb * per + wave * QT * 16;
    Tiles<T, HD, QT, U, WHOLE, BIAS, DROP> q;
    q.load(a, qcols, seg, q0, lane);
    q.start(a, seg, q0, lane);
    if (qb * per < seg.count) {  // (the same for the whole workgroup)
      Ahead<T, HD, WHOLE, false> ahead;
      float next_weight = 0.f;
      int next_pos = 0;
      const auto start = [&](int k0, int to) {
        T* const ks = rows + to * 2 * kStage * HD;
        ahead.start(a, ks, kcols, a.ldq, ks + kStage * HD, vcols, a.ldq, seg, k0);
        if (threadIdx.x < kStage) {
          const int k = k0 + int(threadIdx.x);
          next_weight = k < seg.count ? seg.cf(a, k) : 0.f;
          if constexpr (BIAS) next_pos = k < seg.count ? a.pos[seg.row(k)] : 0;
        }
      };
      const auto land = [&](int k0, int to) {
        T* const ks = rows + to * 2 * kStage * HD;
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
      int at = 0;
      for (int k0 = 0; k0 < seg.count; k0 += kStage, at ^= 1) {
        const bool more = k0 + kStage < seg.count;
        if (more) start(k0 + kStage, at ^ 1);
        if (q0 < seg.count) {
          const T* const ks = rows + at * 2 * kStage * HD;
          const int n_keys = min(kStage, round_up(seg.count - k0, 32));
          for (int kb = 0; kb < n_keys; kb += 32 * U)
            q.keys(a, key, h, ks, ks + kStage * HD, weights + at * kStage, positions + at * kStage, lut, k0, kb, n_keys,
                   lane);
        }
        if (more) land(k0 + kStage, at ^ 1);
      }
    }
    q.finish(a, seg, h, q0, lane, merged, ldm, ml);
  }
}

template <class T>
__global__ __launch_bounds__(256) void zero_dead_kernel(const int* off, int N, int rows, int width, T* x, int64_t ld) {
  int64_t first = int64_t(N) + off[N];
  first = first < 0 ? 0 : first;
  for (int64_t r = first + blockIdx.x; r < rows; r += gridDim.x)
    for (int c = threadIdx.x; c < width; c += 256) x[r * ld + c] = T(0.f);
}

}  // namespace

int zero_dead(const Args& a, void* x, int64_t ld, int width, hipStream_t st) {
  typedef unsigned short u16;
  hipLaunchKernelGGL(zero_dead_kernel<u16>, dim3(unsigned(std::min(a.T, 2048))), dim3(256), 0, st, a.off, a.N, a.T,
                     width, static_cast<u16*>(x), ld);
  return hipGetLastError() == hipSuccess ? PET_ATTN_OK : PET_ATTN_ELAUNCH;
}

// Whether a segment's offsets of a matrix are the product of 24-bit numbers under 2^32.
bool narrow(const Args& a, int64_t ld) {
  return ld < (1 << 23) && a.S < (1 << 24) && int64_t(a.S) * ld * 2 < INT64_C(1) << 32;
}

int check_args(int dtype, const pet_attn_shape* sh, int kv_heads, const void* qkv, int64_t ldq, const int* off,
               const float* cf_seq, int64_t ldc, const pet_attn_bias* bias, const pet_dropout* dropout, Args& a) {
  if (!sh || (dtype != PET_DTYPE_BF16 && dtype != PET_DTYPE_F16)) return PET_ATTN_EINVAL;
  if (sh->n_atoms < 0 || sh->n_rows < sh->n_atoms || sh->slots < 1 || sh->heads < 1) return PET_ATTN_EINVAL;
  if (sh->head_dim < 1 || sh->head_dim > 128) return PET_ATTN_EHEADDIM;
  if (kv_heads < 1 || sh->heads % kv_heads != 0) return PET_ATTN_EINVAL;
  const int64_t width = (int64_t(sh->heads) + 2 * int64_t(kv_heads)) * sh->head_dim;
  if (width > INT32_MAX) return PET_ATTN_EINDEX;
  if (!off || ldq < width || ldc < sh->slots) return PET_ATTN_EINVAL;
  if ((sh->n_rows > 0 && !qkv) || (sh->n_atoms > 0 && !cf_seq)) return PET_ATTN_EINVAL;
  const float scale2 = sh->scale * kLog2e;
  if (!(sh->scale > 0.f) || !std::isfinite(scale2) || !std::isfinite(1.f / scale2)) return PET_ATTN_EINVAL;
  // a query's dropout counter, key / 4 by head, is 32 bits; an item's number is an int
  if ((int64_t(sh->slots) + 3) / 4 * sh->heads > int64_t(UINT32_MAX)) return PET_ATTN_EINDEX;
  if (int64_t(sh->n_atoms) * ((int64_t(sh->slots) + 15) / 16) > (1 << 30)) return PET_ATTN_EINDEX;
  a = Args{};
  if (bias) {
    if (!bias->table || !bias->buckets || (sh->n_rows > 0 && !bias->positions)) return PET_ATTN_EINVAL;
    if (bias->n_buckets < 1 || bias->n_buckets > PET_BIAS_MAX_BUCKETS || bias->reach < 0 ||
        bias->reach > PET_BIAS_MAX_REACH)
      return PET_ATTN_EINVAL;
    for (const void* p : {static_cast<const void*>(bias->table), static_cast<const void*>(bias->buckets),
                          static_cast<const void*>(bias->positions)})
      if (!pet_typed::element_aligned(p, PET_DTYPE_F32)) return PET_ATTN_EALIGN;
    a.table = bias->table, a.buckets = bias->buckets, a.pos = bias->positions;
    a.nb = bias->n_buckets, a.reach = bias->reach;
  }
  if (dropout)
    if (const int e = pet_rng::make_drop(dropout, a.drop)) return e;
  if (!pet_typed::element_aligned(qkv, dtype) || !pet_typed::element_aligned(off, PET_DTYPE_F32) ||
      !pet_typed::element_aligned(cf_seq, PET_DTYPE_F32))
    return PET_ATTN_EALIGN;
  a.qkv = qkv, a.ldq = ldq, a.off = off, a.cf = cf_seq, a.ldc = ldc;
  a.N = sh->n_atoms, a.T = sh->n_rows, a.S = sh->slots, a.H = sh->heads, a.Hk = kv_heads, a.hd = sh->head_dim;
  a.scale = sh->scale, a.scale2 = scale2, a.inv2 = 1.f / scale2;
  a.whole = a.hd % 8 == 0 && narrow(a, ldq);
  return PET_ATTN_OK;
}

}  // namespace pet_tattn

using namespace pet_tattn;

extern "C" int pet_attn_fwd_typed(int dtype, const pet_attn_shape* shape, int kv_heads, const void* qkv, int64_t ldq,
                                  const int* off, const float* cf_seq, int64_t ldc, const pet_attn_bias* bias,
                                  const pet_dropout* dropout, void* merged, int64_t ldm, float* ml, void* stream) {
  Args a;
  if (const int e = check_args(dtype, shape, kv_heads, qkv, ldq, off, cf_seq, ldc, bias, dropout, a)) return e;
  const int D = a.H * a.hd;
  if ((a.T > 0 && !merged) || ldm < D) return PET_ATTN_EINVAL;
  if (!pet_typed::element_aligned(merged, dtype) || (reinterpret_cast<uintptr_t>(ml) & 7u) != 0) return PET_ATTN_EALIGN;
  if (a.T == 0) return PET_ATTN_OK;
  if (merged == qkv || (ml && ml == cf_seq)) return PET_ATTN_EINVAL;  // in place
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (shape->dead)
    if (const int e = zero_dead(a, merged, ldm, D, st)) return e;
  if (a.N == 0) return PET_ATTN_OK;
  return with_row_type(dtype, [&](auto tv) {
    using T = decltype(tv);
    return with_head_dim(a, [&](auto hc, auto wc) {
      constexpr int HD = decltype(hc)::value;
      constexpr bool WHOLE = decltype(wc)::value;
      const auto run = [&](auto bc, auto dc) {
        constexpr bool BIAS = decltype(bc)::value, DROP = decltype(dc)::value;
        const size_t lut = a.table ? size_t(2 * a.reach + 1) * 4 : 0;
        const int64_t qblocks = a.S <= kShort ? 1 : (int64_t(a.S) + 127) / 128;
        const int slots = grid_slots(a.N * qblocks, 2048, a.H);
        if (slots == 0) return int(PET_ATTN_EINDEX);
        if (a.S <= kShort) {
          const auto kernel = typed_fwd_short_kernel<T, HD, WHOLE, BIAS, DROP>;
          const int keys = round_up(a.S, 32);
          const size_t bytes = size_t(fwd_stage_bytes<HD>(keys)) + lut;
          if (const int e = pet_attn::raise_lds(reinterpret_cast<const void*>(kernel), bytes)) return e;
          hipLaunchKernelGGL(kernel, dim3(unsigned(slots * a.H)), dim3(a.S <= 16 ? 64 : a.S <= 32 ? 128 : 256), bytes, st, a,
                             keys, static_cast<T*>(merged), ldm, ml);
        } else {
          const auto kernel = typed_fwd_long_kernel<T, HD, WHOLE, BIAS, DROP>;
          const size_t bytes = size_t(2 * fwd_stage_bytes<HD>(kStage)) + lut;
          if (const int e = pet_attn::raise_lds(reinterpret_cast<const void*>(kernel), bytes)) return e;
          hipLaunchKernelGGL(kernel, dim3(unsigned(slots * a.H)), dim3(256), bytes, st, a, int(qblocks),
                             static_cast<T*>(merged), ldm, ml);
        }
        return hipGetLastError() == hipSuccess ? int(PET_ATTN_OK) : int(PET_ATTN_ELAUNCH);
      };
      if (a.table) return dropout ? run(std::true_type{}, std::true_type{}) : run(std::true_type{}, std::false_type{});
      return dropout ? run(std::false_type{}, std::true_type{}) : run(std::false_type{}, std::false_type{});
    });
  });
}
