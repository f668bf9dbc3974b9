// The token norm for training on gfx950: rows in fp32, bf16 or fp16 up to 16384
// wide, and the backward with the parameters' gradients. In fp32:
//   xhat = (x - mu) inv, inv = 1 / sqrt(mean((x - mu)^2) + eps), mu = 0 for RMSNorm
//   out = xhat w (+ b)
//   in_adj = beta in_adj + inv (g w - [mean(g w), LayerNorm] - xhat mean(g w xhat))
//   w_adj = beta_w w_adj + sum over rows of g xhat, b_adj the same of g.
//
// Both directions are bound by HBM (about 16 flops an element for 6 to 12
// bytes), so a row is read once, 16 bytes a lane, and stays in registers between
// its sums and its result. In the backward a lane keeps the same columns of
// every row it meets, so that the parameters' gradients are sums in its
// registers over a workgroup's rows; a workgroup's sums meet in LDS and go to
// one row of the workspace, whose rows a second kernel adds in double and in
// order. Nothing is atomic: results repeat bit for bit. 498338 x 512 in bf16 takes
// 296 us (5.2 TB/s), 27318 x 128 in fp32 14.4, its two launches' host side; 2000 x 16384
// in fp32 104 (3.8 TB/s: a workgroup a CU, no row ahead). fp32 rows of 1025 to 4096
// columns that are no multiple of four spill 8 to 36 bytes a lane (8193 x 3001 71 us).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "../../include/pet_attn.h"
#include "gemm_common.h"
#include "typed.h"

namespace pet_norm {

using pet_typed::kVec;
using pet_typed::live_rows;
using pet_typed::u4e;

constexpr float kRmsEps = 1.1920928955078125e-07f;  // float32 epsilon
constexpr float kLnEps = 1e-5f;

// A launch's threads at most: HIP takes them modulo 2^32 and reports nothing
// (2^28 + 21 rows of 16 lanes in one: all but the first rows left as they were).
constexpr int64_t kLaunchThreads = int64_t(1) << 31;

constexpr int threads_of(int TPR) { return TPR > 256 ? TPR : 256; }
// Waves a SIMD of the backward, by the elements a lane holds (x, g, the weight and
// the two sums, and the next row's raw ones): the registers are held to it, so
// that a grid of it fills the chip in one round. (1024 workgroups of which 768
// fitted took two: 65536 x 1024 in bf16 131 us.)
constexpr int waves_of(int E, int TPR) { return TPR == 1024 ? 4 : E <= 4 ? 8 : E <= 8 ? 5 : E <= 16 ? 3 : 2; }
// 1 / sqrt(x): the hardware's estimate and a Newton step (0 where the squares passed
// fp32, as 1 / sqrtf gives).
__device__ __forceinline__ float rsqrt_nr(float x) {
  const float y = __builtin_amdgcn_rsqf(x);
  return y == 0.f ? y : y * fmaf(-0.5f * x * y, y, 1.5f);
}

// A lane's value from the lane that a DPP control names.
template <int ctrl>
__device__ __forceinline__ float dpp(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), ctrl, 0xf, 0xf, true));
}
// A row's sums over its TPR threads, the same bits in each of them: in registers
// over the lanes (quads, halves and whole rows of 16 by DPP, then the rows of 16
// exchanged) and, where a row is the whole workgroup's, the waves' sums in order
// through LDS (`red`, double-buffered by `turn`, so that a sum costs one barrier).
template <int TPR, int n>
__device__ __forceinline__ void row_sums(float (&x)[n], float (*red)[2][3], int& turn) {
#pragma unroll
  for (int i = 0; i < n; ++i) {
    x[i] += dpp<0xb1>(x[i]);   // quad_perm 1, 0, 3, 2
    x[i] += dpp<0x4e>(x[i]);   // quad_perm 2, 3, 0, 1
    x[i] += dpp<0x141>(x[i]);  // the half row mirrored
    x[i] += dpp<0x140>(x[i]);  // the row mirrored
  }
  if constexpr (TPR >= 32) {
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x[i]), __float_as_uint(x[i]), false, false);
      x[i] = __uint_as_float(b[0]) + __uint_as_float(b[1]);
    }
  }
  if constexpr (TPR >= 64) {
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x[i]), __float_as_uint(x[i]), false, false);
      x[i] = __uint_as_float(b[0]) + __uint_as_float(b[1]);
    }
  }
  if constexpr (TPR > 64) {
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int i = 0; i < n; ++i) red[threadIdx.x >> 6][turn][i] = x[i];
    pet_gemm::ring_barrier();
#pragma unroll
    for (int i = 0; i < n; ++i) {
      x[i] = 0.f;
#pragma unroll
      for (int w = 0; w < TPR / 64; ++w) x[i] += red[w][turn][i];
    }
    turn ^= 1;
  }
}

// A thread's share of a row as it lies in memory: C chunks of kVec elements, chunk
// j at kVec (t + TPR j), zeros past the width.
template <class T, int TPR, int C, bool WHOLE>
__device__ __forceinline__ void load_row(const T* row, int width, int t, u4e (&q)[C]) {
#pragma unroll
  for (int j = 0; j < C; ++j) q[j] = pet_typed::load_raw<T, WHOLE, TPR == 16>(row, kVec<T> * (t + TPR * j), width);
}
// n floats of a vector at d, zeros past the width.
template <int n>
__device__ __forceinline__ void load_vec(const float* p, int d, int width, float (&x)[n]) {
  if (d + n <= width) {
#pragma unroll
    for (int e = 0; e < n; e += 4) {
      const u4e q = *reinterpret_cast<const u4e*>(p + d + e);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[e + i] = __uint_as_float(q[i]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < n; ++e) x[e] = d + e < width ? p[d + e] : 0.f;
  }
}

// x - mu for the `left` elements that are the row's, 0 for those past it.
template <int n>
__device__ __forceinline__ void center(float (&x)[n], float mu, int left) {
  if (left >= n) {
#pragma unroll
    for (int e = 0; e < n; ++e) x[e] -= mu;
  } else {
#pragma unroll
    for (int e = 0; e < n; ++e) x[e] = e < left ? x[e] - mu : 0.f;
  }
}

// (out may be in: neither is __restrict__, here or in the backward, where in_adj may be either)
template <class T, int TPR, int C, bool WHOLE>
__global__ void __launch_bounds__(threads_of(TPR)) norm_typed_fwd_kernel(int rows, int width, float per, T* out,
                                                                         int64_t ldo, const T* in, int64_t ldi,
                                                                         const float* __restrict__ weight,
                                                                         const float* __restrict__ bias) {
  constexpr int V = kVec<T>, RPB = threads_of(TPR) / TPR;
  __shared__ float red[TPR > 64 ? TPR / 64 : 1][2][3];
  const int t = threadIdx.x % TPR;
  const int64_t r = int64_t(blockIdx.x) * RPB + threadIdx.x / TPR;
  if (r >= rows) return;  // (a row's threads leave together)
  int turn = 0;
  u4e q[C];
  float x[C][V];
  load_row<T, TPR, C, WHOLE>(in + r * ldi, width, t, q);
  float mu = 0.f;
#pragma unroll
  for (int j = 0; j < C; ++j) pet_typed::unpack<T>(q[j], x[j]);
  if (bias) {
    float s[1] = {0.f};
#pragma unroll
    for (int j = 0; j < C; ++j)
#pragma unroll
      for (int e = 0; e < V; ++e) s[0] += x[j][e];
    row_sums<TPR>(s, red, turn);
    mu = s[0] * per;
  }
  float v[1] = {0.f};
#pragma unroll
  for (int j = 0; j < C; ++j) {
    center<V>(x[j], mu, width - V * (t + TPR * j));
#pragma unroll
    for (int e = 0; e < V; ++e) v[0] = fmaf(x[j][e], x[j][e], v[0]);
  }
  row_sums<TPR>(v, red, turn);
  const float inv = rsqrt_nr(fmaf(v[0], per, bias ? kLnEps : kRmsEps));
#pragma unroll
  for (int j = 0; j < C; ++j) {
    const int d = V * (t + TPR * j);
    if (d < width) {
      float w[V], b[V];
      load_vec<V>(weight, d, width, w);
      if (bias) load_vec<V>(bias, d, width, b);
#pragma unroll
      for (int e = 0; e < V; ++e) x[j][e] = x[j][e] * inv * w[e] + (bias ? b[e] : 0.f);
      pet_typed::store<T>(out + r * ldo + d, width - d, x[j]);
    }
  }
}

// in_adj for rows < n_node onto beta_node times itself, for the rows after onto
// beta_edge; in_adj null: the parameters' gradients alone. part [gridDim.x][2][width]:
// this workgroup's sums (null: in_adj alone); of one workgroup they are the
// gradients, and go onto beta_w times w_adj and b_adj themselves.
template <class T, int TPR, int C, bool WHOLE, bool LN>
__global__ void __launch_bounds__(threads_of(TPR), waves_of(C * kVec<T>, TPR))
    norm_grads_kernel(int rows, int width, float per, T* in_adj, int64_t lda, const T* out_adj, int64_t ldg,
                      const T* in, int64_t ldi, const float* __restrict__ weight, int n_node, float beta_node,
                      float beta_edge, int live_base, const int* __restrict__ live, float* __restrict__ part,
                      float* __restrict__ w_adj, float* __restrict__ b_adj, float beta_w) {
  constexpr int V = kVec<T>, RPB = threads_of(TPR) / TPR;
  __shared__ float red[TPR > 64 ? TPR / 64 : 1][2][3];
  const int t = threadIdx.x % TPR, g0 = threadIdx.x / TPR;
  const int end = live_rows(rows, live_base, live);
  int turn = 0;
  float w[C][V], dw[C][V], db[C][V];
#pragma unroll
  for (int j = 0; j < C; ++j) {
    load_vec<V>(weight, V * (t + TPR * j), width, w[j]);
#pragma unroll
    for (int e = 0; e < V; ++e) dw[j][e] = 0.f, db[j][e] = 0.f;
  }
  const int64_t step = int64_t(gridDim.x) * RPB;
  int64_t r = int64_t(blockIdx.x) * RPB + g0;
  constexpr bool AHEAD = C * V <= 16;  // (a lane of 32 elements has no registers for the next row's)
  u4e qx[C], qg[C];
  if (AHEAD && r < end) {
    load_row<T, TPR, C, WHOLE>(in + r * ldi, width, t, qx);
    load_row<T, TPR, C, WHOLE>(out_adj + r * ldg, width, t, qg);
  }
  for (; r < end; r += step) {
    float x[C][V], g[C][V], mu = 0.f;
    if (!AHEAD) {
      load_row<T, TPR, C, WHOLE>(in + r * ldi, width, t, qx);
      load_row<T, TPR, C, WHOLE>(out_adj + r * ldg, width, t, qg);
    }
#pragma unroll
    for (int j = 0; j < C; ++j) pet_typed::unpack<T>(qx[j], x[j]), pet_typed::unpack<T>(qg[j], g[j]);
    if (AHEAD && r + step < end) {  // the next row, while this one is worked on
      load_row<T, TPR, C, WHOLE>(in + (r + step) * ldi, width, t, qx);
      load_row<T, TPR, C, WHOLE>(out_adj + (r + step) * ldg, width, t, qg);
    }
    if (LN) {
      float s[1] = {0.f};
#pragma unroll
      for (int j = 0; j < C; ++j)
#pragma unroll
        for (int e = 0; e < V; ++e) s[0] += x[j][e];
      row_sums<TPR>(s, red, turn);
      mu = s[0] * per;
    }
    // sum (x - mu)^2, g w (x - mu), g w
    float s[LN ? 3 : 2] = {};
#pragma unroll
    for (int j = 0; j < C; ++j) {
      if (LN) center<V>(x[j], mu, width - V * (t + TPR * j));
#pragma unroll
      for (int e = 0; e < V; ++e) {
        if (LN) db[j][e] += g[j][e];
        const float gw = g[j][e] * w[j][e];
        s[0] = fmaf(x[j][e], x[j][e], s[0]);
        s[1] = fmaf(gw, x[j][e], s[1]);
        if (LN) s[2] += gw;
      }
    }
    row_sums<TPR>(s, red, turn);
    const float inv = rsqrt_nr(fmaf(s[0], per, LN ? kLnEps : kRmsEps));
    const float mgx = s[1] * inv * per, mg = LN ? s[LN ? 2 : 0] * per : 0.f;
    const float beta = r < n_node ? beta_node : beta_edge;
    T* a_row = in_adj + r * lda;
#pragma unroll
    for (int j = 0; j < C; ++j) {
      const int d = V * (t + TPR * j);
      if (d < width) {
        float o[V];
        if (in_adj && beta != 0.f)
          pet_typed::unpack<T>(pet_typed::load_raw<T, WHOLE, TPR == 16>(a_row, d, width), o);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float xh = x[j][e] * inv;
          dw[j][e] = fmaf(g[j][e], xh, dw[j][e]);
          const float v = inv * fmaf(-xh, mgx, fmaf(g[j][e], w[j][e], -mg));
          o[e] = beta != 0.f ? fmaf(beta, o[e], v) : v;
        }
        if (in_adj) pet_typed::store<T>(a_row + d, width - d, o);
      }
    }
  }
  if (!part) return;
  // the workgroup's groups of rows, in order
  float* p = part + int64_t(blockIdx.x) * 2 * width;
  __shared__ float sums[RPB > 1 ? RPB * C * V * TPR : 1];
  auto put = [&](const float (&a)[C][V], float* to) {
    if constexpr (RPB > 1) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < C; ++j)
#pragma unroll
        for (int e = 0; e < V; ++e) sums[g0 * C * V * TPR + V * (t + TPR * j) + e] = a[j][e];
      __syncthreads();
      for (int d = threadIdx.x; d < width; d += threads_of(TPR)) {
        float s = 0.f;
#pragma unroll
        for (int q = 0; q < RPB; ++q) s += sums[q * C * V * TPR + d];
        to[d] = s;
      }
    } else {
#pragma unroll
      for (int j = 0; j < C; ++j)
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (V * (t + TPR * j) + e < width) to[V * (t + TPR * j) + e] = a[j][e];
    }
  };
  put(dw, p);
  if (LN) put(db, p + width);
  if (gridDim.x > 1) return;
  __syncthreads();
  for (int d = threadIdx.x; d < width; d += threads_of(TPR)) {
    if (w_adj) w_adj[d] = beta_w != 0.f ? fmaf(beta_w, w_adj[d], p[d]) : p[d];
    if (LN && b_adj) b_adj[d] = beta_w != 0.f ? fmaf(beta_w, b_adj[d], p[width + d]) : p[width + d];
  }
}

// adj = beta adj + the sum of the parts, in double: 16 columns by 64 strips of
// parts a workgroup, a strip's loads eight at a time. (32 columns by 32 strips, one
// load after the other: 11 us for 1024 parts.)
__global__ void __launch_bounds__(1024) norm_parts_kernel(int parts, int width, const float* __restrict__ part,
                                                          float* __restrict__ w_adj, float* __restrict__ b_adj,
                                                          float beta) {
  __shared__ double s[64][17];
  const int c = threadIdx.x & 15, strip = threadIdx.x >> 4;
  const int d = blockIdx.x * 16 + c, which = blockIdx.y;
  float* adj = which ? b_adj : w_adj;
  if (!adj) return;
  double a = 0.0;
  if (d < width) {
    const float* p = part + int64_t(which) * width + d;
    int q = strip;
    for (; q + 7 * 64 < parts; q += 8 * 64) {
      float x[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) x[u] = p[int64_t(q + 64 * u) * 2 * width];
#pragma unroll
      for (int u = 0; u < 8; ++u) a += x[u];
    }
    for (; q < parts; q += 64) a += p[int64_t(q) * 2 * width];
  }
  s[strip][c] = a;
  __syncthreads();
  if (threadIdx.x < 256) {  // four strips' quarters, then those
    const int cc = threadIdx.x & 15, f = threadIdx.x >> 4;
    double v = 0.0;
#pragma unroll
    for (int q = 0; q < 4; ++q) v += s[4 * f + q][cc];
    s[4 * f][cc] = v;
  }
  __syncthreads();
  if (threadIdx.x < 16 && d < width) {
    double v = 0.0;
#pragma unroll
    for (int q = 0; q < 16; ++q) v += s[4 * q][c];
    adj[d] = beta != 0.f ? float(double(beta) * adj[d] + v) : float(v);
  }
}

// f(threads a row, chunks a thread) for rows of the width: a wave's or a part of
// one while a lane holds at most 16 elements (of the backward's four values each,
// in registers), the workgroup's past that.
template <class T, class F>
int with_row(int width, F&& f) {
  constexpr int V = kVec<T>, S = V == 4 ? 2 : 1;  // S: the chunks of 8 elements
  using std::integral_constant;
  if (width <= 16 * V) return f(integral_constant<int, 16>{}, integral_constant<int, 1>{});
  if (width <= 32 * V) return f(integral_constant<int, 32>{}, integral_constant<int, 1>{});
  if (width <= 64 * V) return f(integral_constant<int, 64>{}, integral_constant<int, 1>{});
  if (width <= 512) return f(integral_constant<int, 64>{}, integral_constant<int, S>{});
  if (width <= 1024) return f(integral_constant<int, 64>{}, integral_constant<int, 2 * S>{});
  if (width <= 2048) return f(integral_constant<int, 256>{}, integral_constant<int, S>{});
  if (width <= 4096) return f(integral_constant<int, 256>{}, integral_constant<int, 2 * S>{});
  if (width <= 8192) return f(integral_constant<int, 1024>{}, integral_constant<int, S>{});
  return f(integral_constant<int, 512>{}, integral_constant<int, 4 * S>{});
}

// The backward's workgroups that the chip holds at once: its grid at most.
constexpr int kCus = 256;
constexpr int most_of(int E, int TPR) { return kCus * (waves_of(E, TPR) * 256 / threads_of(TPR)); }
template <class T>
int most_for(int width) {
  return with_row<T>(width, [](auto lc, auto cc) { return most_of(decltype(cc)::value * kVec<T>, decltype(lc)::value); });
}

}  // namespace pet_norm

using namespace pet_norm;

// The norm's backward with the parameters' gradients and the layer's sink
// (in_adj rows < n_node onto beta_node, the rows after onto beta_edge; rows at or
// past live_base + *live neither read nor written).
int pet_norm_grads_sink(int dtype, int rows, int width, void* in_adj, int64_t lda, const void* out_adj, int64_t ldg,
                        const void* in, int64_t ldi, const float* weight, int ln, float* w_adj, float* b_adj,
                        float beta_w, int n_node, float beta_node, float beta_edge, int live_base, const int* live,
                        void* ws, hipStream_t st) {
  const int parts = w_adj || b_adj ? 1 : 0;
  float* part = parts ? static_cast<float*>(ws) : nullptr;
  int blocks = 0;
  const int e = pet_typed::with_dtype(dtype, [&](auto tv) {
    using T = decltype(tv);
    return with_row<T>(width, [&](auto lc, auto cc) {
      constexpr int TPR = decltype(lc)::value, C = decltype(cc)::value, TH = threads_of(TPR), RPB = TH / TPR;
      // as many workgroups as the chip holds at once, each with the same rows to within one
      constexpr int most = most_of(C * kVec<T>, TPR);
      // (few rows are one workgroup's, which spares a launch)
      const int64_t groups = std::max<int64_t>(1, (int64_t(rows) + RPB - 1) / RPB);
      const int64_t each = part && groups <= 4 ? groups : (groups + most - 1) / most;
      blocks = int((groups + each - 1) / each);
      auto run = [&](auto lnc) {
        constexpr bool LN = decltype(lnc)::value;
        const auto kernel = width % kVec<T> ? norm_grads_kernel<T, TPR, C, false, LN> : norm_grads_kernel<T, TPR, C, true, LN>;
        hipLaunchKernelGGL(kernel, dim3(unsigned(blocks)), dim3(TH), 0, st,
                           rows, width, 1.0f / width, static_cast<T*>(in_adj), lda, static_cast<const T*>(out_adj), ldg,
                           static_cast<const T*>(in), ldi, weight, n_node, beta_node, beta_edge, live_base, live, part,
                           w_adj, b_adj, beta_w);
      };
      if (ln) run(std::true_type{});
      else run(std::false_type{});
      return hipGetLastError() == hipSuccess ? int(PET_ATTN_OK) : int(PET_ATTN_ELAUNCH);
    });
  });
  if (e || !parts || blocks == 1) return e;
  hipLaunchKernelGGL(norm_parts_kernel, dim3(unsigned((width + 15) / 16), ln ? 2 : 1), dim3(1024), 0, st, blocks, width,
                     part, w_adj, b_adj, beta_w);
  return hipGetLastError() == hipSuccess ? int(PET_ATTN_OK) : int(PET_ATTN_ELAUNCH);
}

extern "C" {

int pet_norm_rows_typed(int dtype, int rows, int width, void* out, int64_t ldo, const void* in, int64_t ldi,
                        const float* weight, const float* bias, void* stream) {
  if (!pet_typed::dtype_ok(dtype) || rows < 0 || width < 1 || width > PET_NORM_MAX_WIDTH) return PET_ATTN_EINVAL;
  if ((rows > 0 && (!out || !in)) || !weight || ldo < width || ldi < width) return PET_ATTN_EINVAL;
  if (rows > 1 && out == in && ldo != ldi) return PET_ATTN_EINVAL;  // in place, but of other rows
  if (!pet_typed::element_aligned(out, dtype) || !pet_typed::element_aligned(in, dtype) ||
      !pet_typed::element_aligned(weight, PET_DTYPE_F32) || !pet_typed::element_aligned(bias, PET_DTYPE_F32))
    return PET_ATTN_EALIGN;
  if (rows == 0) return PET_ATTN_OK;
  if (dtype == PET_DTYPE_F32 && width <= 2048)
    return pet_norm_rows(rows, width, static_cast<float*>(out), ldo, static_cast<const float*>(in), ldi, weight, bias,
                         stream);
  return pet_typed::with_dtype(dtype, [&](auto tv) {
    using T = decltype(tv);
    return with_row<T>(width, [&](auto lc, auto cc) {
      constexpr int TPR = decltype(lc)::value, C = decltype(cc)::value, TH = threads_of(TPR), RPB = TH / TPR;
      const auto kernel = width % kVec<T> ? norm_typed_fwd_kernel<T, TPR, C, false> : norm_typed_fwd_kernel<T, TPR, C, true>;
      constexpr int64_t most = kLaunchThreads / TPR;
      for (int64_t r = 0; r < rows; r += most) {
        const int n = int(std::min(most, rows - r));
        hipLaunchKernelGGL(kernel, dim3(unsigned((int64_t(n) + RPB - 1) / RPB)), dim3(TH), 0,
                           reinterpret_cast<hipStream_t>(stream), n, width, 1.0f / width, static_cast<T*>(out) + r * ldo,
                           ldo, static_cast<const T*>(in) + r * ldi, ldi, weight, bias);
        if (hipGetLastError() != hipSuccess) return int(PET_ATTN_ELAUNCH);
      }
      return int(PET_ATTN_OK);
    });
  });
}

size_t pet_norm_rows_grads_workspace(int rows, int width) {
  if (rows < 0 || width < 1) return 0;
  const int parts = std::max(1, std::min(rows, std::max(most_for<float>(width), most_for<_Float16>(width))));
  return size_t(parts) * 2 * size_t(width) * sizeof(float);
}

int pet_norm_rows_grads(int dtype, int rows, int width, void* in_adj, int64_t lda, float beta, const void* out_adj,
                        int64_t ldg, const void* in, int64_t ldi, const float* weight, int ln, float* weight_adj,
                        float* bias_adj, float beta_w, const int* live, void* workspace, size_t workspace_bytes,
                        void* stream) {
  if (!pet_typed::dtype_ok(dtype) || rows < 0 || width < 1 || width > PET_NORM_MAX_WIDTH) return PET_ATTN_EINVAL;
  if ((rows > 0 && (!out_adj || !in)) || !weight || ldg < width || ldi < width || (in_adj && lda < width))
    return PET_ATTN_EINVAL;
  if ((rows > 0 && !in_adj && !weight_adj && !bias_adj) || (bias_adj && !ln)) return PET_ATTN_EINVAL;
  if (rows > 1 && ((in_adj == out_adj && lda != ldg) || (in_adj == in && lda != ldi))) return PET_ATTN_EINVAL;
  if (!pet_typed::element_aligned(in_adj, dtype) || !pet_typed::element_aligned(out_adj, dtype) ||
      !pet_typed::element_aligned(in, dtype) || !pet_typed::element_aligned(weight, PET_DTYPE_F32) ||
      !pet_typed::element_aligned(weight_adj, PET_DTYPE_F32) || !pet_typed::element_aligned(bias_adj, PET_DTYPE_F32))
    return PET_ATTN_EALIGN;
  if (weight_adj || bias_adj) {
    if (!workspace || workspace_bytes < pet_norm_rows_grads_workspace(rows, width)) return PET_ATTN_EWORKSPACE;
    if ((reinterpret_cast<uintptr_t>(workspace) & 15u) != 0) return PET_ATTN_EALIGN;
    if (weight_adj == bias_adj) return PET_ATTN_EINVAL;  // one tensor for both
  }
  return pet_norm_grads_sink(dtype, rows, width, in_adj, lda, out_adj, ldg, in, ldi, weight, ln, weight_adj, bias_adj,
                             beta_w, rows, beta, beta, 0, live, workspace, reinterpret_cast<hipStream_t>(stream));
}

}  // extern "C"
