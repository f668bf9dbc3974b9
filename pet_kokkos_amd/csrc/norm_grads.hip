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
// order. Nothing is atomic: results repeat bit for bit.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "../../include/pet_attn.h"
#include "typed.h"

namespace pet_norm {

using pet_typed::kVec;
using pet_typed::live_rows;

constexpr float kRmsEps = 1.1920928955078125e-07f;  // float32 epsilon
constexpr float kLnEps = 1e-5f;

constexpr int threads_of(int TPR) { return TPR > 256 ? TPR : 256; }

// A row's sum over its TPR threads, the same bits in each of them: a butterfly
// over the lanes and, where a row is the whole workgroup's, the waves' sums in
// order through LDS (`red`, one slot a wave; two barriers, so a call may follow a
// call).
template <int TPR>
__device__ __forceinline__ float row_sum(float x, float* red) {
#pragma unroll
  for (int o = (TPR < 64 ? TPR : 64) / 2; o > 0; o >>= 1) x += __shfl_xor(x, o);
  if constexpr (TPR > 64) {
    constexpr int W = TPR / 64;
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
    __syncthreads();
    x = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) x += red[i];
    __syncthreads();
  }
  return x;
}

// A thread's share of a row: C chunks of kVec elements, chunk j at kVec (t + TPR j).
template <class T, int TPR, int C>
__device__ __forceinline__ void load_row(const T* row, int width, int t, float (&x)[C][kVec<T>]) {
#pragma unroll
  for (int j = 0; j < C; ++j) {
    const int d = kVec<T> * (t + TPR * j);
    pet_typed::load<T>(row + (d < width ? d : 0), d < width ? width - d : 0, x[j]);
  }
}
// 1 / sqrt(mean((x - mu)^2) + eps) of the row, mu returned.
template <class T, int TPR, int C>
__device__ __forceinline__ float row_inv(const float (&x)[C][kVec<T>], int width, int t, bool ln, float& mu, float* red) {
  constexpr int V = kVec<T>;
  mu = 0.f;
  if (ln) {
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < C; ++j)
#pragma unroll
      for (int e = 0; e < V; ++e) s += x[j][e];
    mu = row_sum<TPR>(s, red) / width;
  }
  float v = 0.f;
#pragma unroll
  for (int j = 0; j < C; ++j)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float a = x[j][e] - mu;
      v += V * (t + TPR * j) + e < width ? a * a : 0.f;
    }
  v = row_sum<TPR>(v, red);
  return 1.0f / sqrtf(v / width + (ln ? kLnEps : kRmsEps));
}

template <class T, int TPR, int C>
__global__ void __launch_bounds__(threads_of(TPR)) norm_typed_fwd_kernel(int rows, int width, T* __restrict__ out,
                                                                         int64_t ldo, const T* __restrict__ in,
                                                                         int64_t ldi, const float* __restrict__ weight,
                                                                         const float* __restrict__ bias) {
  constexpr int V = kVec<T>, RPB = threads_of(TPR) / TPR;
  __shared__ float red[TPR > 64 ? TPR / 64 : 1];
  const int t = threadIdx.x % TPR;
  const int64_t r = int64_t(blockIdx.x) * RPB + threadIdx.x / TPR;
  if (r >= rows) return;  // (a row's threads leave together)
  float x[C][V], mu;
  load_row<T, TPR, C>(in + r * ldi, width, t, x);
  const float inv = row_inv<T, TPR, C>(x, width, t, bias != nullptr, mu, red);
#pragma unroll
  for (int j = 0; j < C; ++j) {
    const int d = V * (t + TPR * j);
    if (d < width) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const int k = min(d + e, width - 1);
        x[j][e] = (x[j][e] - mu) * inv * weight[k] + (bias ? bias[k] : 0.f);
      }
      pet_typed::store<T>(out + r * ldo + d, width - d, x[j]);
    }
  }
}

// in_adj for rows < n_node onto beta_node times itself, for the rows after onto
// beta_edge; in_adj null: the parameters' gradients alone. part [gridDim.x][2][width]:
// this workgroup's sums (null: in_adj alone).
template <class T, int TPR, int C, bool LN>
__global__ void __launch_bounds__(threads_of(TPR))
    norm_grads_kernel(int rows, int width, T* __restrict__ in_adj, int64_t lda, const T* __restrict__ out_adj,
                      int64_t ldg, const T* __restrict__ in, int64_t ldi, const float* __restrict__ weight, int n_node,
                      float beta_node, float beta_edge, int live_base, const int* __restrict__ live,
                      float* __restrict__ part) {
  constexpr int V = kVec<T>, RPB = threads_of(TPR) / TPR;
  __shared__ float red[TPR > 64 ? TPR / 64 : 1];
  const int t = threadIdx.x % TPR, g0 = threadIdx.x / TPR;
  const int end = live_rows(rows, live_base, live);
  float w[C][V], dw[C][V], db[C][V];
#pragma unroll
  for (int j = 0; j < C; ++j)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int d = V * (t + TPR * j) + e;
      w[j][e] = d < width ? weight[d] : 0.f, dw[j][e] = 0.f, db[j][e] = 0.f;
    }
  for (int64_t r = int64_t(blockIdx.x) * RPB + g0; r < end; r += int64_t(gridDim.x) * RPB) {
    float x[C][V], g[C][V], mu;
    load_row<T, TPR, C>(in + r * ldi, width, t, x);
    load_row<T, TPR, C>(out_adj + r * ldg, width, t, g);
    const float inv = row_inv<T, TPR, C>(x, width, t, LN, mu, red);
    float sg = 0.f, sgx = 0.f;
#pragma unroll
    for (int j = 0; j < C; ++j)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        // (past the width g is 0, and x - mu times it)
        const float xh = (x[j][e] - mu) * inv, gw = g[j][e] * w[j][e];
        if (LN) sg += gw;
        sgx += gw * xh;
        dw[j][e] = fmaf(g[j][e], xh, dw[j][e]);
        if (LN) db[j][e] += g[j][e];
      }
    if (!in_adj) continue;
    const float mg = LN ? row_sum<TPR>(sg, red) / width : 0.f, mgx = row_sum<TPR>(sgx, red) / width;
    const float beta = r < n_node ? beta_node : beta_edge;
    T* a_row = in_adj + r * lda;
#pragma unroll
    for (int j = 0; j < C; ++j) {
      const int d = V * (t + TPR * j);
      if (d < width) {
        float o[V];
        if (beta != 0.f) pet_typed::load<T>(a_row + d, width - d, o);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float xh = (x[j][e] - mu) * inv;
          const float v = inv * fmaf(-xh, mgx, fmaf(g[j][e], w[j][e], -mg));
          o[e] = beta != 0.f ? fmaf(beta, o[e], v) : v;
        }
        pet_typed::store<T>(a_row + d, width - d, o);
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
        if (V * (t + TPR * j) < width) {
#pragma unroll
          for (int e = 0; e < V; ++e)
            if (V * (t + TPR * j) + e < width) to[V * (t + TPR * j) + e] = a[j][e];
        }
    }
  };
  put(dw, p);
  if (LN) put(db, p + width);
}

// adj = beta adj + the sum of the parts, in double: 32 columns by 32 strips of parts a workgroup.
__global__ void __launch_bounds__(1024) norm_parts_kernel(int parts, int width, const float* __restrict__ part,
                                                          float* __restrict__ w_adj, float* __restrict__ b_adj,
                                                          float beta) {
  __shared__ double s[32][33];
  const int c = threadIdx.x & 31, strip = threadIdx.x >> 5;
  const int d = blockIdx.x * 32 + c, which = blockIdx.y;
  float* adj = which ? b_adj : w_adj;
  if (!adj) return;
  double a = 0.0;
  if (d < width)
    for (int q = strip; q < parts; q += 32) a += part[(int64_t(q) * 2 + which) * width + d];
  s[strip][c] = a;
  __syncthreads();
  if (threadIdx.x < 32 && d < width) {
    double v = 0.0;
    for (int q = 0; q < 32; ++q) v += s[q][c];
    adj[d] = beta != 0.f ? float(double(beta) * adj[d] + v) : float(v);
  }
}

// f(threads a row, chunks a thread) for rows of the width.
template <class T, class F>
int with_row(int width, F&& f) {
  constexpr int V = kVec<T>;
  using std::integral_constant;
  if (width <= 16 * V) return f(integral_constant<int, 16>{}, integral_constant<int, 1>{});
  if (width <= 32 * V) return f(integral_constant<int, 32>{}, integral_constant<int, 1>{});
  if (width <= 64 * V) return f(integral_constant<int, 64>{}, integral_constant<int, 1>{});
  if (width <= 128 * V) return f(integral_constant<int, 64>{}, integral_constant<int, 2>{});
  if (width <= 256 * V) return f(integral_constant<int, 64>{}, integral_constant<int, 4>{});
  if (width <= 512 * V) return f(integral_constant<int, 256>{}, integral_constant<int, 2>{});
  if (width <= 1024 * V) return f(integral_constant<int, 256>{}, integral_constant<int, 4>{});
  if (V == 8 || width <= 2048 * V) return f(integral_constant<int, 512>{}, integral_constant<int, 4>{});
  return f(integral_constant<int, 512>{}, integral_constant<int, 8>{});
}

constexpr int kMaxParts = 1024;

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
      blocks = int(std::max<int64_t>(1, std::min<int64_t>((int64_t(rows) + RPB - 1) / RPB, kMaxParts)));
      auto run = [&](auto lnc) {
        hipLaunchKernelGGL((norm_grads_kernel<T, TPR, C, decltype(lnc)::value>), dim3(unsigned(blocks)), dim3(TH), 0, st,
                           rows, width, static_cast<T*>(in_adj), lda, static_cast<const T*>(out_adj), ldg,
                           static_cast<const T*>(in), ldi, weight, n_node, beta_node, beta_edge, live_base, live, part);
      };
      if (ln) run(std::true_type{});
      else run(std::false_type{});
      return hipGetLastError() == hipSuccess ? int(PET_ATTN_OK) : int(PET_ATTN_ELAUNCH);
    });
  });
  if (e || !parts) return e;
  hipLaunchKernelGGL(norm_parts_kernel, dim3(unsigned((width + 31) / 32), ln ? 2 : 1), dim3(1024), 0, st, blocks, width,
                     part, w_adj, b_adj, beta_w);
  return hipGetLastError() == hipSuccess ? int(PET_ATTN_OK) : int(PET_ATTN_ELAUNCH);
}

extern "C" {

int pet_norm_rows_typed(int dtype, int rows, int width, void* out, int64_t ldo, const void* in, int64_t ldi,
                        const float* weight, const float* bias, void* stream) {
  if (!pet_typed::dtype_ok(dtype) || rows < 0 || width < 1 || width > PET_NORM_MAX_WIDTH) return PET_ATTN_EINVAL;
  if ((rows > 0 && (!out || !in)) || !weight || ldo < width || ldi < width) return PET_ATTN_EINVAL;
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
      hipLaunchKernelGGL((norm_typed_fwd_kernel<T, TPR, C>), dim3(unsigned((int64_t(rows) + RPB - 1) / RPB)), dim3(TH),
                         0, reinterpret_cast<hipStream_t>(stream), rows, width, static_cast<T*>(out), ldo,
                         static_cast<const T*>(in), ldi, weight, bias);
      return hipGetLastError() == hipSuccess ? int(PET_ATTN_OK) : int(PET_ATTN_ELAUNCH);
    });
  });
}

size_t pet_norm_rows_grads_workspace(int rows, int width) {
  if (rows < 0 || width < 1) return 0;
  return size_t(kMaxParts) * 2 * size_t(width) * sizeof(float);
}

int pet_norm_rows_grads(int dtype, int rows, int width, void* in_adj, int64_t lda, float beta, const void* out_adj,
                        int64_t ldg, const void* in, int64_t ldi, const float* weight, int ln, float* weight_adj,
                        float* bias_adj, float beta_w, const int* live, void* workspace, size_t workspace_bytes,
                        void* stream) {
  if (!pet_typed::dtype_ok(dtype) || rows < 0 || width < 1 || width > PET_NORM_MAX_WIDTH) return PET_ATTN_EINVAL;
  if ((rows > 0 && (!out_adj || !in)) || !weight || ldg < width || ldi < width || (in_adj && lda < width))
    return PET_ATTN_EINVAL;
  if ((rows > 0 && !in_adj && !weight_adj && !bias_adj) || (bias_adj && !ln)) return PET_ATTN_EINVAL;
  if (!pet_typed::element_aligned(in_adj, dtype) || !pet_typed::element_aligned(out_adj, dtype) ||
      !pet_typed::element_aligned(in, dtype) || !pet_typed::element_aligned(weight, PET_DTYPE_F32) ||
      !pet_typed::element_aligned(weight_adj, PET_DTYPE_F32) || !pet_typed::element_aligned(bias_adj, PET_DTYPE_F32))
    return PET_ATTN_EALIGN;
  if (weight_adj || bias_adj) {
    if (!workspace || workspace_bytes < pet_norm_rows_grads_workspace(rows, width)) return PET_ATTN_EWORKSPACE;
    if ((reinterpret_cast<uintptr_t>(workspace) & 15u) != 0) return PET_ATTN_EALIGN;
  }
  return pet_norm_grads_sink(dtype, rows, width, in_adj, lda, out_adj, ldg, in, ldi, weight, ln, weight_adj, bias_adj,
                             beta_w, rows, beta, beta, 0, live, workspace, reinterpret_cast<hipStream_t>(stream));
}

}  // extern "C"
