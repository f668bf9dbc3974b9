// A dense layer's parameter gradients on gfx950:
//   w_adj[n][k] = beta w_adj[n][k] + sum over m of out_adj[m][n] inp[m][k]
//   b_adj[n]    = beta b_adj[n]    + sum over m of out_adj[m][n]
// over the live rows m, both operands row-major in fp32, bf16 or fp16.
//
// The contraction runs over the rows, the long axis (up to half a million), and
// the result is small: a workgroup takes a tile of the result over one piece of
// the rows, and the pieces' sums, in the workspace, are added in order by a
// second kernel. Nothing is atomic: results repeat bit for bit.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "../../include/pet_model.h"
#include "split_bf16.h"
#include "typed.h"

namespace pet_wgrad {

using pet_split::f4;

// 64 x 64 of the result, four waves of 32 x 32, 32 rows a step through LDS in
// fp32, on the fp32 matrix instruction.
template <class T>
__global__ void __launch_bounds__(256)
    wgrad_fp32_kernel(int M, int N, int K, const T* __restrict__ G, int64_t ldg, const T* __restrict__ X, int64_t ldx,
                      int live_base, const int* __restrict__ live, int chunk, float* __restrict__ part, float* __restrict__ bpart) {
  __shared__ float gs[32][68], xs[32][68];
  const int end = pet_typed::live_rows(M, live_base, live);
  const int k0 = blockIdx.x * 64, n0 = blockIdx.y * 64, s = blockIdx.z;
  const int first = int(min(int64_t(s) * chunk, int64_t(end))), last = int(min(int64_t(first) + chunk, int64_t(end)));
  const int t = threadIdx.x, l = t & 63, c = l & 15, g = l >> 4, w = t >> 6;
  const int wn = 32 * (w >> 1), wk = 32 * (w & 1);
  f4 acc[2][2] = {};
  float bsum = 0.f;
  for (int m0 = first; m0 < last; m0 += 32) {
    __syncthreads();
    for (int i = t; i < 32 * 64; i += 256) {
      const int m = m0 + (i >> 6), j = i & 63;
      gs[i >> 6][j] = m < last && n0 + j < N ? float(G[int64_t(m) * ldg + n0 + j]) : 0.f;
      xs[i >> 6][j] = m < last && k0 + j < K ? float(X[int64_t(m) * ldx + k0 + j]) : 0.f;
    }
    __syncthreads();
    if (t < 64)
      for (int i = 0; i < 32; ++i) bsum += gs[i][t];
#pragma unroll
    for (int i = 0; i < 32; i += 4) {
      float a[2], b[2];
#pragma unroll
      for (int q = 0; q < 2; ++q) a[q] = gs[i + g][wn + 16 * q + c], b[q] = xs[i + g][wk + 16 * q + c];
#pragma unroll
      for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int p = 0; p < 2; ++p) acc[q][p] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[q], b[p], acc[q][p], 0, 0, 0);
    }
  }
  float* out = part + int64_t(s) * N * K;
#pragma unroll
  for (int q = 0; q < 2; ++q)
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int n = n0 + wn + 16 * q + 4 * g + e, k = k0 + wk + 16 * p + c;
        if (n < N && k < K) out[int64_t(n) * K + k] = acc[q][p][e];
      }
  if (bpart && blockIdx.x == 0 && t < 64 && n0 + t < N) bpart[int64_t(s) * N + n0 + t] = bsum;
}

// adj = beta adj + the pieces' sums, in order.
__global__ void __launch_bounds__(256) wgrad_sum_kernel(int N, int K, int pieces, const float* __restrict__ part,
                                                        const float* __restrict__ bpart, float* __restrict__ w_adj,
                                                        int64_t ldw, float* __restrict__ b_adj, float beta) {
  const int64_t nk = int64_t(N) * K, i = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (i >= nk + (b_adj ? N : 0)) return;
  const bool bias = i >= nk;
  const float* p = bias ? bpart + (i - nk) : part + i;
  const int64_t step = bias ? N : nk;
  float v = 0.f;
  for (int s = 0; s < pieces; ++s) v += p[s * step];
  float* o = bias ? b_adj + (i - nk) : w_adj + i / K * ldw + i % K;
  *o = beta != 0.f ? fmaf(beta, *o, v) : v;
}

// Pieces of the rows: enough workgroups for every CU to hold two, each of at least 256 rows.
int pieces_of(int M, int N, int K) {
  const int64_t tiles = ((int64_t(N) + 63) / 64) * ((int64_t(K) + 63) / 64);
  const int64_t want = std::max<int64_t>(1, 512 / tiles), most = std::max<int64_t>(1, (int64_t(M) + 255) / 256);
  return int(std::min(want, most));
}

}  // namespace pet_wgrad

using namespace pet_wgrad;

size_t pet_linear_grads_bytes(int dtype, int M, int N, int K) {
  return size_t(pieces_of(M, N, K)) * (size_t(N) * K + N) * sizeof(float);
}

// pet_linear_grads past its checks; rows at or past live_base + *live (all with no live) are not read.
int pet_linear_grads_run(int dtype, int M, int N, int K, const void* out_adj, int64_t ldo, const void* in, int64_t ldi,
                         int live_base, const int* live, float* w_adj, int64_t ldw, float* b_adj, float beta, void* ws,
                         hipStream_t st) {
  const int pieces = pieces_of(M, N, K), chunk = int((int64_t(M) + pieces - 1) / pieces);
  float *part = static_cast<float*>(ws), *bpart = part + int64_t(pieces) * N * K;
  const int e = pet_typed::with_dtype(dtype, [&](auto tv) {
    using T = decltype(tv);
    hipLaunchKernelGGL(wgrad_fp32_kernel<T>,
                       dim3(unsigned((int64_t(K) + 63) / 64), unsigned((int64_t(N) + 63) / 64), unsigned(pieces)),
                       dim3(256), 0, st, M, N, K, static_cast<const T*>(out_adj), ldo, static_cast<const T*>(in), ldi,
                       live_base, live, chunk, part, b_adj ? bpart : nullptr);
    return hipGetLastError() == hipSuccess ? int(PET_ATTN_OK) : int(PET_ATTN_ELAUNCH);
  });
  if (e) return e;
  const int64_t total = int64_t(N) * K + N;
  hipLaunchKernelGGL(wgrad_sum_kernel, dim3(unsigned((total + 255) / 256)), dim3(256), 0, st, N, K, pieces, part, bpart,
                     w_adj, ldw, b_adj, beta);
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
  if (int64_t(N) > (int64_t(1) << 31) / K) return PET_ATTN_EINDEX;
  if (!pet_typed::element_aligned(out_adj, dtype) || !pet_typed::element_aligned(in, dtype) ||
      !pet_typed::element_aligned(w_adj, PET_DTYPE_F32) || !pet_typed::element_aligned(b_adj, PET_DTYPE_F32))
    return PET_ATTN_EALIGN;
  if (!workspace || workspace_bytes < pet_linear_grads_bytes(dtype, M, N, K)) return PET_ATTN_EWORKSPACE;
  if ((reinterpret_cast<uintptr_t>(workspace) & 15u) != 0) return PET_ATTN_EALIGN;
  return pet_linear_grads_run(dtype, M, N, K, out_adj, ldo, in, ldi, 0, live, w_adj, ldw, b_adj, beta, workspace,
                              reinterpret_cast<hipStream_t>(stream));
}

}  // extern "C"
