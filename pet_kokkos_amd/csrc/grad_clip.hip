// The norm of a list of gradients and their clipping on gfx950:
//   norm = |scale| (sum over every element of |g|^p)^(1/p), p = 1, 2 or infinity,
//   g   *= scale min(1, max_norm / (norm + eps)).
//
// Bound by HBM: every gradient read once for the norm, read again and written
// to clip it. The tensors' addresses and extents travel in the kernels'
// arguments (kTensors a launch), so a call copies nothing to the device and can be
// captured. A launch's tensors are cut into chunks of kChunk elements that the
// workgroups take in turn; a workgroup's sum (in double, so that no square
// over- or underflows and a sum's length costs no digits) goes to its slot of the
// workspace, and whoever needs the norm adds the slots in order: results repeat
// bit for bit.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "../../include/pet_model.h"
#include "typed.h"

namespace pet_clip {

constexpr int kTensors = 88;    // a launch's tensors: 29 bytes each in its 4 KB of arguments
constexpr int kChunk = 8192;    // elements: 64 or 128 bytes a thread in flight
constexpr int kBlocks = 2048;   // a launch's workgroups at most, each with a slot: 8 a CU

struct Batch {
  void* data[kTensors];
  int64_t numel[kTensors];
  int64_t cols[kTensors];  // 0: the elements are consecutive
  int64_t ld[kTensors];
  unsigned char dtype[kTensors];
  unsigned first[kTensors + 1];  // a tensor's first chunk
  int n;
};
static_assert(sizeof(Batch) <= 3584, "the arguments' 4 KB");

// Chunk q's tensor.
__device__ __forceinline__ int tensor_of(const Batch& b, unsigned q) {
  int lo = 0, hi = b.n;  // first[lo] <= q < first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (b.first[mid] <= q) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ double wave_all(double x, int p) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const double y = __shfl_xor(x, o);
    x = p ? x + y : (y > x || y != y) ? y : x;
  }
  return x;
}
// |a|^p summed, or for p = 0 the largest |a| (a NaN stays).
template <int p>
__device__ __forceinline__ double take(double s, float x) {
  const double a = fabs(double(x));
  return p == 2 ? fma(a, a, s) : p == 1 ? s + a : (a > s || a != a) ? a : s;
}
__device__ __forceinline__ double join(double s, double y, int p) { return p ? s + y : (y > s || y != y) ? y : s; }

// The workgroup's value from its threads', in thread 0.
template <int TH>
__device__ __forceinline__ double block_all(double x, int p, double* red) {
  x = wave_all(x, p);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
  __syncthreads();
  double s = red[0];
  for (int i = 1; i < TH / 64; ++i) s = join(s, red[i], p);
  __syncthreads();
  return s;
}

template <class T, class F>
__device__ __forceinline__ void chunk_each(const Batch& b, int i, unsigned q, F&& f) {
  constexpr int V = pet_typed::kVec<T>;
  const int64_t n = b.numel[i], e0 = int64_t(q - b.first[i]) * kChunk;
  T* p = static_cast<T*>(b.data[i]);
  const int64_t cols = b.cols[i];
  if (cols == 0) {
    if (e0 + kChunk <= n) {  // whole: no bounds between the loads
#pragma unroll
      for (int j = 0; j < kChunk / (256 * V); ++j) f(p + e0 + (j * 256 + int(threadIdx.x)) * V, int64_t(V));
    } else {
      for (int64_t e = e0 + int(threadIdx.x) * V; e < n; e += 256 * V) f(p + e, n - e);
    }
  } else {  // rows of a wider matrix, element by element
    const int64_t ld = b.ld[i];
    for (int64_t e = e0 + threadIdx.x; e < min(n, e0 + kChunk); e += 256) f(p + e / cols * ld + e % cols, int64_t(1));
  }
}

template <class F>
__device__ __forceinline__ void with_type(int dtype, F&& f) {
  if (dtype == PET_DTYPE_F32) f(float{});
  else if (dtype == PET_DTYPE_BF16) f(__bf16{});
  else f(_Float16{});
}

template <int p>
__global__ void __launch_bounds__(256) grad_norm_kernel(Batch b, double* __restrict__ slots) {
  __shared__ double red[4];
  double v[4] = {0.0, 0.0, 0.0, 0.0};  // (one sum's chain of adds held 16-bit types to 4.1 TB/s)
  for (unsigned q = blockIdx.x; q < b.first[b.n]; q += gridDim.x) {
    const int i = tensor_of(b, q);
    with_type(b.dtype[i], [&](auto tv) {
      using T = decltype(tv);
      chunk_each<T>(b, i, q, [&](T* at, int64_t left) {
        float x[pet_typed::kVec<T>];
        pet_typed::load<T>(at, 0, left, x);
#pragma unroll
        for (int e = 0; e < pet_typed::kVec<T>; ++e) v[e & 3] = take<p>(v[e & 3], x[e]);
      });
    });
  }
  const double s = block_all<256>(join(join(v[0], v[1], p), join(v[2], v[3], p), p), p, red);
  if (threadIdx.x == 0) slots[blockIdx.x] = s;
}

struct Ends {
  double scale, max_norm, eps;
  int p, slots;
};
// The norm of the scaled gradients from the slots, the same bits in every thread.
template <int TH>
__device__ __forceinline__ double norm_of(const Ends& a, const double* __restrict__ slots, double* red) {
  double s = 0.0;
  for (int i = threadIdx.x; i < a.slots; i += TH) s = join(s, slots[i], a.p);
  s = block_all<TH>(s, a.p, red);
  return fabs(a.scale) * (a.p == 2 ? sqrt(s) : s);
}

__global__ void __launch_bounds__(256) grad_finish_kernel(Ends a, const double* __restrict__ slots, float* __restrict__ norm) {
  __shared__ double red[4];
  const double v = norm_of<256>(a, slots, red);
  if (threadIdx.x == 0) *norm = float(v);
}

// scale min(1, max_norm / (norm + eps)); a norm of 0 with no eps, or no bound, clips nothing.
__device__ __forceinline__ float clip_factor(const Ends& a, double v) {
  double r = 1.0;
  if (v != v) r = v;
  else if (v + a.eps > a.max_norm) r = a.max_norm / (v + a.eps);
  return float(a.scale * r);
}

__global__ void __launch_bounds__(256) grad_clip_kernel(Batch b, Ends a, const double* __restrict__ slots, float* __restrict__ norm) {
  __shared__ double red[4];
  const double v = norm_of<256>(a, slots, red);
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = float(v);
  const float f = clip_factor(a, v);
  if (f == 1.f) return;  // (a factor of one leaves every gradient as it is)
  for (unsigned q = blockIdx.x; q < b.first[b.n]; q += gridDim.x) {
    const int i = tensor_of(b, q);
    with_type(b.dtype[i], [&](auto tv) {
      using T = decltype(tv);
      chunk_each<T>(b, i, q, [&](T* at, int64_t left) {
        float x[pet_typed::kVec<T>];
        pet_typed::load<T>(at, 0, left, x);
#pragma unroll
        for (int e = 0; e < pet_typed::kVec<T>; ++e) x[e] *= f;
        pet_typed::store<T>(at, left, x);
      });
    });
  }
}

int check(const pet_grad_tensor* t, int n) {
  if (n < 0 || (n > 0 && !t)) return PET_ATTN_EINVAL;
  for (int i = 0; i < n; ++i) {
    const pet_grad_tensor& x = t[i];
    if (!pet_typed::dtype_ok(x.dtype) || x.rows < 0 || x.cols < 0) return PET_ATTN_EINVAL;
    if (x.rows == 0 || x.cols == 0) continue;
    if (!x.data || (x.rows > 1 && x.ld < x.cols)) return PET_ATTN_EINVAL;
    if (x.rows > (int64_t(1) << 36) / x.cols) return PET_ATTN_EINDEX;
    if (!pet_typed::element_aligned(x.data, x.dtype)) return PET_ATTN_EALIGN;
  }
  return PET_ATTN_OK;
}

int batches_of(int n) { return n / kTensors + (n % kTensors != 0); }

// Tensors [i, n) into b, as many as it takes; the next one's index.
int fill(Batch& b, const pet_grad_tensor* t, int i, int n) {
  b.n = 0;
  b.first[0] = 0;
  for (; i < n && b.n < kTensors; ++i) {
    const pet_grad_tensor& x = t[i];
    const int64_t numel = x.rows * x.cols, chunks = (numel + kChunk - 1) / kChunk;
    if (chunks == 0) continue;
    const bool flat = x.rows == 1 || x.ld == x.cols;
    b.data[b.n] = x.data, b.numel[b.n] = numel, b.cols[b.n] = flat ? 0 : x.cols, b.ld[b.n] = x.ld;
    b.dtype[b.n] = static_cast<unsigned char>(x.dtype);
    b.first[b.n + 1] = b.first[b.n] + unsigned(chunks);
    ++b.n;
  }
  return i;
}

int run(const pet_grad_tensor* t, int n, int p, double scale, bool clip, double max_norm, double eps, float* norm,
        void* ws, size_t bytes, hipStream_t st) {
  if (p < 0 || p > 2) return PET_ATTN_EINVAL;
  if (int e = check(t, n)) return e;
  if (!ws || bytes < pet_grad_workspace(n)) return PET_ATTN_EWORKSPACE;
  if ((reinterpret_cast<uintptr_t>(ws) & 15u) != 0 || !pet_typed::element_aligned(norm, PET_DTYPE_F32))
    return PET_ATTN_EALIGN;
  double* slots = static_cast<double*>(ws);
  Ends a{scale, max_norm, eps, p, 0};
  Batch b;
  for (int i = 0; i < n;) {
    i = fill(b, t, i, n);
    if (b.n == 0) continue;
    const int blocks = int(std::min<unsigned>(b.first[b.n], kBlocks));
    const dim3 grid{unsigned(blocks)}, block{256};
    if (p == 2) hipLaunchKernelGGL(grad_norm_kernel<2>, grid, block, 0, st, b, slots + a.slots);
    else if (p == 1) hipLaunchKernelGGL(grad_norm_kernel<1>, grid, block, 0, st, b, slots + a.slots);
    else hipLaunchKernelGGL(grad_norm_kernel<0>, grid, block, 0, st, b, slots + a.slots);
    if (hipGetLastError() != hipSuccess) return PET_ATTN_ELAUNCH;
    a.slots += blocks;
  }
  if (!clip || a.slots == 0) {
    hipLaunchKernelGGL(grad_finish_kernel, dim3(1), dim3(256), 0, st, a, slots, norm);
    return hipGetLastError() == hipSuccess ? int(PET_ATTN_OK) : int(PET_ATTN_ELAUNCH);
  }
  bool first = true;
  for (int i = 0; i < n;) {
    i = fill(b, t, i, n);
    if (b.n == 0) continue;
    const int blocks = int(std::min<unsigned>(b.first[b.n], kBlocks));
    hipLaunchKernelGGL(grad_clip_kernel, dim3(unsigned(blocks)), dim3(256), 0, st, b, a, slots, first ? norm : nullptr);
    if (hipGetLastError() != hipSuccess) return PET_ATTN_ELAUNCH;
    first = false;
  }
  return PET_ATTN_OK;
}

}  // namespace pet_clip

using namespace pet_clip;

extern "C" {

size_t pet_grad_workspace(int n) { return n < 0 ? 0 : size_t(std::max(1, batches_of(n))) * kBlocks * sizeof(double); }

int pet_grad_norm(const pet_grad_tensor* grads, int n, int p, double scale, float* norm, void* workspace,
                  size_t workspace_bytes, void* stream) {
  if (!norm || !std::isfinite(scale)) return PET_ATTN_EINVAL;
  return run(grads, n, p, scale, false, 0.0, 0.0, norm, workspace, workspace_bytes, reinterpret_cast<hipStream_t>(stream));
}

int pet_grad_clip(const pet_grad_tensor* grads, int n, int p, double scale, double max_norm, double eps, float* norm,
                  void* workspace, size_t workspace_bytes, void* stream) {
  if (!norm || !std::isfinite(scale) || !(max_norm >= 0.0) || !(eps >= 0.0) || std::isinf(eps)) return PET_ATTN_EINVAL;
  return run(grads, n, p, scale, true, max_norm, eps, norm, workspace, workspace_bytes,
             reinterpret_cast<hipStream_t>(stream));
}

}  // extern "C"
