// The norm of a list of gradients and their clipping on gfx950:
//   norm = |scale| (sum over every element of |g|^p)^(1/p), p = 1, 2 or infinity,
//   g   *= scale min(1, max_norm / (norm + eps)).
//
// Bound by HBM: every gradient read once for the norm, read again and written
// to clip it. The tensors' addresses and extents travel in the kernels'
// arguments, so a call copies nothing to the device and can be captured. A
// launch's tensors are cut into chunks of kChunk elements that the workgroups
// take in turn; a workgroup's sum (in double, so that no square over- or
// underflows and a sum's length costs no digits) goes to its slot of the
// workspace, and whoever needs the norm adds the slots in order: results repeat
// bit for bit. 1733 MB are clipped in 984 us; tensors whose rows are apart go an element
// a load with two divisions each (96 MB 74 us, 102 MB consecutive 49).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include "../../include/pet_model.h"
#include "typed.h"

namespace pet_clip {

using pet_typed::u4e;

constexpr int kChunk = 8192;   // elements: 64 or 128 bytes a thread in flight
constexpr int kBlocks = 1536;  // a launch's workgroups at most, each with a slot: the 6 a CU that its registers leave

// A tensor of a launch, or (from the table's end) the extents of one whose rows are apart.
struct Entry {
  void* data;
  unsigned first;  // its first chunk
  unsigned rest;   // the last chunk's elements less one, the type from bit 13, from bit 15 the extents' slot plus one
};
struct Extents {
  int64_t cols, ld;
};
union Slot {
  Entry tensor;
  Extents rows;
};
// What norm_of needs besides the slots.
struct Ends {
  double scale, max_norm, eps;
  int p, slots;
};
// A launch's arguments are 4 KB: the clipping's others (Ends and two addresses), the
// table's two counts, and as many slots as are left: a tensor's, or two where its rows
// are apart. MI355X, 200 tensors of 27 MB in one launch instead of two (100 slots): the
// norm 9.3 -> 6.9 us, the clipping with it 19.0 -> 13.0; of 1.7 GB 1018 -> 1015.
constexpr int kSlots = (4096 - int(sizeof(Ends)) - 2 * int(sizeof(void*)) - 8) / int(sizeof(Slot));
struct Batch {
  Slot slot[kSlots];
  int n;
  unsigned chunks;
};
static_assert(sizeof(Batch) + sizeof(Ends) + 2 * sizeof(void*) <= 4096, "the arguments' 4 KB");

// A chunk's elements, the same in every lane.
struct Piece {
  char* data;          // the tensor's
  unsigned at, dtype;  // the chunk in it
  int left;            // of kChunk
  int rows;            // its extents' slot, or -1: consecutive
};

// The tensors' first chunks by lanes (tensors l, l + 64, ...): a chunk's tensor is
// one comparison of all, where a search's reads of the arguments went one after
// the other (88 tensors of 12 MB: clipping 10.3 -> 9.2 us, half of it by the loads
// ahead of the norm below).
constexpr int kPer = (kSlots + 63) / 64;
__device__ __forceinline__ void load_firsts(const Batch& b, unsigned (&first)[kPer]) {
  const int l = threadIdx.x & 63;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const unsigned f = b.slot[min(l + 64 * j, kSlots - 1)].tensor.first;
    first[j] = l + 64 * j < b.n ? f : ~0u;
  }
}
// Chunk q's piece, from the tensors that start at or before it.
__device__ __forceinline__ Piece find(const Batch& b, const unsigned (&first)[kPer], unsigned q) {
  int n = 0;
#pragma unroll
  for (int j = 0; j < kPer; ++j) n += __builtin_popcountll(__builtin_amdgcn_ballot_w64(first[j] <= q));
  const Entry t = b.slot[n - 1].tensor;
  const unsigned next = n < b.n ? b.slot[n].tensor.first : b.chunks;
  Piece p;
  p.data = static_cast<char*>(t.data);
  p.at = q - t.first;
  p.left = q + 1 < next ? kChunk : int(t.rest & (kChunk - 1)) + 1;
  p.dtype = t.rest >> 13 & 3;
  p.rows = int(t.rest >> 15) - 1;
  return p;
}

__device__ __forceinline__ double wave_all(double x, int p) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const double y = __shfl_xor(x, o);
    x = p ? x + y : (y > x || y != y) ? y : x;
  }
  return x;
}
// |a|^p summed, or for p = 0 the largest |a| (a NaN stays), which is a float's.
template <int p>
using Sum = typename std::conditional<p == 0, float, double>::type;
template <int p>
__device__ __forceinline__ Sum<p> take(Sum<p> s, float x) {
  const Sum<p> a = fabsf(x);
  if constexpr (p == 0) return a > s || a != a ? a : s;
  else return p == 2 ? fma(a, a, s) : s + a;
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

// f(address, elements from there) for a thread's vectors of a chunk, or (rows apart) its elements.
template <class T, class F>
__device__ __forceinline__ void chunk_each(const Batch& b, const Piece& c, F&& f) {
  constexpr int V = pet_typed::kVec<T>;
  T* p = reinterpret_cast<T*>(c.data);
  const int64_t e0 = int64_t(c.at) * kChunk;
  if (c.rows < 0) {
    if (c.left == kChunk) {  // whole: no bounds between the loads
#pragma unroll
      for (int j = 0; j < kChunk / (256 * V); ++j) f(p + e0 + (j * 256 + int(threadIdx.x)) * V, int64_t(V));
    } else {
      for (int e = int(threadIdx.x) * V; e < c.left; e += 256 * V) f(p + e0 + e, int64_t(c.left - e));
    }
  } else {
    const int64_t cols = b.slot[c.rows].rows.cols, ld = b.slot[c.rows].rows.ld;
    for (int64_t e = e0 + threadIdx.x; e < e0 + c.left; e += 256) f(p + e / cols * ld + e % cols, int64_t(1));
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
  Sum<p> v[4] = {};  // (one sum's chain of adds held 16-bit types to 4.1 TB/s)
  unsigned first[kPer];
  load_firsts(b, first);
  for (unsigned q = blockIdx.x; q < b.chunks; q += gridDim.x) {
    const Piece c = find(b, first, q);
    with_type(c.dtype, [&](auto tv) {
      using T = decltype(tv);
      chunk_each<T>(b, c, [&](T* at, int64_t left) {
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
  unsigned first[kPer];
  load_firsts(b, first);
  // the first chunk's loads go out before the norm is there
  constexpr int N = kChunk * 4 / (256 * 16);
  u4e raw[N];
  const Piece c0 = find(b, first, blockIdx.x);
  const bool early = c0.rows < 0 && c0.left == kChunk;
  const int bytes = c0.dtype == PET_DTYPE_F32 ? 4 : 2;
  char* const p0 = c0.data + int64_t(c0.at) * kChunk * bytes + threadIdx.x * 16;
  if (early)
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j < N * bytes / 4) raw[j] = *reinterpret_cast<const u4e*>(p0 + j * 4096);
  const double v = norm_of<256>(a, slots, red);
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = float(v);
  const float f = clip_factor(a, v);
  if (f == 1.f) return;  // (a factor of one leaves every gradient as it is)
  unsigned q = blockIdx.x;
  if (early) {
    with_type(c0.dtype, [&](auto tv) {
      using T = decltype(tv);
      constexpr int V = pet_typed::kVec<T>;
#pragma unroll
      for (int j = 0; j < kChunk / (256 * V); ++j) {
        float x[V];
        pet_typed::unpack<T>(raw[j], x);
#pragma unroll
        for (int e = 0; e < V; ++e) x[e] *= f;
        *reinterpret_cast<u4e*>(p0 + j * 4096) = pet_typed::pack<T>(x);
      }
    });
    q += gridDim.x;
  }
  for (; q < b.chunks; q += gridDim.x) {
    const Piece c = find(b, first, q);
    with_type(c.dtype, [&](auto tv) {
      using T = decltype(tv);
      chunk_each<T>(b, c, [&](T* at, int64_t left) {
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

// (a launch takes at least half its slots' tensors)
int batches_of(int n) { return n / (kSlots / 2) + (n % (kSlots / 2) != 0); }

// Tensors [i, n) into b, as many as it takes; the next one's index.
int fill(Batch& b, const pet_grad_tensor* t, int i, int n) {
  b.n = 0, b.chunks = 0;
  int apart = kSlots;  // the extents so far
  for (; i < n; ++i) {
    const pet_grad_tensor& x = t[i];
    const int64_t numel = x.rows * x.cols;
    if (numel == 0) continue;
    const bool flat = x.rows == 1 || x.ld == x.cols;
    if (b.n + (flat ? 1 : 2) > apart) break;
    unsigned rest = unsigned((numel - 1) % kChunk) | unsigned(x.dtype) << 13;
    if (!flat) b.slot[--apart].rows = {x.cols, x.ld}, rest |= unsigned(apart + 1) << 15;
    b.slot[b.n++].tensor = {x.data, b.chunks, rest};
    b.chunks += unsigned((numel + kChunk - 1) / kChunk);
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
    const int blocks = int(std::min<unsigned>(b.chunks, kBlocks));
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
    const int blocks = int(std::min<unsigned>(b.chunks, kBlocks));
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
