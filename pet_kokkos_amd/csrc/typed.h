// Rows and tensors in fp32, bf16 or fp16 (PET_DTYPE_*): 16 bytes at a time, in
// fp32 in registers, rounded to nearest once as they are stored.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "../../include/pet_attn.h"

namespace pet_typed {

// 16 bytes at an element's alignment: one instruction on gfx950 at any address.
typedef unsigned u4e __attribute__((ext_vector_type(4), aligned(2)));

template <class T>
constexpr int kVec = 16 / int(sizeof(T));

template <class T>
__device__ __forceinline__ void unpack(const u4e& q, float (&x)[kVec<T>]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(q[i]);
  } else if constexpr (std::is_same<T, __bf16>::value) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(q[i] << 16), x[2 * i + 1] = __uint_as_float(q[i] & 0xffff0000u);
  } else {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned u = q[i];  // (a bit cast of the element itself reads the vector's first)
      const h2 h = __builtin_bit_cast(h2, u);
      x[2 * i] = float(h[0]), x[2 * i + 1] = float(h[1]);
    }
  }
}
template <class T>
__device__ __forceinline__ u4e pack(const float (&x)[kVec<T>]) {
  u4e q;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = __float_as_uint(x[i]);
  } else {
    typedef T t2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = __builtin_bit_cast(unsigned, t2{T(x[2 * i]), T(x[2 * i + 1])});
  }
  return q;
}
// n elements at p (at least one; from the vector's on: all of it), zeros past them.
template <class T>
__device__ __forceinline__ void load(const T* p, int64_t n, float (&x)[kVec<T>]) {
  if (n >= kVec<T>) {
    unpack<T>(*reinterpret_cast<const u4e*>(p), x);
  } else {
#pragma unroll
    for (int i = 0; i < kVec<T>; ++i) x[i] = float(p[min(int64_t(i), n - 1)]);  // (all in flight)
#pragma unroll
    for (int i = 0; i < kVec<T>; ++i) x[i] = i < n ? x[i] : 0.f;
  }
}
template <class T>
__device__ __forceinline__ void store(T* p, int64_t n, const float (&x)[kVec<T>]) {
  if (n >= kVec<T>) {
    *reinterpret_cast<u4e*>(p) = pack<T>(x);
  } else {
#pragma unroll
    for (int i = 0; i < kVec<T>; ++i)
      if (i < n) p[i] = T(x[i]);
  }
}

inline int dtype_size(int dtype) { return dtype == PET_DTYPE_F32 ? 4 : 2; }
inline bool dtype_ok(int dtype) { return dtype == PET_DTYPE_F32 || dtype == PET_DTYPE_BF16 || dtype == PET_DTYPE_F16; }
inline bool element_aligned(const void* p, int dtype) {
  return (reinterpret_cast<uintptr_t>(p) & uintptr_t(dtype_size(dtype) - 1)) == 0;
}
// f(a T) for the element type of a dtype that dtype_ok.
template <class F>
int with_dtype(int dtype, F&& f) {
  if (dtype == PET_DTYPE_F32) return f(float{});
  if (dtype == PET_DTYPE_BF16) return f(__bf16{});
  return f(_Float16{});
}
// The rows that count of a buffer of `rows`: base + *live, brought into 0 .. rows (all of them without live).
__device__ __forceinline__ int live_rows(int rows, int base, const int* live) {
  if (!live) return rows;
  const int64_t n = int64_t(base) + *live;
  return n < 0 ? 0 : n > rows ? rows : int(n);
}

}  // namespace pet_typed
