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
// The 16 bytes at element d of a row of n, as they lie, with zeros past its end.
// whole: n is a multiple of the vector. Else the row's last 16 bytes, moved down, or
// (few: n may be less than a vector) its elements one by one.
template <class T, bool whole = false, bool few = true>
__device__ __forceinline__ u4e load_raw(const T* row, int64_t d, int64_t n) {
  constexpr int V = kVec<T>, BITS = 8 * int(sizeof(T));
  u4e q = {0u, 0u, 0u, 0u};
  if constexpr (whole) {
    if (d < n) q = *reinterpret_cast<const u4e*>(row + d);
  } else if (!few || n >= V) {
    if (d < n) {
      q = *reinterpret_cast<const u4e*>(row + (d + V <= n ? d : n - V));
      if (d + V > n) {
        uint64_t lo = uint64_t(q[1]) << 32 | q[0], hi = uint64_t(q[3]) << 32 | q[2];
        const int by = int(d + V - n) * BITS;  // 16 .. 112 bits
        lo = by >= 64 ? hi >> (by - 64) : lo >> by | hi << (64 - by);
        hi = by >= 64 ? 0 : hi >> by;
        q = u4e{unsigned(lo), unsigned(lo >> 32), unsigned(hi), unsigned(hi >> 32)};
      }
    }
  } else {
#pragma unroll 1
    for (int i = 0; i < int(n - d); ++i) {
      unsigned v;
      if constexpr (BITS == 32) v = __float_as_uint(row[d + i]);
      else v = unsigned(__builtin_bit_cast(unsigned short, row[d + i])) << (16 * (i & 1));
#pragma unroll
      for (int w = 0; w < 4; ++w) q[w] |= w == i * BITS / 32 ? v : 0u;
    }
  }
  return q;
}
template <class T>
__device__ __forceinline__ void load(const T* row, int64_t d, int64_t n, float (&x)[kVec<T>]) {
  unpack<T>(load_raw<T>(row, d, n), x);
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
