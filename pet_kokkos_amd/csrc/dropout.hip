// Dropout of rows, onto a residual or not: out = residual + M x, M 0 or 1 / (1 - p)
// an element, from the counter generator (counter_rng.h) at (row, column / 4). It
// is its own backward (without the residual), and nothing of the mask is kept.
//
// Bound by memory: each row is read once and written once (and the residual
// read), 2 or 4 bytes an element a pass, against some 14 instructions. A thread
// takes four 16-byte pieces of the flat sequence of all rows' pieces, 256 apart,
// with all their loads ahead of the first block of numbers. 498338 x 512 bf16 onto a
// residual: 281 us, 5.4 TB/s (a large copy reaches 5.0).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "../../include/pet_attn.h"
#include "counter_rng.h"
#include "typed.h"

namespace {

using pet_rng::Drop;
using pet_rng::Words;
using pet_typed::kVec;
using pet_typed::u4e;

constexpr int kThreads = 256, kEach = 4, kPieces = kThreads * kEach;

// x / per for x < per + kPieces: per <= 2^15 by its rounded-up reciprocal
// (x per < 2^32), larger ones by a comparison (the quotient is 0 or 1).
struct Split {
  uint32_t per, magic;
  __host__ explicit Split(uint32_t p) : per(p), magic(p <= 32768u && p > 1u ? uint32_t((uint64_t(1) << 32) / p + 1) : 0u) {}
  __device__ __forceinline__ uint32_t quotient(uint32_t x) const {
    return per == 1u ? x : magic ? __umulhi(x, magic) : uint32_t(x >= per);
  }
};

// WHOLE: the width is a multiple of a piece.
template <class T, bool WHOLE, bool RES>
__global__ __launch_bounds__(kThreads) void dropout_kernel(int rows, int width, T* out, int64_t ldo, const T* in,
                                                           int64_t ldi, const T* residual, int64_t ldr, Drop drop,
                                                           const int* live, Split split, int64_t pieces) {
  constexpr int V = kVec<T>;
  const int last = pet_typed::live_rows(rows, 0, live);
  const Words key = drop.key();
  for (int64_t first = int64_t(blockIdx.x) * kPieces; first < pieces; first += int64_t(gridDim.x) * kPieces) {
    const int64_t row0 = first / split.per;
    const uint32_t at0 = uint32_t(first - row0 * split.per);
    if (row0 >= last) break;
    u4e x[kEach], r[kEach];
    int64_t row[kEach];
    int col[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const uint32_t p = at0 + threadIdx.x + i * kThreads, q = split.quotient(p);
      row[i] = row0 + q;
      col[i] = int(p - q * split.per) * V;
      if (row[i] < last) {
        x[i] = pet_typed::load_raw<T, WHOLE>(in + row[i] * ldi, col[i], width);
        if constexpr (RES) r[i] = pet_typed::load_raw<T, WHOLE>(residual + row[i] * ldr, col[i], width);
      }
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      if (row[i] >= last) continue;
      float a[V], b[V];
      pet_typed::unpack<T>(x[i], a);
      if constexpr (RES) pet_typed::unpack<T>(r[i], b);
#pragma unroll
      for (int j = 0; j < V; j += 4) {
        const Words w = drop.block(key, uint32_t(row[i]), uint32_t(col[i] + j) >> 2);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float y = Drop::number(w, e) >= drop.least ? a[j + e] : 0.f;
          a[j + e] = RES ? fmaf(y, drop.scale, b[j + e]) : y * drop.scale;
        }
      }
      T* to = out + row[i] * ldo + col[i];
      if constexpr (WHOLE) *reinterpret_cast<u4e*>(to) = pet_typed::pack<T>(a);
      else pet_typed::store<T>(to, width - col[i], a);
    }
  }
}

}  // namespace

extern "C" int pet_dropout_rows(int dtype, int rows, int width, void* out, int64_t ldo, const void* in, int64_t ldi,
                                const void* residual, int64_t ldr, const pet_dropout* dropout, const int* live,
                                void* stream) {
  if (!pet_typed::dtype_ok(dtype) || rows < 0 || width < 1 || !dropout) return PET_ATTN_EINVAL;
  if ((rows > 0 && (!out || !in)) || ldo < width || ldi < width || (residual && ldr < width)) return PET_ATTN_EINVAL;
  if (rows > 1 && ((out == in && ldo != ldi) || (out == residual && ldo != ldr))) return PET_ATTN_EINVAL;  // in place, but of other rows
  Drop drop;
  if (const int e = pet_rng::make_drop(dropout, drop)) return e;
  if (!pet_typed::element_aligned(out, dtype) || !pet_typed::element_aligned(in, dtype) ||
      !pet_typed::element_aligned(residual, dtype) || !pet_typed::element_aligned(live, PET_DTYPE_F32))
    return PET_ATTN_EALIGN;
  if (rows == 0) return PET_ATTN_OK;
  return pet_typed::with_dtype(dtype, [&](auto tv) {
    using T = decltype(tv);
    constexpr int V = kVec<T>;
    const int64_t per = (int64_t(width) + V - 1) / V, pieces = per * rows;
    const unsigned blocks = unsigned(std::min<int64_t>((pieces + kPieces - 1) / kPieces, 1 << 20));
    auto run = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3(blocks), dim3(kThreads), 0, reinterpret_cast<hipStream_t>(stream), rows, width,
                         static_cast<T*>(out), ldo, static_cast<const T*>(in), ldi, static_cast<const T*>(residual),
                         ldr, drop, live, Split(uint32_t(per)), pieces);
    };
    if (width % V == 0) residual ? run(dropout_kernel<T, true, true>) : run(dropout_kernel<T, true, false>);
    else residual ? run(dropout_kernel<T, false, true>) : run(dropout_kernel<T, false, false>);
    return hipGetLastError() == hipSuccess ? int(PET_ATTN_OK) : int(PET_ATTN_ELAUNCH);
  });
}
