// Dropout's mask: a function of a seed, a step, the call and an element's
// place, made anew wherever it is needed and never stored.
//
// The generator is Threefry-2x32 (Salmon, Moraes, Dror and Shaw, "Parallel random
// numbers: as easy as 1, 2, 3", SC 2011) of 13 rounds, the fewest that its authors
// found to pass every battery: additions, rotations and exclusive ors of 32-bit
// words, one instruction each at full rate here, where the multipliers of the
// counter generators that have them run at a quarter. A block of 64 bits is four
// 16-bit numbers, so p counts in steps of 2^-16, and costs about 12
// instructions an element.
//
// The key of a call is the block of (step, call) under the seed, so a captured
// graph whose program raises the step on the device draws a new mask each replay.
#pragma once

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "../../include/pet_attn.h"

namespace pet_rng {

struct Words {
  uint32_t x, y;
};

__device__ __forceinline__ uint32_t turn(uint32_t v, int r) { return __builtin_amdgcn_alignbit(v, v, 32 - r); }

__device__ __forceinline__ Words threefry13(uint32_t k0, uint32_t k1, uint32_t x, uint32_t y) {
  constexpr int R[8] = {13, 15, 26, 6, 17, 29, 16, 24};
  const uint32_t k[3] = {k0, k1, k0 ^ k1 ^ 0x1BD11BDAu};
  x += k0, y += k1;
#pragma unroll
  for (int i = 0; i < 13; ++i) {
    x += y;
    y = turn(y, R[i % 8]) ^ x;
    if (i % 4 == 3) {
      const int j = (i + 1) / 4;
      x += k[j % 3];
      y += k[(j + 1) % 3] + uint32_t(j);
    }
  }
  return {x, y};
}

// What a kernel needs of a call's dropout: least is 65536 p to the nearest, a
// number under it leaves its element out, the rest are scaled by 65536 / (65536 - least).
struct Drop {
  const int64_t* state = nullptr;  // device: seed, step
  uint32_t least = 0, call = 0;
  float scale = 1.f;

  __device__ __forceinline__ Words key() const {
    const uint64_t seed = uint64_t(state[0]);
    return threefry13(uint32_t(seed), uint32_t(seed >> 32), uint32_t(uint64_t(state[1])), call);
  }
  __device__ __forceinline__ Words block(const Words& k, uint32_t x, uint32_t y) const {
    return threefry13(k.x, k.y, x, y);
  }
  // number i (0 .. 3) of a block
  static __device__ __forceinline__ uint32_t number(const Words& w, int i) {
    const uint32_t v = i < 2 ? w.x : w.y;
    return i & 1 ? v >> 16 : v & 0xffffu;
  }
};

// The host's half: refuses a p outside 0 .. 65534 / 65536 (the scale of what stays
// is then at most 2^15, which fp16 holds) and a state that no int64 load reaches.
inline int make_drop(const pet_dropout* d, Drop& out) {
  if (!d->state || !(d->p >= 0.0) || !(d->p <= 1.0)) return PET_ATTN_EINVAL;
  if ((reinterpret_cast<uintptr_t>(d->state) & 7u) != 0) return PET_ATTN_EALIGN;
  const long least = std::lrint(65536.0 * d->p);
  if (least > 65534) return PET_ATTN_EINVAL;
  out.state = d->state;
  out.least = uint32_t(least);
  out.call = d->call;
  out.scale = float(65536.0 / (65536.0 - double(least)));
  return PET_ATTN_OK;
}

}  // namespace pet_rng
