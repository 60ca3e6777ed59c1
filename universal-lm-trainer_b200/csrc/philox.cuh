// Dropout masks that are computed and never stored (sm_100a).
//
// Element i of a tensor (its row-major index) belongs to the group i / 8.  Philox4x32 with ten rounds (Salmon, Moraes, Dror and
// Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011), keyed with the 64-bit seed, turns the group's number into
// 128 bits; element j of the group has their j-th 16.  It is dropped where they are below threshold = 65536 p rounded to
// an integer, at least 1 for p > 0 and at most 65535 for p < 1; the others are multiplied by 65536 / (65536 - threshold), the
// inverse of the share that really stays, so the mean is exact although p is taken in steps of 2^-16.
//
// Sixteen bits an element and not 32: ten rounds are twenty 32 x 32 -> 64 products and twenty three-input XORs, so 16 bits cost
// 5 instructions an element.  At the copy rate a 16-bit elementwise pass leaves an SM about 23 issue slots an element in all.
#pragma once

#include <cmath>

#include "common.cuh"

namespace ulm {

constexpr int kPhiloxRounds = 10;

struct DropMask {
  uint32_t k0[kPhiloxRounds], k1[kPhiloxRounds];         // the rounds' keys: the same for all threads, so made on the host
  uint32_t least;                                        // threshold << 16: 16 bits in the upper half of a word stay from here on
  uint32_t bits;                                         // ANDed to the generator's words: 0 where everything is dropped
  float scale;
};

// p in [0, 1], checked by the caller
inline DropMask make_drop_mask(double p, uint64_t seed) {
  DropMask m;
  for (int r = 0; r < kPhiloxRounds; ++r) {
    m.k0[r] = (uint32_t)seed + (uint32_t)r * 0x9E3779B9u;
    m.k1[r] = (uint32_t)(seed >> 32) + (uint32_t)r * 0xBB67AE85u;
  }
  const double t = nearbyint(p * 65536.0);
  const uint32_t threshold = p <= 0. ? 0u : t < 1. ? 1u : t > 65535. ? 65535u : (uint32_t)t;
  m.least = p >= 1. ? 0xffffffffu : threshold << 16;
  m.bits = p >= 1. ? 0u : 0xffffffffu;
  m.scale = p >= 1. ? 0.f : (float)(65536.0 / (65536.0 - threshold));
  return m;
}
inline bool drop_p_ok(double p) { return p >= 0. && p <= 1.; }      // false for NaN

__device__ __forceinline__ uint4 philox(const DropMask& m, uint64_t group) {
  uint32_t c0 = (uint32_t)group, c1 = (uint32_t)(group >> 32), c2 = 0u, c3 = 0u;
#pragma unroll
  for (int r = 0; r < kPhiloxRounds; ++r) {
    const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ m.k0[r];
    c1 = (uint32_t)b;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ m.k1[r];
    c3 = (uint32_t)a;
  }
  return make_uint4(c0, c1, c2, c3);
}

// The mask of N consecutive elements that start at index v * N.  Kept as the generator's words and compared where an element is
// used: a shift for every second element, a compare and a select, instead of gathering the N answers into bits first
// (dropout of 32768 x 768 bf16 20.9 -> 17.9 us; the gate's backward at 32768 x 2048 113 -> 101).
template <int N> struct Keep {
  static_assert(N == 8 || N == 4, "a group or half of one");
  uint32_t w[N / 2], least;
  __device__ __forceinline__ bool operator()(int j) const { return (j & 1 ? w[j >> 1] : w[j >> 1] << 16) >= least; }
};
template <int N>
__device__ __forceinline__ Keep<N> keep_of(const DropMask& m, uint64_t v) {
  const uint4 u = philox(m, N == 8 ? v : v >> 1);
  Keep<N> k;
  k.least = m.least;
  if constexpr (N == 8) {
    k.w[0] = u.x & m.bits; k.w[1] = u.y & m.bits; k.w[2] = u.z & m.bits; k.w[3] = u.w & m.bits;
  } else {
    const bool upper = v & 1;
    k.w[0] = (upper ? u.z : u.x) & m.bits;
    k.w[1] = (upper ? u.w : u.y) & m.bits;
  }
  return k;
}
// element i by itself
__device__ __forceinline__ bool keep_one(const DropMask& m, uint64_t i) {
  const Keep<8> k = keep_of<8>(m, i >> 3);
  bool stays = false;
#pragma unroll
  for (int j = 0; j < 8; ++j) stays = (int)(i & 7) == j ? k(j) : stays;
  return stays;
}

// A dropped element is zero whatever it held, infinities and NaN included.
__device__ __forceinline__ float dropped(const DropMask& m, bool stays, float v) { return stays ? v * m.scale : 0.f; }

}  // namespace ulm
