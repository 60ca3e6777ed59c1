// Tensors in 8 bits: blocks of 32 consecutive elements with one exponent, signed integers beside it (sm_100a).
//
//   e = the exponent of the block's largest magnitude (2^e <= max < 2^(e + 1)), at least -120
//   code = x / 2^(e - 6) rounded to an integer, ties to even, held to +-127;  x~ = code 2^(e - 6)
//
// kept as the bytes code and e + 127; a block with an infinity or a NaN has the exponent byte 255 and stands for NaN throughout.  With a power of
// two for a step every quotient and product is exact, so codes are the same in any arithmetic, and every x~ is a number of the
// tensor's own type: seven bits, at or above its smallest step.  |x~ - x| <= 2^(e - 7), and <= 2^(e - 6) where 127 holds it: 1/128 and 1/64 of the
// block's largest at most.  That is the layout of the microscaling format MXINT8 (Open Compute Project, "OCP Microscaling Formats (MX)
// Specification", 2023), with -128 left out.  A scale of max / 127 would use half a bit more on average and cost a division whose
// rounding decides ties.
#pragma once

#include "gate_math.cuh"
#include "pairs.cuh"

namespace ulm {
namespace {

constexpr int kBlock8 = 32;

// the largest magnitude of a vector, as the bits of an fp32 number; infinities and NaN stay above all others
template <typename T>
__device__ __forceinline__ uint32_t magnitude(const uint4& u) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  if constexpr (sizeof(T) == 4) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) m = max(m, w[i] & 0x7fffffffu);
    return m;
  } else {
    uint32_t m = __vmaxu2(__vimax3_u16x2(w[0] & 0x7fff7fffu, w[1] & 0x7fff7fffu, w[2] & 0x7fff7fffu), w[3] & 0x7fff7fffu);
    m = max(m & 0xffffu, m >> 16);
    const uint16_t h = (uint16_t)m;
    return __float_as_uint(Cvt<T>::to_f(*reinterpret_cast<const T*>(&h)));
  }
}
// over the lanes that share a block of 32: 4 with 16-bit elements, 8 with fp32
template <typename T>
__device__ __forceinline__ uint32_t block_magnitude(uint32_t m) {
#pragma unroll
  for (int o = kBlock8 / VecN<T>::N / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  return m;
}
__device__ __forceinline__ uint32_t exponent_byte(uint32_t magnitude) {
  const uint32_t e = magnitude >> 23;
  return e < 7u ? 7u : e;                                // 255 for infinities and NaN already
}
__device__ __forceinline__ float per_step(uint32_t byte) { return __uint_as_float(byte == 255u ? 0u : (260u - byte) << 23); }            // 2^(6 - e)
// 2^(e - 6); bytes below 7 do not come from a tensor packed here, and their steps are subnormal
__device__ __forceinline__ float step_of(uint32_t byte) { return __uint_as_float(byte == 255u ? 0x7fc00000u : byte > 6u ? (byte - 6u) << 23 : 1u << (byte + 16u)); }

// whether a block's largest rounds to 128, which 127 holds: an element of it may have to be held
__device__ __forceinline__ bool rounds_past(uint32_t magnitude) { return (magnitude & 0x7fffffu) >= 0x7f0000u; }

// the elements of a 16-byte vector in pairs, and back
template <typename T>
__device__ __forceinline__ void unpack_pairs(const uint4& u, float2 (&v)[VecN<T>::N / 2]) {
  if constexpr (sizeof(T) == 4) {
    v[0] = make_float2(__uint_as_float(u.x), __uint_as_float(u.y));
    v[1] = make_float2(__uint_as_float(u.z), __uint_as_float(u.w));
  } else {
    v[0] = Cvt<T>::unpack2(u.x); v[1] = Cvt<T>::unpack2(u.y); v[2] = Cvt<T>::unpack2(u.z); v[3] = Cvt<T>::unpack2(u.w);
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack_pairs(const float2 (&v)[VecN<T>::N / 2]) {
  if constexpr (sizeof(T) == 4) return make_uint4(__float_as_uint(v[0].x), __float_as_uint(v[0].y), __float_as_uint(v[1].x), __float_as_uint(v[1].y));
  else return make_uint4(Cvt<T>::pack2(v[0].x, v[0].y), Cvt<T>::pack2(v[1].x, v[1].y), Cvt<T>::pack2(v[2].x, v[2].y), Cvt<T>::pack2(v[3].x, v[3].y));
}

// Four codes in a word.  v + 1.5 2^23 has the integer nearest v in its low bits, ties to even, in two's complement; v = x inv is exact.
constexpr float kCodeMagic = 12582912.f;
__device__ __forceinline__ uint32_t low_bytes(float2 a, float2 b) {
  const uint32_t p = __byte_perm(__float_as_uint(a.x), __float_as_uint(a.y), 0x0040), q = __byte_perm(__float_as_uint(b.x), __float_as_uint(b.y), 0x0040);
  return __byte_perm(p, q, 0x5410);
}
__device__ __forceinline__ float held(float v) { return fminf(fmaxf(v, -127.f), 127.f); }
__device__ __forceinline__ uint32_t codes4(float2 a, float2 b, float inv) { return low_bytes(fma2(a, both(inv), both(kCodeMagic)), fma2(b, both(inv), both(kCodeMagic))); }
__device__ __forceinline__ uint32_t codes4_held(float2 a, float2 b, float inv) {
  return low_bytes(make_float2(held(a.x * inv) + kCodeMagic, held(a.y * inv) + kCodeMagic), make_float2(held(b.x * inv) + kCodeMagic, held(b.y * inv) + kCodeMagic));
}
// and back: 2^23 + (code + 128) as the bits of a number, less 2^23 + 128
__device__ __forceinline__ void values4(uint32_t codes, float step, float2* x) {
  const uint32_t u = codes ^ 0x80808080u;
  const float2 a = make_float2(__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7440)), __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7441)));
  const float2 b = make_float2(__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7442)), __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7443)));
  x[0] = mul2(add2(a, both(-8388736.f)), both(step));
  x[1] = mul2(add2(b, both(-8388736.f)), both(step));
}

// codes of a 16-byte vector's elements: 8 bytes of 16-bit tensors, 4 of fp32
template <typename T> struct Codes { uint32_t w[VecN<T>::N / 4]; };
// `past`: an element may have to be held (rounds_past); for one block in a hundred or so
template <typename T>
__device__ __forceinline__ void store_codes(int8_t* codes, int64_t vec, const float2 (&x)[VecN<T>::N / 2], float inv, bool past) {
  if constexpr (VecN<T>::N == 8) {
    uint2 c = make_uint2(codes4(x[0], x[1], inv), codes4(x[2], x[3], inv));
    if (past) c = make_uint2(codes4_held(x[0], x[1], inv), codes4_held(x[2], x[3], inv));
    reinterpret_cast<uint2*>(codes)[vec] = c;
  } else {
    reinterpret_cast<uint32_t*>(codes)[vec] = past ? codes4_held(x[0], x[1], inv) : codes4(x[0], x[1], inv);
  }
}
template <typename T>
__device__ __forceinline__ Codes<T> load_codes(const int8_t* codes, int64_t vec) {
  Codes<T> c;
  if constexpr (VecN<T>::N == 8) {
    const uint2 u = reinterpret_cast<const uint2*>(codes)[vec];
    c.w[0] = u.x; c.w[1] = u.y;
  } else {
    c.w[0] = reinterpret_cast<const uint32_t*>(codes)[vec];
  }
  return c;
}
template <typename T>
__device__ __forceinline__ void values_of(const Codes<T>& c, uint32_t byte, float2 (&x)[VecN<T>::N / 2]) {
#pragma unroll
  for (int i = 0; i < VecN<T>::N / 4; ++i) values4(c.w[i], step_of(byte), x + 2 * i);
}
// an element of the last block, which is no whole one: a warp has it, lane by lane
__device__ __forceinline__ uint32_t tail_exponent(float x) {
  uint32_t m = __float_as_uint(x) & 0x7fffffffu;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  return exponent_byte(m);
}
__device__ __forceinline__ int8_t tail_code(float x, uint32_t byte) { return (int8_t)(__float_as_uint(held(x * per_step(byte)) + kCodeMagic) & 0xffu); }
__device__ __forceinline__ float tail_value(int8_t code, uint32_t byte) { return (float)code * step_of(byte); }

}  // namespace
}  // namespace ulm
