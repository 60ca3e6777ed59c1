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
    uint32_t m = w[0] & 0x7fff7fffu;
#pragma unroll
    for (int i = 1; i < 4; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
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
__device__ __forceinline__ float step_of(uint32_t byte) { return __uint_as_float(byte == 255u ? 0x7fc00000u : (byte - 6u) << 23); }     // 2^(e - 6)

// Four codes in a word.  v + 1.5 2^23 has the integer nearest v in its low bits, ties to even, in two's complement.
__device__ __forceinline__ uint32_t code_bits(float x, float inv) { return __float_as_uint(fminf(fmaxf(x * inv, -127.f), 127.f) + 12582912.f); }
__device__ __forceinline__ uint32_t codes4(const float* x, float inv) {
  const uint32_t a = __byte_perm(code_bits(x[0], inv), code_bits(x[1], inv), 0x0040), b = __byte_perm(code_bits(x[2], inv), code_bits(x[3], inv), 0x0040);
  return __byte_perm(a, b, 0x5410);
}
// and back: 2^23 + (code + 128) as the bits of a number, less 2^23 + 128
__device__ __forceinline__ void values4(uint32_t codes, float step, float* x) {
  const uint32_t u = codes ^ 0x80808080u;
  x[0] = (__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7440)) - 8388736.f) * step;
  x[1] = (__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7441)) - 8388736.f) * step;
  x[2] = (__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7442)) - 8388736.f) * step;
  x[3] = (__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7443)) - 8388736.f) * step;
}

// codes of a 16-byte vector's elements: 8 bytes of 16-bit tensors, 4 of fp32
template <typename T> struct Codes { uint32_t w[VecN<T>::N / 4]; };
template <typename T>
__device__ __forceinline__ void store_codes(int8_t* codes, int64_t vec, const float (&x)[VecN<T>::N], float inv) {
  if constexpr (VecN<T>::N == 8) reinterpret_cast<uint2*>(codes)[vec] = make_uint2(codes4(x, inv), codes4(x + 4, inv));
  else reinterpret_cast<uint32_t*>(codes)[vec] = codes4(x, inv);
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
__device__ __forceinline__ void values_of(const Codes<T>& c, uint32_t byte, float (&x)[VecN<T>::N]) {
#pragma unroll
  for (int i = 0; i < VecN<T>::N / 4; ++i) values4(c.w[i], step_of(byte), x + 4 * i);
}
// an element of the last block, which is no whole one: a warp has it, lane by lane
__device__ __forceinline__ uint32_t tail_exponent(float x) {
  uint32_t m = __float_as_uint(x) & 0x7fffffffu;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  return exponent_byte(m);
}
__device__ __forceinline__ int8_t tail_code(float x, uint32_t byte) { return (int8_t)(code_bits(x, per_step(byte)) & 0xffu); }
__device__ __forceinline__ float tail_value(int8_t code, uint32_t byte) { return (float)code * step_of(byte); }

}  // namespace
}  // namespace ulm
