// Vectors, sigmoid and operand layout shared by the feed-forward gate's kernels (sm_100a).
#pragma once

#include "common.cuh"

namespace ulm {
namespace {

template <typename T> struct VecN { static constexpr int N = 16 / sizeof(T); };

template <typename T>
__device__ __forceinline__ void unpack(const uint4& u, float (&f)[VecN<T>::N]) {
  if constexpr (sizeof(T) == 4) {
    const float* p = reinterpret_cast<const float*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = p[i];
  } else {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) { const float2 t = Cvt<T>::unpack2(w[i]); f[2 * i] = t.x; f[2 * i + 1] = t.y; }
  }
}

template <typename T>
__device__ __forceinline__ uint4 pack(const float (&f)[VecN<T>::N]) {
  uint4 u;
  if constexpr (sizeof(T) == 4) {
    float* p = reinterpret_cast<float*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = f[i];
  } else {
    uint32_t* w = reinterpret_cast<uint32_t*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = Cvt<T>::pack2(f[2 * i], f[2 * i + 1]);
  }
  return u;
}

template <typename T>
__device__ __forceinline__ float rnd(float v) { return Cvt<T>::to_f(Cvt<T>::from_f(v)); }

// s = sigmoid(a) and silu(a).  fp32 tensors: the forms ATen's kernels use.  16-bit tensors: one ex2 and one reciprocal
// on the special-function unit instead of expf and an IEEE division each: the divisions' fix-up code, not memory, was what
// the kernels waited for.  Relative error of s and u: 2^-19 for |a| <= 16, 2^-17 down to a = -88, below which s
// is 0 as in the divided form.  Over 0.4 G random values of each type and of deviation 0.3, 1 and 3, the rms error of y, da
// and db against float64 is that of the divided form within what so many roundings can show (1e-6 of itself, da of fp16
// 4e-6).  Newton steps that bring s and u to within an ulp of the divisions flip fewer roundings and cost 14 us of 66
// forward, 6 of 104 backward (32768 x 2048 bf16).
template <typename T>
__device__ __forceinline__ void sigmoid_silu(float a, float& s, float& u) {
  if constexpr (sizeof(T) == 4) {
    const float d = 1.f + expf(-a);
    s = 1.f / d;
    u = a / d;                                           // the form ATen's kernel uses
  } else {
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(a * -1.4426950408889634f));
    asm("rcp.approx.f32 %0, %1;" : "=f"(s) : "f"(1.f + e));   // no ftz: s goes down to 2^-128 before e overflows
    u = a * s;
  }
}

// Where vector v of the gate's operands lies: a and b (da and db) are dense, or column blocks of a wider matrix (the two
// halves of one projection's output): rows of vpr vectors, `stride` vectors apart.
struct Rows { uint32_t vpr; int64_t stride; };
template <bool ROWS>
__device__ __forceinline__ int64_t operand_vec(int64_t v, const Rows& rw) {
  if constexpr (!ROWS) return v;
  const uint32_t u = (uint32_t)v, r = u / rw.vpr;        // fewer than 2^32 vectors (checked by the host)
  return (int64_t)r * rw.stride + (u - r * rw.vpr);
}

}  // namespace
}  // namespace ulm
