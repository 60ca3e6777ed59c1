// Two fp32 values at a time (sm_100a): one instruction of the multiply-add pipe for both.  Each half is rounded as the operation by itself would be.
// Where a kernel that is to run at memory speed keeps that pipe busy, this is half of its instructions: the backward of
// norm_add_norm has 65 an element instead of 82.
#pragma once

#include "common.cuh"

namespace ulm {
namespace {

__device__ __forceinline__ uint64_t bits(const float2& v) { return reinterpret_cast<const uint64_t&>(v); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits(a)), "l"(bits(b)));
  return reinterpret_cast<float2&>(r);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits(a)), "l"(bits(b)));
  return reinterpret_cast<float2&>(r);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(bits(a)), "l"(bits(b)), "l"(bits(c)));
  return reinterpret_cast<float2&>(r);
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

}  // namespace
}  // namespace ulm
