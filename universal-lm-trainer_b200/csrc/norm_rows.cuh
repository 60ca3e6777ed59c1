// Rows of a norm spread over the lanes of one or more warps: vectors, sums over a row, how rows are dealt to CTAs (sm_100a).
#pragma once

#include "common.cuh"

namespace ulm {
namespace {

template <int E>
__device__ __forceinline__ void load_f32(const float* p, float (&v)[E]) {
#pragma unroll
  for (int j = 0; j < E; j += 4) {
    const float4 f = *reinterpret_cast<const float4*>(p + j);
    v[j] = f.x; v[j + 1] = f.y; v[j + 2] = f.z; v[j + 3] = f.w;
  }
}
template <int E>
__device__ __forceinline__ void store_f32(float* p, const float (&v)[E]) {
#pragma unroll
  for (int j = 0; j < E; j += 4) *reinterpret_cast<float4*>(p + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
}
// E 16-bit elements as they lie in memory
template <int E> struct Raw { uint32_t u[E / 2]; };
template <typename TY, int E>
__device__ __forceinline__ Raw<E> load_raw(const TY* p) {
  Raw<E> r;
  if constexpr (E == 8) {
    const uint4 q = *reinterpret_cast<const uint4*>(p);
    r.u[0] = q.x; r.u[1] = q.y; r.u[2] = q.z; r.u[3] = q.w;
  } else {
    const uint2 q = *reinterpret_cast<const uint2*>(p);
    r.u[0] = q.x; r.u[1] = q.y;
  }
  return r;
}
template <typename TY, int E>
__device__ __forceinline__ void unpack_raw(const Raw<E>& r, float (&v)[E]) {
#pragma unroll
  for (int j = 0; j < E / 2; ++j) { const float2 f = Cvt<TY>::unpack2(r.u[j]); v[2 * j] = f.x; v[2 * j + 1] = f.y; }
}
template <typename TY, int E>
__device__ __forceinline__ void store_16(TY* p, const float (&v)[E]) {
  uint32_t u[E / 2];
#pragma unroll
  for (int j = 0; j < E / 2; ++j) u[j] = Cvt<TY>::pack2(v[2 * j], v[2 * j + 1]);
  if constexpr (E == 8) *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
  else *reinterpret_cast<uint2*>(p) = make_uint2(u[0], u[1]);
}

// Sum over the W warps of a row.  `slots`: this call's own kMaxWarps floats; consecutive calls of a warp alternate between two
// sets, so that one barrier a call is enough.
__device__ __forceinline__ float row_sum(float v, int W, int group, int warp, int lane, float* slots) {
  v = warp_sum(v);
  if (W == 1) return v;
  if (lane == 0) slots[warp] = v;
  asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(32 * W) : "memory");
  float t = 0.f;
  for (int i = 0; i < W; ++i) t += slots[group * W + i];
  return t;
}

int ceil_div(int a, int b) { return (a + b - 1) / b; }

// Warps a row and rows a CTA.  Few rows (less than the SMs take at full CTAs) are spread over more, smaller CTAs.
struct Split { int W, groups; };
Split split_rows(int64_t rows, int nvec, int nv, int warps) {
  Split s;
  s.W = ceil_div(nvec, 32 * nv);
  s.groups = warps / s.W > 0 ? warps / s.W : 1;
  const int64_t spread = (rows + kNumSMs - 1) / kNumSMs;
  if (spread < s.groups) s.groups = spread < 1 ? 1 : (int)spread;
  return s;
}
bool ok16(const void* p, int64_t stride, int E) { return !(reinterpret_cast<uintptr_t>(p) & (2 * E - 1)) && stride % E == 0; }
bool ok32(const void* p, int64_t stride) { return !(reinterpret_cast<uintptr_t>(p) & 15) && stride % 4 == 0; }

}  // namespace
}  // namespace ulm
