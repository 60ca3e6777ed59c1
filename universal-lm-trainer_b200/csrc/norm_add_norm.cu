// The norms behind and in front of a block with the residual add between them (sm_100a): one pass each way.
//
//   fwd  u = b r1, r1 = rsqrt(mean(b^2) + eps);  z = x + s sig(g) v u;  y = w z r2, r2 = rsqrt(mean(z^2) + eps)
//   bwd  h = z r2, G = w dy;  dz = r2 (G - h mean(G h)) + gz;  dx = dz
//        n = s sig(g) v dz;  db = r1 (n - u mean(n u));  dg = s v u dz sig(g) (1 - sig(g))
//        dw = sum over rows of dy h;  C = sum over rows of dz sig(g) u;  dv = s C;  ds = v C, for one s its sum over the columns
//
// x, z and their gradients fp32; b, g, y and theirs 16-bit; s one number or one a column, g may be left out.  Statistics and sums fp32,
// one rounding to 16 bits.
//
// What bounds it: HBM, 12 bytes an element forward and 18 backward, 2 and 4 more with a gate.  A row belongs to L lanes of a CTA (half a warp, or
// whole ones) and stays in registers between its uses; a lane owns vectors of E elements.  The backward's second mean needs dz and so the first one:
// with dz = p - m q (p = r2 G + gz, q = r2 h, m = mean(G h)), sum(n u) = sum(t p u) - m sum(t q u) for t = s sig(g) v, so that all three
// sums of a row are formed before one barrier.  Column sums: per lane over a CTA's rows, added up over its groups in shared memory, a partial
// row per CTA, joined in a fixed order: no atomics.
#include <type_traits>

#include "common.cuh"
#include "norm_rows.cuh"
#include "pairs.cuh"

namespace ulm {
namespace {

constexpr int kMaxRow = 8192;
constexpr int kMostCtas = 2;                             // on an SM, of all forms of the backward: each leaves one partial row

// The sigmoid as its smaller side s = sig(-|g|) with the sign of g: sig(g) is s or 1 - s, its slope s (1 - s) without a difference that cancels.
// 2^x and the reciprocal are the special-function unit's, within 2^-22 and 2^-23; with the exponent's rounding s is within 2^-21 + |g| 2^-24 of
// itself, its other side within 2^-23.  With expf and an IEEE division, evaluated at both uses, 12011 x 1024 took 50 + 91 us.
__device__ __forceinline__ float2 shut(float2 g) {
  const float2 t = mul2(make_float2(fabsf(g.x), fabsf(g.y)), both(-1.44269504f));
  float2 e, q;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(t.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(t.y));
  const float2 d = add2(e, both(1.f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(q.x) : "f"(d.x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(q.y) : "f"(d.y));
  const float2 s = mul2(e, q);
  return make_float2(copysignf(s.x, g.x), copysignf(s.y, g.y));
}
// by its sign bit: s may be a zero; a NaN stays one
__device__ __forceinline__ float opened(float s) { return __float_as_int(s) < 0 ? -s : 1.f - s; }
__device__ __forceinline__ float2 opened(float2 s) { return make_float2(opened(s.x), opened(s.y)); }
// sig (1 - sig) = |s| - s^2
__device__ __forceinline__ float2 slope(float2 s) { return fma2(s, make_float2(-s.x, -s.y), make_float2(fabsf(s.x), fabsf(s.y))); }

// E fp32 columns: with E = 8 a lane takes 32 bytes in one access, so that a warp's is a kilobyte without gaps.  As two accesses of 16 bytes each
// would touch the same eight lines, and L1 was 72 % busy.  p on a multiple of 4 E bytes.
template <int E> __device__ __forceinline__ void load_row(const float* p, float2 (&v)[E / 2]) {
  if constexpr (E == 8) {
    asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=f"(v[0].x), "=f"(v[0].y), "=f"(v[1].x), "=f"(v[1].y), "=f"(v[2].x), "=f"(v[2].y), "=f"(v[3].x), "=f"(v[3].y) : "l"(p));
  } else {
    const float4 f = *reinterpret_cast<const float4*>(p);
    v[0] = make_float2(f.x, f.y); v[1] = make_float2(f.z, f.w);
  }
}
template <int E> __device__ __forceinline__ void store_row(float* p, const float2 (&v)[E / 2]) {
  if constexpr (E == 8)
    asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 :: "l"(p), "f"(v[0].x), "f"(v[0].y), "f"(v[1].x), "f"(v[1].y), "f"(v[2].x), "f"(v[2].y), "f"(v[3].x), "f"(v[3].y) : "memory");
  else *reinterpret_cast<float4*>(p) = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
}
template <typename TY, int E> __device__ __forceinline__ void unpack_row(const Raw<E>& r, float2 (&v)[E / 2]) {
#pragma unroll
  for (int j = 0; j < E / 2; ++j) v[j] = Cvt<TY>::unpack2(r.u[j]);
}
template <typename TY, int E> __device__ __forceinline__ void store_row16(TY* p, const float2 (&v)[E / 2]) {
  uint32_t u[E / 2];
#pragma unroll
  for (int j = 0; j < E / 2; ++j) u[j] = Cvt<TY>::pack2(v[j].x, v[j].y);
  if constexpr (E == 8) *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
  else *reinterpret_cast<uint2*>(p) = make_uint2(u[0], u[1]);
}

// the branch's factor: one number (on the device, or from the host) or one a column
struct Scale { const float* dev; float value; int channels; };
__device__ __forceinline__ float whole_scale(const Scale& s) { return s.channels ? 1.f : s.dev ? *s.dev : s.value; }
// v, times s where it is one a column: of E columns.  One s for all is applied by whoever calls, because its gradient, which may not
// be divided by it, is the sum without it.
template <int E>
__device__ __forceinline__ void load_tv(const float* v, const Scale& s, int col, float2 (&t)[E / 2]) {
  load_row<E>(v + col, t);
  if (s.channels) {
    float2 c[E / 2];
    load_row<E>(s.dev + col, c);
#pragma unroll
    for (int j = 0; j < E / 2; ++j) t[j] = mul2(t[j], c[j]);
  }
}

// A row belongs to L lanes: half a warp, or whole warps.
__device__ __forceinline__ uint32_t row_mask(int L, int lane) { return L == 16 ? 0xffffu << (lane & 16) : 0xffffffffu; }
// Sum over them.  `slots`: this call's own float a warp; consecutive calls of a warp alternate between two sets, so that one barrier a
// call is enough.
__device__ __forceinline__ float row_sum(float v, int L, int group, float* slots) {
  const int lane = threadIdx.x & 31;
  const uint32_t mask = row_mask(L, lane);
  if (L != 16) v += __shfl_xor_sync(mask, v, 16);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(mask, v, o);
  if (L <= 32) return v;
  const int warp = threadIdx.x >> 5, W = L >> 5;
  if (lane == 0) slots[warp] = v;
  asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(L) : "memory");
  float t = 0.f;
  for (int i = 0; i < W; ++i) t += slots[group * W + i];
  return t;
}

struct FwdParams {
  const float* x; const void* branch; const void* gate; const float* v; const float* w; Scale scale;
  float* x_out; void* y; float* rstd1; float* rstd2;
  int64_t x_stride, branch_stride, gate_stride, xout_stride, y_stride, rows;
  int d, L; float eps;
};

template <typename TY, int E, int NV, int WARPS, int CTAS, bool GATE>
__global__ void __launch_bounds__(WARPS * 32, CTAS)
norm_add_norm_fwd_kernel(const __grid_constant__ FwdParams p) {
  __shared__ float slots[2][WARPS];
  grid_dependents_go();
  grid_dependency_wait();
  const TY* br = static_cast<const TY*>(p.branch);
  const TY* gt = static_cast<const TY*>(p.gate);
  TY* y = static_cast<TY*>(p.y);
  const int L = p.L, group = threadIdx.x / L, groups = blockDim.x / L, nvec = p.d / E, first = threadIdx.x - group * L, hop = L;
  const float inv_d = 1.f / (float)p.d, whole = whole_scale(p.scale);
  for (int64_t r = (int64_t)blockIdx.x * groups + group; r < p.rows; r += (int64_t)gridDim.x * groups) {
    float2 z[NV][E / 2];
    Raw<E> b[NV], g[GATE ? NV : 1];
#pragma unroll
    for (int it = 0; it < NV; ++it) {                    // the whole row is requested before any of it is used
      const int vi = first + it * hop;
      if (vi < nvec) {
        b[it] = load_raw<TY, E>(br + r * p.branch_stride + vi * E);
        load_row<E>(p.x + r * p.x_stride + vi * E, z[it]);
        if constexpr (GATE) g[it] = load_raw<TY, E>(gt + r * p.gate_stride + vi * E);
      }
    }
    float2 sum = both(0.f);
#pragma unroll
    for (int it = 0; it < NV; ++it)
      if (first + it * hop < nvec) {
        float2 f[E / 2];
        unpack_row<TY, E>(b[it], f);
#pragma unroll
        for (int j = 0; j < E / 2; ++j) sum = fma2(f[j], f[j], sum);
      }
    const float r1 = rsqrtf(row_sum(sum.x + sum.y, L, group, slots[0]) * inv_d + p.eps);
    const float2 r1s = both(r1 * whole);
    sum = both(0.f);
#pragma unroll
    for (int it = 0; it < NV; ++it) {
      const int vi = first + it * hop;
      if (vi < nvec) {
        float2 f[E / 2], t[E / 2];
        unpack_row<TY, E>(b[it], f);
        load_tv<E>(p.v, p.scale, vi * E, t);
        if constexpr (GATE) {
          float2 o[E / 2];
          unpack_row<TY, E>(g[it], o);
#pragma unroll
          for (int j = 0; j < E / 2; ++j) t[j] = mul2(t[j], opened(shut(o[j])));
        }
#pragma unroll
        for (int j = 0; j < E / 2; ++j) {
          z[it][j] = fma2(mul2(f[j], r1s), t[j], z[it][j]);
          sum = fma2(z[it][j], z[it][j], sum);
        }
        store_row<E>(p.x_out + r * p.xout_stride + vi * E, z[it]);
      }
    }
    const float r2 = rsqrtf(row_sum(sum.x + sum.y, L, group, slots[1]) * inv_d + p.eps);
    if (first == 0) {
      p.rstd1[r] = r1;
      p.rstd2[r] = r2;
    }
#pragma unroll
    for (int it = 0; it < NV; ++it) {
      const int vi = first + it * hop;
      if (vi < nvec) {
        float2 wv[E / 2];
        load_row<E>(p.w + vi * E, wv);
#pragma unroll
        for (int j = 0; j < E / 2; ++j) wv[j] = mul2(mul2(z[it][j], both(r2)), wv[j]);
        store_row16<TY, E>(y + r * p.y_stride + vi * E, wv);
      }
    }
  }
}

// Asks for a row that will be wanted soon, into L2: the whole 16 bytes of it.
__device__ __forceinline__ void fetch_to_l2(const void* from, int bytes) {
  const uint64_t begin = (reinterpret_cast<uint64_t>(from) + 15) & ~15ull, end = (reinterpret_cast<uint64_t>(from) + bytes) & ~15ull;
  if (end > begin) asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(begin), "r"((uint32_t)(end - begin)) : "memory");
}

struct BwdParams {
  const float* z; const void* branch; const void* gate; const float* v; const float* w; Scale scale;
  const void* dy; const float* gz; const float* rstd1; const float* rstd2;
  float* dx; void* db; void* dg; float* partial;
  int64_t z_stride, branch_stride, gate_stride, dy_stride, gz_stride, dx_stride, db_stride, dg_stride, rows;
  int d, L, ahead;                                       // ahead: whether the next row is asked for
};

// Three sums over the L lanes of a row, one barrier where they are more than a warp.  Every exchange between lanes halves the number of sums
// that a lane carries: six of them instead of fifteen.  `slots` as for row_sum, a float4 a warp.
__device__ __forceinline__ void row_sums(float& a, float& b, float& c, int L, int group, float4* slots) {
  const int lane = threadIdx.x & 31, top = L == 16 ? 8 : 16;
  const uint32_t mask = row_mask(L, lane);
  const bool up = lane & top, right = lane & (top >> 1);
  float s0 = up ? c : a, s1 = up ? 0.f : b;              // the lower half of the lanes goes on with a and b, the upper with c
  s0 += __shfl_xor_sync(mask, up ? a : c, top);
  s1 += __shfl_xor_sync(mask, up ? b : 0.f, top);
  float t = right ? s1 : s0;
  t += __shfl_xor_sync(mask, right ? s0 : s1, top >> 1);
  if (L != 16) t += __shfl_xor_sync(mask, t, 4);
  t += __shfl_xor_sync(mask, t, 2);
  t += __shfl_xor_sync(mask, t, 1);
  if (L <= 32) {
    const int base = L == 16 ? lane & 16 : 0;
    a = __shfl_sync(mask, t, base);
    b = __shfl_sync(mask, t, base + (top >> 1));
    c = __shfl_sync(mask, t, base + top);
    return;
  }
  const int warp = threadIdx.x >> 5, W = L >> 5;
  if ((lane & 7) == 0) reinterpret_cast<float*>(slots + warp)[lane >> 3] = t;
  asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(L) : "memory");
  a = b = c = 0.f;
  for (int k = 0; k < W; ++k) {
    const float4 q = slots[group * W + k];
    a += q.x; b += q.y; c += q.z;
  }
}

template <typename TY, int E, int NV, int WARPS, int CTAS, bool GATE>
__global__ void __launch_bounds__(WARPS * 32, CTAS)
norm_add_norm_bwd_kernel(const __grid_constant__ BwdParams p) {
  extern __shared__ float s_sum[];                       // [groups][d]
  __shared__ float4 slots[2][WARPS];
  grid_dependents_go();
  grid_dependency_wait();
  const TY* br = static_cast<const TY*>(p.branch);
  const TY* gt = static_cast<const TY*>(p.gate);
  const TY* dy = static_cast<const TY*>(p.dy);
  TY* db = static_cast<TY*>(p.db);
  TY* dg = static_cast<TY*>(p.dg);
  const int L = p.L, group = threadIdx.x / L, groups = blockDim.x / L, nvec = p.d / E, first = threadIdx.x - group * L, hop = L;
  const float inv_d = 1.f / (float)p.d, whole = whole_scale(p.scale);
  // a lane has the same columns of every row: their weights stay in registers where there are few
  constexpr bool kHold = NV * E <= 16, kKeepGate = GATE && NV * E <= 16;      // as do the gate's values of a row, formed twice otherwise
  float2 wv[kHold ? NV : 1][E / 2], tv[kHold ? NV : 1][E / 2], acc_w[NV][E / 2], acc_c[NV][E / 2];
  float acc_s = 0.f;
#pragma unroll
  for (int it = 0; it < NV; ++it) {
    if (kHold && first + it * hop < nvec) {
      load_row<E>(p.w + (first + it * hop) * E, wv[it]);
      load_tv<E>(p.v, p.scale, (first + it * hop) * E, tv[it]);
    }
#pragma unroll
    for (int j = 0; j < E / 2; ++j) acc_w[it][j] = acc_c[it][j] = both(0.f);
  }
  int phase = 0;
  for (int64_t r = (int64_t)blockIdx.x * groups + group; r < p.rows; r += (int64_t)gridDim.x * groups, phase ^= 1) {
    float2 z[NV][E / 2], gz[NV][E / 2], shuts[kKeepGate ? NV : 1][E / 2];
    Raw<E> b[NV], q[NV], g[GATE ? NV : 1];
#pragma unroll
    for (int it = 0; it < NV; ++it) {                    // the whole row is requested before any of it is used
      const int vi = first + it * hop;
      if (vi < nvec) {
        load_row<E>(p.z + r * p.z_stride + vi * E, z[it]);
        q[it] = load_raw<TY, E>(dy + r * p.dy_stride + vi * E);
        b[it] = load_raw<TY, E>(br + r * p.branch_stride + vi * E);
        if constexpr (GATE) g[it] = load_raw<TY, E>(gt + r * p.gate_stride + vi * E);
        if (p.gz) {
          load_row<E>(p.gz + r * p.gz_stride + vi * E, gz[it]);
        } else {
#pragma unroll
          for (int j = 0; j < E / 2; ++j) gz[it][j] = both(0.f);
        }
      }
    }
    if (p.ahead && first == 0) {               // the group's next row is on its way to L2 while this one is worked on
      const int64_t next = r + (int64_t)gridDim.x * groups;
      if (next < p.rows) {
        fetch_to_l2(p.z + next * p.z_stride, 4 * p.d);
        fetch_to_l2(dy + next * p.dy_stride, 2 * p.d);
        fetch_to_l2(br + next * p.branch_stride, 2 * p.d);
        if (p.gz) fetch_to_l2(p.gz + next * p.gz_stride, 4 * p.d);
        if constexpr (GATE) fetch_to_l2(gt + next * p.gate_stride, 2 * p.d);
      }
    }
    const float r1 = p.rstd1[r], r2 = p.rstd2[r];
    float2 gh2 = both(0.f), pt2 = gh2, ht2 = gh2;
#pragma unroll
    for (int it = 0; it < NV; ++it) {
      const int vi = first + it * hop, at = kHold ? it : 0, keep = kKeepGate ? it : 0;
      if (vi < nvec) {
        float2 G[E / 2], u[E / 2];
        if constexpr (!kHold) {
          load_row<E>(p.w + vi * E, wv[0]);
          load_tv<E>(p.v, p.scale, vi * E, tv[0]);
        }
        unpack_row<TY, E>(q[it], G);
        unpack_row<TY, E>(b[it], u);
        if constexpr (GATE) {
          unpack_row<TY, E>(g[it], shuts[keep]);
#pragma unroll
          for (int j = 0; j < E / 2; ++j) shuts[keep][j] = shut(shuts[keep][j]);
        }
#pragma unroll
        for (int j = 0; j < E / 2; ++j) {
          z[it][j] = mul2(z[it][j], both(r2));           // h from here on
          const float2 tu = mul2(GATE ? mul2(tv[at][j], opened(shuts[keep][j])) : tv[at][j], mul2(u[j], both(r1))), a = mul2(G[j], z[it][j]);
          acc_w[it][j] = add2(acc_w[it][j], a);
          gh2 = fma2(a, wv[at][j], gh2);
          gz[it][j] = fma2(mul2(G[j], wv[at][j]), both(r2), gz[it][j]);      // p from here on
          pt2 = fma2(gz[it][j], tu, pt2);
          ht2 = fma2(z[it][j], tu, ht2);
        }
      }
    }
    float gh = gh2.x + gh2.y, pt = pt2.x + pt2.y, ht = ht2.x + ht2.y;
    row_sums(gh, pt, ht, L, group, slots[phase]);
    const float m = gh * inv_d * r2, nu = pt - m * ht, rs = r1 * whole, k = nu * inv_d * rs * r1;      // dz = p - m h
    acc_s += nu;
#pragma unroll
    for (int it = 0; it < NV; ++it) {
      const int vi = first + it * hop, at = kHold ? it : 0, keep = kKeepGate ? it : 0;
      if (vi < nvec) {
        float2 u[E / 2], o[E / 2];
        unpack_row<TY, E>(b[it], u);
        if constexpr (!kHold) load_tv<E>(p.v, p.scale, vi * E, tv[0]);
        if constexpr (GATE && !kKeepGate) {
          unpack_row<TY, E>(g[it], shuts[0]);
#pragma unroll
          for (int j = 0; j < E / 2; ++j) shuts[0][j] = shut(shuts[0][j]);
        }
#pragma unroll
        for (int j = 0; j < E / 2; ++j) gz[it][j] = fma2(both(-m), z[it][j], gz[it][j]);      // dz from here on
        store_row<E>(p.dx + r * p.dx_stride + vi * E, gz[it]);
#pragma unroll
        for (int j = 0; j < E / 2; ++j) {
          const float2 ds = GATE ? mul2(gz[it][j], opened(shuts[keep][j])) : gz[it][j];
          acc_c[it][j] = fma2(ds, mul2(u[j], both(r1)), acc_c[it][j]);
          o[j] = fma2(mul2(ds, both(rs)), tv[at][j], mul2(u[j], both(-k)));
          if constexpr (GATE) gz[it][j] = mul2(mul2(gz[it][j], slope(shuts[keep][j])), mul2(mul2(u[j], both(rs)), tv[at][j]));
        }
        store_row16<TY, E>(db + r * p.db_stride + vi * E, o);
        if constexpr (GATE) store_row16<TY, E>(dg + r * p.dg_stride + vi * E, gz[it]);
      }
    }
  }
  // a CTA's partial row: dw, C, and the sum of n u / s over its rows
  float* out = p.partial + (int64_t)blockIdx.x * (2 * p.d + 1);
#pragma unroll
  for (int set = 0; set < 2; ++set) {
    if (set) __syncthreads();                            // the first set has been read
#pragma unroll
    for (int it = 0; it < NV; ++it) {
      const int vi = first + it * hop;
      if (vi < nvec) {
#pragma unroll
        for (int j = 0; j < E / 2; ++j) *reinterpret_cast<float2*>(s_sum + group * p.d + vi * E + 2 * j) = set ? acc_c[it][j] : acc_w[it][j];
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < p.d; c += (int)blockDim.x) {
      float t = 0.f;
      for (int g = 0; g < groups; ++g) t += s_sum[g * p.d + c];
      out[set * p.d + c] = t;
    }
  }
  __syncthreads();
  if (first == 0) s_sum[group] = acc_s;
  __syncthreads();
  if (threadIdx.x == 0) {
    float t = 0.f;
    for (int g = 0; g < groups; ++g) t += s_sum[g];
    out[2 * p.d] = t;
  }
}

// The partial rows' sums in a fixed order, as col_sum_kernel has them, and what follows from them: columns [0, d) are dw, [d, 2d) C,
// the last is the gradient of the one s.
__global__ void __launch_bounds__(1024)
norm_add_norm_finish_kernel(const float* partial, const float* v, const Scale scale, float* dw, float* dv, float* ds, int nparts, int d) {
  __shared__ float sub[32][33];
  grid_dependency_wait();
  const int c = blockIdx.x * 32 + threadIdx.x, width = 2 * d + 1;
  constexpr int kParts = (kMostCtas * kNumSMs + 31) / 32;
  float t = 0.f, part[kParts];                           // all requested before the first is added
  if (c < width) {
#pragma unroll
    for (int k = 0; k < kParts; ++k) {
      const int row = threadIdx.y + 32 * k;
      part[k] = row < nparts ? partial[(int64_t)row * width + c] : 0.f;
    }
#pragma unroll
    for (int k = 0; k < kParts; ++k) t += part[k];
  }
  sub[threadIdx.y][threadIdx.x] = t;
  __syncthreads();
  if (threadIdx.y != 0 || c >= width) return;
  float sum = 0.f;
#pragma unroll
  for (int g = 0; g < 32; ++g) sum += sub[g][threadIdx.x];
  if (c < d) dw[c] = sum;
  else if (c < 2 * d) {
    const int i = c - d;
    dv[i] = sum * (scale.channels ? scale.dev[i] : whole_scale(scale));
    if (ds && scale.channels) ds[i] = sum * v[i];
  } else if (ds && !scale.channels) {
    ds[0] = sum;
  }
}

// fp32 rows that vectors of eight may be read from
bool ok256(const void* p, int64_t stride) { return !(reinterpret_cast<uintptr_t>(p) & 31) && stride % 8 == 0; }

int check_shape(const char* who, int dtype, int d, int64_t rows) {
  if (dtype != ULM_F16 && dtype != ULM_BF16) return fail(ULM_ERR_ARG, "%s: branch, gate and y are fp16 or bf16", who);
  if (d <= 0 || d % 4 || rows < 0) return fail(ULM_ERR_ARG, "%s: need rows >= 0 and d a positive multiple of 4", who);
  if (d > kMaxRow) return fail(ULM_ERR_TOO_LARGE, "%s: rows of at most %d elements", who, kMaxRow);
  return ULM_OK;
}

// A kernel's form: vectors of E columns a lane, warps of a CTA, CTAs on an SM, rows that a full CTA has at least; the columns that this allows.
template <int E_, int NV_, int WARPS_, int CTAS_, int ROWS> struct Form {
  static constexpr int E = E_, NV = NV_, WARPS = WARPS_, CTAS = CTAS_, kMost = E * NV * 32 * (WARPS / ROWS);
};
template <typename...> struct Forms {};
// The first form whose columns suffice.  us at us of the bytes alone (bf16, without a gate, then with one):
//   forward   32768 x 768 47 (46), x 1024 63 (61), 16396 x 4096 125 (123); 48044 x 1024 105 (105), 16396 x 4096 146 (144).  One warp a row up to
//             1024 columns: with eight columns a lane, and so three warps and two barriers for 768, 32768 x 768 took 65.  Nine warps where a row takes
//             three: 8192 x 2560 53 -> 45, 5000 x 2816 36 -> 32
//   backward  32768 x 768 76 (69), x 1024 99 (92), 16396 x 4096 196 (184); 48044 x 1024 169 (165), 16396 x 4096 252 (225).  Eight columns a lane and
//             24 warps an SM without a gate up to 1024 (sixteen a lane: 87 at 768); the gate's values do not fit the 80 registers of that,
//             and with sixteen a lane 48044 x 1024 went from 204 to 181.  Thirty-two from where two rows no longer fit a CTA, the gate formed at both uses:
//             16396 x 4096 with a gate 340 -> 281; above 4096 columns one row is on an SM: 4096 x 5120 90 (58), x 8192 110 (92).  A group then waits for a row, meets at a barrier and stores before it loads the
//             next, and few rows are on an SM at a time: the next row asked for into L2 meanwhile took 48044 x 1024 from 181 to 169,
//             16396 x 4096 with a gate from 281 to 252, 5000 x 2816 from 55 to 48; rows of 128 and 256 columns, of which many are under
//             way, from 18.5 to 20.6 (so from kAheadFrom on only: 512 with a gate 38.9 -> 38.0).  Copies of the row itself, by cp.async into shared memory
//             a row ahead, cost more load and store instructions than the wait they saved: 32768 x 768 98, 4099 x 4096 with a gate 94
constexpr int kAheadFrom = 512;
using Fwd8 = Forms<Form<8, 1, 8, 4, 8>, Form<8, 2, 8, 3, 8>, Form<8, 3, 8, 3, 8>, Form<8, 4, 8, 2, 4>, Form<8, 4, 9, 2, 3>, Form<8, 4, 8, 2, 1>>;
using Bwd8 = Forms<Form<8, 1, 12, 2, 3>, Form<8, 2, 12, 1, 2>, Form<8, 4, 8, 1, 1>>;
using Bwd8Gate = Forms<Form<8, 1, 20, 1, 6>, Form<8, 2, 12, 1, 2>, Form<8, 4, 8, 1, 1>>;
// widths of 4 modulo 8, and tensors that lie on multiples of 8 or 16 bytes only: 20000 x 772 with a gate 50 + 85 (33 + 52), 22721 x 796 49 + 65 (33 + 50),
// 30000 x 300 with a gate 30 + 70 (19 + 30; eight vectors a lane 43 + 64), 4096 x 4100 53 + 120 (31 + 46), with a gate 61 + 166 (36 + 56).  The backward's
// forms were chosen without a gate; with one, 80 registers spill (184 bytes a thread for 132 to 768 columns), and 128 do above 4096 (420; 188 without)
using Fwd4 = Forms<Form<4, 1, 8, 4, 8>, Form<4, 4, 8, 3, 8>, Form<4, 6, 8, 2, 8>, Form<4, 8, 8, 2, 1>>;
using Bwd4 = Forms<Form<4, 1, 16, 2, 16>, Form<4, 2, 12, 2, 4>, Form<4, 4, 12, 1, 2>, Form<4, 8, 8, 1, 2>, Form<4, 4, 16, 1, 1>>;

// Lanes a row and rows a CTA.  Few rows (less than the SMs take at full CTAs) are spread over more, smaller CTAs.
struct Deal { int L, groups, threads; };
template <typename F> Deal deal(int64_t rows, int d) {
  Deal s;
  const int nvec = d / F::E;
  s.L = nvec <= 16 ? 16 : 32 * ceil_div(nvec, 32 * F::NV);
  s.groups = F::WARPS * 32 / s.L;
  const int64_t spread = (rows + kNumSMs - 1) / kNumSMs;
  if (spread < s.groups) s.groups = spread < 1 ? 1 : (int)spread;
  s.threads = ceil_div(s.groups * s.L, 32) * 32;
  s.groups = s.threads / s.L;
  return s;
}

template <typename TY, bool GATE, typename F, typename... Rest>
int launch_fwd(Forms<F, Rest...>, FwdParams p, cudaStream_t st, const char* who) {
  if constexpr (sizeof...(Rest) > 0) {
    if (p.d > F::kMost) return launch_fwd<TY, GATE>(Forms<Rest...>(), p, st, who);
  } else {
    static_assert(F::kMost >= kMaxRow, "the last form takes every row");
  }
  const Deal s = deal<F>(p.rows, p.d);
  p.L = s.L;
  const int64_t blocks = (p.rows + s.groups - 1) / s.groups;
  auto kern = norm_add_norm_fwd_kernel<TY, F::E, F::NV, F::WARPS, F::CTAS, GATE>;
  return launch_dependent(who, kern, (unsigned)(blocks < 64 * kNumSMs ? blocks : 64 * kNumSMs), s.threads, 0, st, p);
}

template <typename TY, bool GATE, typename F, typename... Rest>
int launch_bwd(Forms<F, Rest...>, BwdParams p, int64_t* parts, cudaStream_t st, const char* who) {
  if constexpr (sizeof...(Rest) > 0) {
    if (p.d > F::kMost) return launch_bwd<TY, GATE>(Forms<Rest...>(), p, parts, st, who);
  } else {
    static_assert(F::kMost >= kMaxRow, "the last form takes every row");
  }
  const Deal s = deal<F>(p.rows, p.d);
  p.L = s.L;
  p.ahead = p.d >= kAheadFrom;
  const size_t smem = (size_t)s.groups * p.d * sizeof(float);       // a warp has E NV 32 columns at most
  static_assert(F::CTAS <= kMostCtas && (F::E * F::NV * F::WARPS * 32 + 8 * F::WARPS) * sizeof(float) <= 48 * 1024, "partial rows; shared memory without an opt-in");
  auto kern = norm_add_norm_bwd_kernel<TY, F::E, F::NV, F::WARPS, F::CTAS, GATE>;
  const int64_t want = (p.rows + s.groups - 1) / s.groups;
  *parts = want < F::CTAS * kNumSMs ? want : F::CTAS * kNumSMs;
  return launch_dependent(who, kern, (unsigned)*parts, s.threads, smem, st, p);
}
template <typename TY, bool GATE>
int launch(const FwdParams& p, int E, cudaStream_t st, const char* who) {
  return E == 8 ? launch_fwd<TY, GATE>(Fwd8(), p, st, who) : launch_fwd<TY, GATE>(Fwd4(), p, st, who);
}
template <typename TY, bool GATE>
int launch(const BwdParams& p, int E, int64_t* parts, cudaStream_t st, const char* who) {
  using Wide = std::conditional_t<GATE, Bwd8Gate, Bwd8>;
  return E == 8 ? launch_bwd<TY, GATE>(Wide(), p, parts, st, who) : launch_bwd<TY, GATE>(Bwd4(), p, parts, st, who);
}

}  // namespace
}  // namespace ulm

extern "C" int ulm_norm_add_norm_fwd(const ulm_norm_add_norm_fwd_args* a) {
  using namespace ulm;
  const char* who = "ulm_norm_add_norm_fwd";
  if (!a) return fail(ULM_ERR_ARG, "%s: null args", who);
  if (int rc = check_shape(who, a->dtype, a->d, a->rows)) return rc;
  if (a->scale_channels && !a->scale) return fail(ULM_ERR_ARG, "%s: a scale a column is read from the device", who);
  if (a->rows == 0) return ULM_OK;
  if (!a->x || !a->branch || !a->v || !a->w || !a->x_out || !a->y || !a->rstd_branch || !a->rstd) return fail(ULM_ERR_ARG, "%s: null tensor", who);
  if (!ok32(a->x, a->x_stride) || !ok32(a->x_out, a->xout_stride) || !ok32(a->v, 0) || !ok32(a->w, 0) || (a->scale_channels && !ok32(a->scale, 0)) ||
      !ok16(a->branch, a->branch_stride, 4) || !ok16(a->gate, a->gate_stride, 4) || !ok16(a->y, a->y_stride, 4))
    return fail(ULM_ERR_ARG, "%s: fp32 rows must be 16-byte aligned, 16-bit rows 8-byte aligned", who);
  const int E = a->d % 8 == 0 && ok16(a->branch, a->branch_stride, 8) && ok16(a->gate, a->gate_stride, 8) && ok16(a->y, a->y_stride, 8) && ok256(a->x, a->x_stride) &&
                        ok256(a->x_out, a->xout_stride) && ok256(a->v, 0) && ok256(a->w, 0) && (!a->scale_channels || ok256(a->scale, 0)) ? 8 : 4;
  const FwdParams p{a->x, a->branch, a->gate, a->v, a->w, {a->scale, a->scale_value, a->scale_channels}, a->x_out, a->y, a->rstd_branch, a->rstd,
                    a->x_stride, a->branch_stride, a->gate_stride, a->xout_stride, a->y_stride, a->rows, a->d, 1, a->eps};
  cudaStream_t st = (cudaStream_t)a->stream;
  auto go = [&](auto t) { return a->gate ? launch<decltype(t), true>(p, E, st, who) : launch<decltype(t), false>(p, E, st, who); };
  return a->dtype == ULM_F16 ? go(__half()) : go(__nv_bfloat16());
}

// one CTA a row, or as many as run at a time
extern "C" int64_t ulm_norm_add_norm_partial(int64_t rows, int32_t d) {
  const int64_t most = ulm::kMostCtas * ulm::kNumSMs, n = rows < 1 ? 1 : rows < most ? rows : most;
  return n * (2 * (int64_t)d + 1);
}

extern "C" int ulm_norm_add_norm_bwd(const ulm_norm_add_norm_bwd_args* a) {
  using namespace ulm;
  const char* who = "ulm_norm_add_norm_bwd";
  if (!a) return fail(ULM_ERR_ARG, "%s: null args", who);
  if (int rc = check_shape(who, a->dtype, a->d, a->rows)) return rc;
  if (a->scale_channels && !a->scale) return fail(ULM_ERR_ARG, "%s: a scale a column is read from the device", who);
  if (!a->dw || !a->dv || !a->v || (a->rows > 0 && (!a->x || !a->branch || !a->w || !a->dy || !a->rstd_branch || !a->rstd || !a->dx || !a->d_branch || !a->partial)) ||
      (a->rows > 0 && (a->gate != nullptr) != (a->d_gate != nullptr)))
    return fail(ULM_ERR_ARG, "%s: null tensor", who);
  if (a->rows > 0 && (!ok32(a->x, a->x_stride) || !ok32(a->dx, a->dx_stride) || !ok32(a->g_add, a->gadd_stride) || !ok32(a->v, 0) || !ok32(a->w, 0) ||
                      (a->scale_channels && !ok32(a->scale, 0)) || !ok16(a->branch, a->branch_stride, 4) || !ok16(a->gate, a->gate_stride, 4) ||
                      !ok16(a->dy, a->dy_stride, 4) || !ok16(a->d_branch, a->dbranch_stride, 4) || !ok16(a->d_gate, a->dgate_stride, 4)))
    return fail(ULM_ERR_ARG, "%s: fp32 rows must be 16-byte aligned, 16-bit rows 8-byte aligned", who);
  const int E = a->d % 8 == 0 && ok16(a->branch, a->branch_stride, 8) && ok16(a->gate, a->gate_stride, 8) && ok16(a->dy, a->dy_stride, 8) &&
                        ok16(a->d_branch, a->dbranch_stride, 8) && ok16(a->d_gate, a->dgate_stride, 8) && ok256(a->x, a->x_stride) && ok256(a->dx, a->dx_stride) &&
                        ok256(a->g_add, a->gadd_stride) && ok256(a->v, 0) && ok256(a->w, 0) && (!a->scale_channels || ok256(a->scale, 0)) ? 8 : 4;
  cudaStream_t st = (cudaStream_t)a->stream;
  const Scale scale{a->scale, a->scale_value, a->scale_channels};
  int64_t blocks = 0;
  if (a->rows > 0) {
    const BwdParams p{a->x, a->branch, a->gate, a->v, a->w, scale, a->dy, a->g_add, a->rstd_branch, a->rstd, a->dx, a->d_branch, a->d_gate, a->partial,
                      a->x_stride, a->branch_stride, a->gate_stride, a->dy_stride, a->gadd_stride, a->dx_stride, a->dbranch_stride, a->dgate_stride, a->rows, a->d, 1};
    auto go = [&](auto t) { return a->gate ? launch<decltype(t), true>(p, E, &blocks, st, who) : launch<decltype(t), false>(p, E, &blocks, st, who); };
    if (int rc = a->dtype == ULM_F16 ? go(__half()) : go(__nv_bfloat16())) return rc;
  }
  return launch_dependent(who, norm_add_norm_finish_kernel, (2 * a->d + 1 + 31) / 32, dim3(32, 32), 0, st, a->partial, a->v, scale, a->dw, a->dv, a->dscale, (int)blocks, a->d);
}
