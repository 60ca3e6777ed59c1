// The norms behind and in front of a block with the residual add between them (sm_100a): one pass each way.
//
//   fwd  u = b r1, r1 = rsqrt(mean(b^2) + eps);  z = x + s sig(g) v u;  y = w z r2, r2 = rsqrt(mean(z^2) + eps)
//   bwd  h = z r2, G = w dy;  dz = r2 (G - h mean(G h)) + gz;  dx = dz
//        n = s sig(g) v dz;  db = r1 (n - u mean(n u));  dg = s v u dz sig(g) (1 - sig(g))
//        dw = sum over rows of dy h;  C = sum over rows of dz sig(g) u;  dv = s C;  ds = v C, for one s its sum over the columns
//
// x, z and their gradients fp32; b, g, y and theirs 16-bit; s one number or one a column, g may be left out.  Statistics and sums fp32,
// one rounding to 16 bits; exponent and division of the sigmoid in full, because z keeps what they leave.
//
// What bounds it: HBM, 12 bytes an element forward and 18 backward, 2 and 4 more with a gate.  A row belongs to W warps of a CTA and stays
// in registers between its uses; a lane owns vectors of E elements.  The backward's second mean needs dz and so the first one:
// with dz = p - m q (p = r2 G + gz, q = r2 h, m = mean(G h)), sum(n u) = sum(t p u) - m sum(t q u) for t = s sig(g) v, so that all three
// sums of a row are formed before one barrier.  Column sums: per lane over a CTA's rows, added up over its groups in shared memory, a partial
// row per CTA, joined in a fixed order: no atomics.
#include "common.cuh"
#include "norm_rows.cuh"

namespace ulm {
namespace {

constexpr int kMaxRow = 8192;
constexpr int kFwdWarps = 8, kBwdWarps = 12, kBwdWideWarps = 16;

// sig(g), and sig(g) (1 - sig(g)) without a difference
__device__ __forceinline__ float opened(float g, float& slope) {
  const float e = expf(-fabsf(g)), q = 1.f / (1.f + e);
  slope = e * q * q;
  return g >= 0.f ? q : e * q;                           // a NaN is not, and stays one
}
__device__ __forceinline__ float opened(float g) { float slope; return opened(g, slope); }

// the branch's factor: one number (on the device, or from the host) or one a column
struct Scale { const float* dev; float value; int channels; };
__device__ __forceinline__ float whole_scale(const Scale& s) { return s.channels ? 1.f : s.dev ? *s.dev : s.value; }
// v, times s where it is one a column: of E columns.  One s for all is applied by whoever calls, because its gradient, which may not
// be divided by it, is the sum without it.
template <int E>
__device__ __forceinline__ void load_tv(const float* v, const Scale& s, int col, float (&t)[E]) {
  load_f32<E>(v + col, t);
  if (s.channels) {
    float c[E];
    load_f32<E>(s.dev + col, c);
#pragma unroll
    for (int j = 0; j < E; ++j) t[j] *= c[j];
  }
}

struct FwdParams {
  const float* x; const void* branch; const void* gate; const float* v; const float* w; Scale scale;
  float* x_out; void* y; float* rstd1; float* rstd2;
  int64_t x_stride, branch_stride, gate_stride, xout_stride, y_stride, rows;
  int d, W; float eps;
};

template <typename TY, int E, int NV, bool GATE>
__global__ void __launch_bounds__(kFwdWarps * 32, 3)
norm_add_norm_fwd_kernel(const __grid_constant__ FwdParams p) {
  __shared__ float slots[2][kFwdWarps];
  grid_dependents_go();
  grid_dependency_wait();
  const TY* br = static_cast<const TY*>(p.branch);
  const TY* gt = static_cast<const TY*>(p.gate);
  TY* y = static_cast<TY*>(p.y);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, W = p.W;
  const int group = warp / W, part = warp - group * W, groups = (int)(blockDim.x >> 5) / W;
  const int nvec = p.d / E, first = part * 32 + lane, hop = W * 32;
  const float inv_d = 1.f / (float)p.d, whole = whole_scale(p.scale);
  for (int64_t r = (int64_t)blockIdx.x * groups + group; r < p.rows; r += (int64_t)gridDim.x * groups) {
    float z[NV][E];
    Raw<E> b[NV], g[GATE ? NV : 1];
#pragma unroll
    for (int it = 0; it < NV; ++it) {                    // the whole row is requested before any of it is used
      const int vi = first + it * hop;
      if (vi < nvec) {
        b[it] = load_raw<TY, E>(br + r * p.branch_stride + vi * E);
        load_f32<E>(p.x + r * p.x_stride + vi * E, z[it]);
        if constexpr (GATE) g[it] = load_raw<TY, E>(gt + r * p.gate_stride + vi * E);
      }
    }
    float sum = 0.f;
#pragma unroll
    for (int it = 0; it < NV; ++it)
      if (first + it * hop < nvec) {
        float f[E];
        unpack_raw<TY, E>(b[it], f);
#pragma unroll
        for (int j = 0; j < E; ++j) sum += f[j] * f[j];
      }
    const float r1 = rsqrtf(row_sum(sum, W, group, warp, lane, slots[0]) * inv_d + p.eps), r1s = r1 * whole;
    sum = 0.f;
#pragma unroll
    for (int it = 0; it < NV; ++it) {
      const int vi = first + it * hop;
      if (vi < nvec) {
        float f[E], t[E];
        unpack_raw<TY, E>(b[it], f);
        load_tv<E>(p.v, p.scale, vi * E, t);
        if constexpr (GATE) {
          float o[E];
          unpack_raw<TY, E>(g[it], o);
#pragma unroll
          for (int j = 0; j < E; ++j) t[j] *= opened(o[j]);
        }
#pragma unroll
        for (int j = 0; j < E; ++j) {
          z[it][j] = fmaf(f[j] * r1s, t[j], z[it][j]);
          sum += z[it][j] * z[it][j];
        }
        store_f32<E>(p.x_out + r * p.xout_stride + vi * E, z[it]);
      }
    }
    const float r2 = rsqrtf(row_sum(sum, W, group, warp, lane, slots[1]) * inv_d + p.eps);
    if (first == 0) {
      p.rstd1[r] = r1;
      p.rstd2[r] = r2;
    }
#pragma unroll
    for (int it = 0; it < NV; ++it) {
      const int vi = first + it * hop;
      if (vi < nvec) {
        float wv[E], o[E];
        load_f32<E>(p.w + vi * E, wv);
#pragma unroll
        for (int j = 0; j < E; ++j) o[j] = z[it][j] * r2 * wv[j];
        store_16<TY, E>(y + r * p.y_stride + vi * E, o);
      }
    }
  }
}

struct BwdParams {
  const float* z; const void* branch; const void* gate; const float* v; const float* w; Scale scale;
  const void* dy; const float* gz; const float* rstd1; const float* rstd2;
  float* dx; void* db; void* dg; float* partial;
  int64_t z_stride, branch_stride, gate_stride, dy_stride, gz_stride, dx_stride, db_stride, dg_stride, rows;
  int d, W;
};

// Three sums over the W warps of a row, one barrier; `slots` as for row_sum, three floats a warp.
template <int WARPS>
__device__ __forceinline__ void row_sums(float (&v)[3], int W, int group, int warp, int lane, float (*slots)[WARPS]) {
#pragma unroll
  for (int i = 0; i < 3; ++i) v[i] = warp_sum(v[i]);
  if (W == 1) return;
  if (lane < 3) slots[lane][warp] = lane == 0 ? v[0] : lane == 1 ? v[1] : v[2];
  asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(32 * W) : "memory");
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    v[i] = 0.f;
    for (int k = 0; k < W; ++k) v[i] += slots[i][group * W + k];
  }
}

template <typename TY, int E, int NV, int WARPS, bool GATE>
__global__ void __launch_bounds__(WARPS * 32, WARPS == kBwdWideWarps ? 1 : 2)
norm_add_norm_bwd_kernel(const __grid_constant__ BwdParams p) {
  extern __shared__ float s_sum[];                       // [groups][d]
  __shared__ float slots[2][3][WARPS];
  grid_dependents_go();
  grid_dependency_wait();
  const TY* br = static_cast<const TY*>(p.branch);
  const TY* gt = static_cast<const TY*>(p.gate);
  const TY* dy = static_cast<const TY*>(p.dy);
  TY* db = static_cast<TY*>(p.db);
  TY* dg = static_cast<TY*>(p.dg);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, W = p.W;
  const int group = warp / W, part = warp - group * W, groups = (int)(blockDim.x >> 5) / W;
  const int nvec = p.d / E, first = part * 32 + lane, hop = W * 32;
  const float inv_d = 1.f / (float)p.d, whole = whole_scale(p.scale);
  float acc_w[NV][E], acc_c[NV][E], acc_s = 0.f;
#pragma unroll
  for (int it = 0; it < NV; ++it)
#pragma unroll
    for (int j = 0; j < E; ++j) acc_w[it][j] = acc_c[it][j] = 0.f;
  int phase = 0;
  for (int64_t r = (int64_t)blockIdx.x * groups + group; r < p.rows; r += (int64_t)gridDim.x * groups, phase ^= 1) {
    float z[NV][E], gz[NV][E];
    Raw<E> b[NV], q[NV], g[GATE ? NV : 1];
#pragma unroll
    for (int it = 0; it < NV; ++it) {
      const int vi = first + it * hop;
      if (vi < nvec) {
        load_f32<E>(p.z + r * p.z_stride + vi * E, z[it]);
        q[it] = load_raw<TY, E>(dy + r * p.dy_stride + vi * E);
        b[it] = load_raw<TY, E>(br + r * p.branch_stride + vi * E);
        if constexpr (GATE) g[it] = load_raw<TY, E>(gt + r * p.gate_stride + vi * E);
        if (p.gz) {
          load_f32<E>(p.gz + r * p.gz_stride + vi * E, gz[it]);
        } else {
#pragma unroll
          for (int j = 0; j < E; ++j) gz[it][j] = 0.f;
        }
      }
    }
    const float r1 = p.rstd1[r], r2 = p.rstd2[r];
    float sums[3] = {0.f, 0.f, 0.f};
#pragma unroll
    for (int it = 0; it < NV; ++it) {
      const int vi = first + it * hop;
      if (vi < nvec) {
        float G[E], u[E], wv[E], t[E];
        unpack_raw<TY, E>(q[it], G);
        unpack_raw<TY, E>(b[it], u);
        load_f32<E>(p.w + vi * E, wv);
        load_tv<E>(p.v, p.scale, vi * E, t);
        if constexpr (GATE) {
          float o[E];
          unpack_raw<TY, E>(g[it], o);
#pragma unroll
          for (int j = 0; j < E; ++j) t[j] *= opened(o[j]);
        }
#pragma unroll
        for (int j = 0; j < E; ++j) {
          z[it][j] *= r2;                                // h from here on
          acc_w[it][j] += G[j] * z[it][j];
          G[j] *= wv[j];
          gz[it][j] += r2 * G[j];                        // p from here on
          const float tu = t[j] * u[j] * r1;
          sums[0] += G[j] * z[it][j];
          sums[1] += gz[it][j] * tu;
          sums[2] += z[it][j] * tu;
        }
      }
    }
    row_sums<WARPS>(sums, W, group, warp, lane, slots[phase]);
    const float m = sums[0] * inv_d * r2, nu = sums[1] - m * sums[2], k = nu * inv_d, rs = r1 * whole;      // dz = p - m h
    acc_s += nu;
#pragma unroll
    for (int it = 0; it < NV; ++it) {
      const int vi = first + it * hop;
      if (vi < nvec) {
        float u[E], t[E], o[E];
        unpack_raw<TY, E>(b[it], u);
        load_tv<E>(p.v, p.scale, vi * E, t);
#pragma unroll
        for (int j = 0; j < E; ++j) {
          gz[it][j] -= m * z[it][j];                     // dz from here on
          u[j] *= r1;
        }
        store_f32<E>(p.dx + r * p.dx_stride + vi * E, gz[it]);
        if constexpr (GATE) {
          float a[E];
          unpack_raw<TY, E>(g[it], a);
#pragma unroll
          for (int j = 0; j < E; ++j) {
            float slope;
            const float sig = opened(a[j], slope), n = gz[it][j] * t[j];
            o[j] = rs * (n * sig - u[j] * k);
            acc_c[it][j] += gz[it][j] * sig * u[j];
            a[j] = whole * (n * u[j] * slope);
          }
          store_16<TY, E>(dg + r * p.dg_stride + vi * E, a);
        } else {
#pragma unroll
          for (int j = 0; j < E; ++j) {
            o[j] = rs * (gz[it][j] * t[j] - u[j] * k);
            acc_c[it][j] += gz[it][j] * u[j];
          }
        }
        store_16<TY, E>(db + r * p.db_stride + vi * E, o);
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
        for (int j = 0; j < E; ++j) s_sum[group * p.d + vi * E + j] = set ? acc_c[it][j] : acc_w[it][j];
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
  if (lane == 0 && part == 0) s_sum[group] = acc_s;
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
  float t = 0.f;
  if (c < width)
    for (int p = threadIdx.y; p < nparts; p += 32) t += partial[(int64_t)p * width + c];
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

int check_shape(const char* who, int dtype, int d, int64_t rows) {
  if (dtype != ULM_F16 && dtype != ULM_BF16) return fail(ULM_ERR_ARG, "%s: branch, gate and y are fp16 or bf16", who);
  if (d <= 0 || d % 4 || rows < 0) return fail(ULM_ERR_ARG, "%s: need rows >= 0 and d a positive multiple of 4", who);
  if (d > kMaxRow) return fail(ULM_ERR_TOO_LARGE, "%s: rows of at most %d elements", who, kMaxRow);
  return ULM_OK;
}

// vectors of a lane
int fwd_nv(int nvec, int E) { const int most = E == 8 || nvec <= 1024 ? 4 : 8, need = ceil_div(nvec, 32); return need < most ? need : most; }
int bwd_nv(int d, int E) { return (d <= 2048 ? 8 : 16) / E; }
constexpr int kBwdElems = 32 * 16;                       // columns a warp of the backward has at most
static_assert(kMaxRow <= kBwdWideWarps * kBwdElems, "rows");
static_assert((kBwdWideWarps * kBwdElems + 6 * kBwdWideWarps) * sizeof(float) <= 48 * 1024, "shared memory");

constexpr int kBwdWarpsPerSm = 24, kMostBwdCtas = 3;
int64_t bwd_blocks(int64_t rows, const Split& s) {
  const int64_t want = (rows + s.groups - 1) / s.groups;
  int per_sm = kBwdWarpsPerSm / (s.W * s.groups);
  per_sm = per_sm < 1 ? 1 : per_sm > kMostBwdCtas ? kMostBwdCtas : per_sm;
  return want < per_sm * kNumSMs ? want : per_sm * kNumSMs;
}

template <typename TY, bool GATE>
int launch_fwd(FwdParams p, int E, cudaStream_t st, const char* who) {
  const int nvec = p.d / E, nv = fwd_nv(nvec, E);
  const Split s = split_rows(p.rows, nvec, nv, kFwdWarps);
  p.W = s.W;
  int64_t blocks = (p.rows + s.groups - 1) / s.groups;
  if (blocks > 64 * kNumSMs) blocks = 64 * kNumSMs;
  auto go = [&](auto kern) { return launch_dependent(who, kern, (unsigned)blocks, s.W * s.groups * 32, 0, st, p); };
  if (E == 8)
    return nv == 1 ? go(norm_add_norm_fwd_kernel<TY, 8, 1, GATE>) : nv == 2 ? go(norm_add_norm_fwd_kernel<TY, 8, 2, GATE>)
         : nv == 3 ? go(norm_add_norm_fwd_kernel<TY, 8, 3, GATE>) : go(norm_add_norm_fwd_kernel<TY, 8, 4, GATE>);
  return nv <= 2 ? go(norm_add_norm_fwd_kernel<TY, 4, 2, GATE>) : nv <= 4 ? go(norm_add_norm_fwd_kernel<TY, 4, 4, GATE>) : go(norm_add_norm_fwd_kernel<TY, 4, 8, GATE>);
}

template <typename TY, bool GATE>
int launch_bwd(BwdParams p, int E, int64_t* parts, cudaStream_t st, const char* who) {
  const int nvec = p.d / E, nv = bwd_nv(p.d, E);
  const Split s = split_rows(p.rows, nvec, nv, kBwdWarps);
  p.W = s.W;
  const int64_t blocks = bwd_blocks(p.rows, s);
  // a warp has at most kBwdElems columns of a row, so groups x d is at most that for every warp of the CTA (32 KB)
  const size_t smem = (size_t)s.groups * p.d * sizeof(float);
  *parts = blocks;
  auto go = [&](auto kern) { return launch_dependent(who, kern, (unsigned)blocks, s.W * s.groups * 32, smem, st, p); };
  const bool wide = s.W > kBwdWarps;
  if (E == 8)
    return nv == 1 ? go(norm_add_norm_bwd_kernel<TY, 8, 1, kBwdWarps, GATE>)
         : wide ? go(norm_add_norm_bwd_kernel<TY, 8, 2, kBwdWideWarps, GATE>) : go(norm_add_norm_bwd_kernel<TY, 8, 2, kBwdWarps, GATE>);
  return nv == 2 ? go(norm_add_norm_bwd_kernel<TY, 4, 2, kBwdWarps, GATE>)
       : wide ? go(norm_add_norm_bwd_kernel<TY, 4, 4, kBwdWideWarps, GATE>) : go(norm_add_norm_bwd_kernel<TY, 4, 4, kBwdWarps, GATE>);
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
  const int E = a->d % 8 == 0 && ok16(a->branch, a->branch_stride, 8) && ok16(a->gate, a->gate_stride, 8) && ok16(a->y, a->y_stride, 8) ? 8 : 4;
  const FwdParams p{a->x, a->branch, a->gate, a->v, a->w, {a->scale, a->scale_value, a->scale_channels}, a->x_out, a->y, a->rstd_branch, a->rstd,
                    a->x_stride, a->branch_stride, a->gate_stride, a->xout_stride, a->y_stride, a->rows, a->d, 1, a->eps};
  cudaStream_t st = (cudaStream_t)a->stream;
  auto go = [&](auto t) { return a->gate ? launch_fwd<decltype(t), true>(p, E, st, who) : launch_fwd<decltype(t), false>(p, E, st, who); };
  return a->dtype == ULM_F16 ? go(__half()) : go(__nv_bfloat16());
}

// one CTA a row, or as many as run at a time
extern "C" int64_t ulm_norm_add_norm_partial(int64_t rows, int32_t d) {
  const int64_t most = ulm::kMostBwdCtas * ulm::kNumSMs, n = rows < 1 ? 1 : rows < most ? rows : most;
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
                        ok16(a->d_branch, a->dbranch_stride, 8) && ok16(a->d_gate, a->dgate_stride, 8) ? 8 : 4;
  cudaStream_t st = (cudaStream_t)a->stream;
  const Scale scale{a->scale, a->scale_value, a->scale_channels};
  int64_t blocks = 0;
  if (a->rows > 0) {
    const BwdParams p{a->x, a->branch, a->gate, a->v, a->w, scale, a->dy, a->g_add, a->rstd_branch, a->rstd, a->dx, a->d_branch, a->d_gate, a->partial,
                      a->x_stride, a->branch_stride, a->gate_stride, a->dy_stride, a->gadd_stride, a->dx_stride, a->dbranch_stride, a->dgate_stride, a->rows, a->d, 1};
    auto go = [&](auto t) { return a->gate ? launch_bwd<decltype(t), true>(p, E, &blocks, st, who) : launch_bwd<decltype(t), false>(p, E, &blocks, st, who); };
    if (int rc = a->dtype == ULM_F16 ? go(__half()) : go(__nv_bfloat16())) return rc;
  }
  return launch_dependent(who, norm_add_norm_finish_kernel, (2 * a->d + 1 + 31) / 32, dim3(32, 32), 0, st, a->partial, a->v, scale, a->dw, a->dv, a->dscale, (int)blocks, a->d);
}
