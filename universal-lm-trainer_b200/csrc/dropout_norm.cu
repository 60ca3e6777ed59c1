// Residual add with dropout on the branch, and the RMS norm that follows it (sm_100a): one pass each way, no stored mask.
//
//   fwd  z = x + drop(b);  r = rsqrt(mean(z^2) + eps);  y = w z r        x, z fp32; b, y 16-bit
//   bwd  dz = r (w dy - z r mean(w dy z r)) + gz;  dx = dz;  db = drop(dz);  dw = sum over rows of dy z r
//
// drop and its mask: philox.cuh, over the branch's elements.  Sums and statistics are fp32; y, db are rounded once.
//
// What bounds it: HBM, 12 bytes an element forward and 16 backward: 32768 x 768 fp16 45.5 us (6.6 TB/s) and 67.6 us (6.0 TB/s) and
// 3 us for dw's column sums.  A row belongs to W warps of a CTA (W = 1 up to 1024
// elements forward) and is held in registers between its two uses; a lane owns vectors of E elements: eight where all
// rows are whole 16-byte vectors of the 16-bit tensors, so that a vector is exactly one group of the mask, else four
// (two lanes then form the same group, twice the generator's work: 20000 x 772 42 and 69 us, x 768 31 and 44).
// From 2048 columns on the backward is at 4.6-5.0 TB/s (1024: 5.2): a row's loads, barrier and stores follow one another in its group.
// dw: per-lane sums over a CTA's rows, added up over the CTA's groups in shared memory, one partial row per CTA, column
// sums in a fixed order: no atomics.
#include "col_sum.cuh"
#include "norm_rows.cuh"
#include "philox.cuh"

namespace ulm {
namespace {

constexpr int kMaxRow = 8192;
constexpr int kFwdWarps = 8, kBwdWarps = 12, kBwdWideWarps = 16;

struct FwdParams {
  const float* x; const void* branch; const float* w; float* x_out; void* y; float* rstd;
  int64_t x_stride, branch_stride, xout_stride, y_stride, rows;
  int d, W; float eps;
};

template <typename TY, int E, int NV>
__global__ void __launch_bounds__(kFwdWarps * 32, NV * E <= 24 ? 4 : 3)
add_dropout_norm_fwd_kernel(const FwdParams p, const __grid_constant__ DropMask mask) {
  __shared__ float slots[2][kFwdWarps];
  grid_dependents_go();
  grid_dependency_wait();
  const TY* br = static_cast<const TY*>(p.branch);
  TY* y = static_cast<TY*>(p.y);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, W = p.W;
  const int group = warp / W, part = warp - group * W, groups = (int)(blockDim.x >> 5) / W;
  const int nvec = p.d / E, first = part * 32 + lane, hop = W * 32;
  const float inv_d = 1.f / (float)p.d;
  int phase = 0;
  for (int64_t r = (int64_t)blockIdx.x * groups + group; r < p.rows; r += (int64_t)gridDim.x * groups, phase ^= 1) {
    float v[NV][E];
    Raw<E> b[NV];
#pragma unroll
    for (int it = 0; it < NV; ++it) {                    // the whole row is requested before any of it is used
      const int vi = first + it * hop;
      if (vi < nvec) {
        load_f32<E>(p.x + r * p.x_stride + vi * E, v[it]);
        b[it] = load_raw<TY, E>(br + r * p.branch_stride + vi * E);
      }
    }
    float ss = 0.f;
#pragma unroll
    for (int it = 0; it < NV; ++it) {
      const int vi = first + it * hop;
      if (vi < nvec) {
        const Keep<E> keep = keep_of<E>(mask, (uint64_t)r * nvec + vi);
        float f[E];
        unpack_raw<TY, E>(b[it], f);
#pragma unroll
        for (int j = 0; j < E; ++j) {
          v[it][j] += dropped(mask, keep(j), f[j]);
          ss += v[it][j] * v[it][j];
        }
        store_f32<E>(p.x_out + r * p.xout_stride + vi * E, v[it]);
      }
    }
    const float inv = rsqrtf(row_sum(ss, W, group, warp, lane, slots[phase]) * inv_d + p.eps);
    if (p.rstd && first == 0) p.rstd[r] = inv;
#pragma unroll
    for (int it = 0; it < NV; ++it) {
      const int vi = first + it * hop;
      if (vi < nvec) {
        float wv[E], o[E];
        load_f32<E>(p.w + vi * E, wv);
#pragma unroll
        for (int j = 0; j < E; ++j) o[j] = v[it][j] * inv * wv[j];
        store_16<TY, E>(y + r * p.y_stride + vi * E, o);
      }
    }
  }
}

struct BwdParams {
  const float* x; const float* w; const void* dy; const float* rstd; const float* g_add;
  float* dx; void* d_branch; float* partial;
  int64_t x_stride, dy_stride, gadd_stride, dx_stride, dbranch_stride, rows;
  int d, W;
};

template <typename TY, int E, int NV, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, WARPS == kBwdWideWarps ? 1 : 2)
add_dropout_norm_bwd_kernel(const BwdParams p, const __grid_constant__ DropMask mask) {
  extern __shared__ float s_dw[];                        // [groups][d]
  __shared__ float slots[2][WARPS];
  grid_dependents_go();
  grid_dependency_wait();
  const TY* dy = static_cast<const TY*>(p.dy);
  TY* db = static_cast<TY*>(p.d_branch);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, W = p.W;
  const int group = warp / W, part = warp - group * W, groups = (int)(blockDim.x >> 5) / W;
  const int nvec = p.d / E, first = part * 32 + lane, hop = W * 32;
  const float inv_d = 1.f / (float)p.d;
  float acc[NV][E];
#pragma unroll
  for (int it = 0; it < NV; ++it)
#pragma unroll
    for (int j = 0; j < E; ++j) acc[it][j] = 0.f;
  int phase = 0;
  for (int64_t r = (int64_t)blockIdx.x * groups + group; r < p.rows; r += (int64_t)gridDim.x * groups, phase ^= 1) {
    float z[NV][E], ga[NV][E];
    Raw<E> gr[NV];
#pragma unroll
    for (int it = 0; it < NV; ++it) {
      const int vi = first + it * hop;
      if (vi < nvec) {
        load_f32<E>(p.x + r * p.x_stride + vi * E, z[it]);
        gr[it] = load_raw<TY, E>(dy + r * p.dy_stride + vi * E);
        if (p.g_add) {
          load_f32<E>(p.g_add + r * p.gadd_stride + vi * E, ga[it]);
        } else {
#pragma unroll
          for (int j = 0; j < E; ++j) ga[it][j] = 0.f;
        }
      }
    }
    const float inv = p.rstd[r];
    float dot = 0.f;
#pragma unroll
    for (int it = 0; it < NV; ++it) {
      const int vi = first + it * hop;
      if (vi < nvec) {
        float g[E], wv[E];
        unpack_raw<TY, E>(gr[it], g);
        load_f32<E>(p.w + vi * E, wv);
#pragma unroll
        for (int j = 0; j < E; ++j) {
          z[it][j] *= inv;                               // the normalised row from here on
          acc[it][j] += g[j] * z[it][j];
          dot += g[j] * wv[j] * z[it][j];
        }
      }
    }
    const float dm = row_sum(dot, W, group, warp, lane, slots[phase]) * inv_d;
#pragma unroll
    for (int it = 0; it < NV; ++it) {
      const int vi = first + it * hop;
      if (vi < nvec) {
        float g[E], wv[E], o[E];
        unpack_raw<TY, E>(gr[it], g);
        load_f32<E>(p.w + vi * E, wv);
#pragma unroll
        for (int j = 0; j < E; ++j) o[j] = inv * (g[j] * wv[j] - z[it][j] * dm) + ga[it][j];
        store_f32<E>(p.dx + r * p.dx_stride + vi * E, o);
        const Keep<E> keep = keep_of<E>(mask, (uint64_t)r * nvec + vi);
#pragma unroll
        for (int j = 0; j < E; ++j) o[j] = dropped(mask, keep(j), o[j]);
        store_16<TY, E>(db + r * p.dbranch_stride + vi * E, o);
      }
    }
  }
#pragma unroll
  for (int it = 0; it < NV; ++it) {
    const int vi = first + it * hop;
    if (vi < nvec) {
#pragma unroll
      for (int j = 0; j < E; ++j) s_dw[group * p.d + vi * E + j] = acc[it][j];
    }
  }
  __syncthreads();
  for (int c = threadIdx.x; c < p.d; c += (int)blockDim.x) {
    float t = 0.f;
    for (int g = 0; g < groups; ++g) t += s_dw[g * p.d + c];
    p.partial[(int64_t)blockIdx.x * p.d + c] = t;
  }
}

// Elements a lane holds.  Forward 32 with vectors of eight (one warp a row up to 1024), with vectors of four 16 up to rows of
// 4096 and 32 beyond.  Backward, where a
// row's z, dy, g and dw are alive together, 8 up to rows of 2048 and 16 beyond: us with 8 / 16, bf16,
// 4096 x 2048 28.5 / 29.3, x 2560 39.2 / 36.3, x 4096 77.6 / 54.5 (4.7, 4.6 and 4.9 TB/s
// with what is taken).
int fwd_nv(int nvec, int E) { const int most = E == 8 || nvec <= 1024 ? 4 : 8, need = ceil_div(nvec, 32); return need < most ? need : most; }
int bwd_nv(int d, int E) { return (d <= 2048 ? 8 : 16) / E; }
// columns of a row that a warp of the backward has at most; a whole row fits the widest CTA, and a CTA's dw the 48 KB that need no opt-in
constexpr int kBwdElems = 32 * 16;
static_assert(kMaxRow <= kBwdWideWarps * kBwdElems, "rows");
static_assert((kBwdWideWarps * kBwdElems + 2 * kBwdWideWarps) * sizeof(float) <= 48 * 1024, "shared memory");

// A CTA of the backward per `groups` rows, 24 warps per SM at most (their registers fill it): each leaves one partial row
constexpr int kBwdWarpsPerSm = 24, kMostBwdCtas = 3;
int64_t bwd_blocks(int64_t rows, const Split& s) {
  const int64_t want = (rows + s.groups - 1) / s.groups;
  int per_sm = kBwdWarpsPerSm / (s.W * s.groups);
  per_sm = per_sm < 1 ? 1 : per_sm > kMostBwdCtas ? kMostBwdCtas : per_sm;
  return want < per_sm * kNumSMs ? want : per_sm * kNumSMs;
}

int check_shape(const char* who, int x_dtype, int w_dtype, int kind, int d, int64_t rows, double p) {
  if (x_dtype != ULM_F32 || w_dtype != ULM_F32 || (kind != ULM_Y_F16 && kind != ULM_Y_BF16))
    return fail(ULM_ERR_ARG, "%s: takes an fp32 x and weight with a 16-bit branch and y", who);
  if (d <= 0 || d % 4 || rows < 0) return fail(ULM_ERR_ARG, "%s: need rows >= 0 and d a positive multiple of 4", who);
  if (d > kMaxRow) return fail(ULM_ERR_TOO_LARGE, "%s: rows of at most %d elements", who, kMaxRow);
  if (!drop_p_ok(p)) return fail(ULM_ERR_ARG, "%s: p must lie between 0 and 1", who);
  return ULM_OK;
}

template <typename TY>
int launch_fwd(FwdParams p, int E, const DropMask& mask, cudaStream_t st, const char* who) {
  const int nvec = p.d / E, nv = fwd_nv(nvec, E);
  const Split s = split_rows(p.rows, nvec, nv, kFwdWarps);
  p.W = s.W;
  int64_t blocks = (p.rows + s.groups - 1) / s.groups;
  if (blocks > 64 * kNumSMs) blocks = 64 * kNumSMs;
  const int threads = s.W * s.groups * 32;
  auto go = [&](auto kern) { return launch_dependent(who, kern, (unsigned)blocks, threads, 0, st, p, mask); };
  if (E == 8)
    return nv == 1 ? go(add_dropout_norm_fwd_kernel<TY, 8, 1>) : nv == 2 ? go(add_dropout_norm_fwd_kernel<TY, 8, 2>)
         : nv == 3 ? go(add_dropout_norm_fwd_kernel<TY, 8, 3>) : go(add_dropout_norm_fwd_kernel<TY, 8, 4>);
  return nv <= 2 ? go(add_dropout_norm_fwd_kernel<TY, 4, 2>) : nv <= 4 ? go(add_dropout_norm_fwd_kernel<TY, 4, 4>) : go(add_dropout_norm_fwd_kernel<TY, 4, 8>);
}

template <typename TY>
int launch_bwd(BwdParams p, int E, const DropMask& mask, int64_t* parts, cudaStream_t st, const char* who) {
  const int nvec = p.d / E, nv = bwd_nv(p.d, E);
  const Split s = split_rows(p.rows, nvec, nv, kBwdWarps);
  p.W = s.W;
  const int64_t blocks = bwd_blocks(p.rows, s);
  const int threads = s.W * s.groups * 32;
  // a warp has at most kBwdElems columns of a row, so groups x d is at most that for every warp of the CTA (32 KB)
  const size_t smem = (size_t)s.groups * p.d * sizeof(float);
  *parts = blocks;
  auto go = [&](auto kern) { return launch_dependent(who, kern, (unsigned)blocks, threads, smem, st, p, mask); };
  const bool wide = s.W > kBwdWarps;
  if (E == 8)
    return nv == 1 ? go(add_dropout_norm_bwd_kernel<TY, 8, 1, kBwdWarps>)
         : wide ? go(add_dropout_norm_bwd_kernel<TY, 8, 2, kBwdWideWarps>) : go(add_dropout_norm_bwd_kernel<TY, 8, 2, kBwdWarps>);
  return nv == 2 ? go(add_dropout_norm_bwd_kernel<TY, 4, 2, kBwdWarps>)
       : wide ? go(add_dropout_norm_bwd_kernel<TY, 4, 4, kBwdWideWarps>) : go(add_dropout_norm_bwd_kernel<TY, 4, 4, kBwdWarps>);
}

}  // namespace
}  // namespace ulm

extern "C" int ulm_add_dropout_norm_fwd(const ulm_rmsnorm_fwd_args* a, double p, uint64_t seed) {
  using namespace ulm;
  const char* who = "ulm_add_dropout_norm_fwd";
  if (!a) return fail(ULM_ERR_ARG, "%s: null args", who);
  if (int rc = check_shape(who, a->x_dtype, a->w_dtype, a->y_kind, a->d, a->rows, p)) return rc;
  if (a->rows == 0) return ULM_OK;
  if (!a->x || !a->branch || !a->w || !a->x_out || !a->y) return fail(ULM_ERR_ARG, "%s: null tensor", who);
  if (!ok32(a->x, a->x_stride) || !ok32(a->x_out, a->xout_stride) || !ok32(a->w, 0) || !ok16(a->branch, a->branch_stride, 4) || !ok16(a->y, a->y_stride, 4))
    return fail(ULM_ERR_ARG, "%s: fp32 rows must be 16-byte aligned, 16-bit rows 8-byte aligned", who);
  const int E = a->d % 8 == 0 && ok16(a->branch, a->branch_stride, 8) && ok16(a->y, a->y_stride, 8) ? 8 : 4;
  const FwdParams q{(const float*)a->x, a->branch, (const float*)a->w, (float*)a->x_out, a->y, a->rstd,
                    a->x_stride, a->branch_stride, a->xout_stride, a->y_stride, a->rows, a->d, 1, a->eps};
  const DropMask mask = make_drop_mask(p, seed);
  cudaStream_t st = (cudaStream_t)a->stream;
  return a->y_kind == ULM_Y_F16 ? launch_fwd<__half>(q, E, mask, st, who) : launch_fwd<__nv_bfloat16>(q, E, mask, st, who);
}

// one CTA a row, or as many as run at a time
extern "C" int64_t ulm_add_dropout_norm_partial_rows(int64_t rows) {
  const int64_t most = ulm::kMostBwdCtas * ulm::kNumSMs;
  return rows < 1 ? 1 : rows < most ? rows : most;
}

extern "C" int ulm_add_dropout_norm_bwd(const ulm_rmsnorm_bwd_args* a, double p, uint64_t seed) {
  using namespace ulm;
  const char* who = "ulm_add_dropout_norm_bwd";
  if (!a) return fail(ULM_ERR_ARG, "%s: null args", who);
  if (int rc = check_shape(who, a->x_dtype, a->w_dtype, a->dy_kind, a->d, a->rows, p)) return rc;
  if (!a->dw || (a->rows > 0 && (!a->x || !a->w || !a->dy || !a->rstd || !a->dx || !a->d_branch || !a->partial)))
    return fail(ULM_ERR_ARG, "%s: null tensor", who);
  if (a->rows > 0 && (!ok32(a->x, a->x_stride) || !ok32(a->dx, a->dx_stride) || !ok32(a->g_add, a->gadd_stride) || !ok32(a->w, 0) ||
                      !ok16(a->dy, a->dy_stride, 4) || !ok16(a->d_branch, a->dbranch_stride, 4)))
    return fail(ULM_ERR_ARG, "%s: fp32 rows must be 16-byte aligned, 16-bit rows 8-byte aligned", who);
  const int E = a->d % 8 == 0 && ok16(a->dy, a->dy_stride, 8) && ok16(a->d_branch, a->dbranch_stride, 8) ? 8 : 4;
  cudaStream_t st = (cudaStream_t)a->stream;
  int64_t blocks = 0;
  if (a->rows > 0) {
    const BwdParams q{(const float*)a->x, (const float*)a->w, a->dy, a->rstd, (const float*)a->g_add, (float*)a->dx, a->d_branch, a->partial,
                      a->x_stride, a->dy_stride, a->gadd_stride, a->dx_stride, a->dbranch_stride, a->rows, a->d, 1};
    const DropMask mask = make_drop_mask(p, seed);
    if (int rc = a->dy_kind == ULM_Y_F16 ? launch_bwd<__half>(q, E, mask, &blocks, st, who) : launch_bwd<__nv_bfloat16>(q, E, mask, &blocks, st, who)) return rc;
  }
  return launch_dependent(who, col_sum_kernel, (a->d + 31) / 32, dim3(32, 32), 0, st, a->partial, a->dw, (int)blocks, a->d);
}
