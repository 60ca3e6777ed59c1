// Dropout whose mask is computed and never stored (sm_100a), alone and inside the feed-forward gate.
//
//   dropout        y = keep ? c x : 0                     dx = keep ? c dy : 0: the same kernel on dy
//   gated dropout  y = keep ? c a s b : 0, s = sigmoid(a)
//                  g = keep ? c dy : 0;  da = g b s (1 + a (1 - s)),  db = g a s
//
// The mask is that of philox.cuh over y's elements, so the backward forms it again instead of reading it.  Values are fp32
// from the load to the one rounding of the store: what the gate rounds to 16 bits between its steps when it runs without
// dropout (the roundings of separate eager kernels) is kept in 32 here.
// What bounds them: HBM.  Every tensor is read or written once; the generator's instructions fit beside that (philox.cuh).
// A grid that covers the tensor once, 16-byte vectors, every load of a thread before its first use, as the gate without
// dropout has it.
#include "gate_math.cuh"
#include "philox.cuh"

namespace ulm {
namespace {

constexpr int kThreads = 256;
// 16-byte vectors a thread takes of each tensor; their masks are formed while the loads are on their way, without which the
// gate's forward took 72 us instead of 64 (32768 x 2048 bf16: 6.3 TB/s) and its backward 101 instead of 95 (7.1 TB/s).
// One / two / four vectors: dropout of 32768 x 768 in bf16 19.4 / 17.4 / 16.4 us (6.1 TB/s), in fp32 35.7 / 30.6 / 31.5 (6.6
// TB/s), the gate's forward 82 / 64 / 64, its backward 107 / 95 / -.  The gate in fp32, 8192 x 2048: 31.7 us (6.3 TB/s) and 47.6 (7.0).
template <typename T> constexpr int kVecsDrop = sizeof(T) == 4 ? 2 : 4;
constexpr int kVecsGate = 2;

template <typename T>
__global__ void __launch_bounds__(kThreads)
dropout_kernel(const T* x, T* y, int64_t nvec, int64_t n, const __grid_constant__ DropMask mask) {
  constexpr int N = VecN<T>::N, K = kVecsDrop<T>;
  const int64_t v0 = (int64_t)blockIdx.x * (kThreads * K) + threadIdx.x;
  grid_dependents_go();
  grid_dependency_wait();
  uint4 rx[K];
#pragma unroll
  for (int k = 0; k < K; ++k)
    if (v0 + k * kThreads < nvec) rx[k] = *(reinterpret_cast<const uint4*>(x) + v0 + k * kThreads);
  Keep<N> keep[K];                                       // while the loads are on their way
#pragma unroll
  for (int k = 0; k < K; ++k) keep[k] = keep_of<N>(mask, (uint64_t)(v0 + k * kThreads));
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int64_t v = v0 + k * kThreads;
    if (v < nvec) {
      float f[N];
      unpack<T>(rx[k], f);
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = dropped(mask, keep[k](i), f[i]);
      reinterpret_cast<uint4*>(y)[v] = pack<T>(f);
    }
  }
  if (blockIdx.x == 0 && threadIdx.x < (int)(n - nvec * N)) {            // a tail shorter than a vector
    const int64_t i = nvec * N + threadIdx.x;
    y[i] = Cvt<T>::from_f(dropped(mask, keep_one(mask, (uint64_t)i), Cvt<T>::to_f(x[i])));
  }
}

template <typename T>
__device__ __forceinline__ float gate_fwd_one(const DropMask& m, bool stays, float a, float b) {
  float s, u;
  sigmoid_silu<T>(a, s, u);
  return dropped(m, stays, u * b);
}
template <typename T>
__device__ __forceinline__ void gate_bwd_one(const DropMask& m, bool stays, float a, float b, float dy, float& da, float& db) {
  float s, u;
  sigmoid_silu<T>(a, s, u);
  da = dropped(m, stays, dy * b * (s * (1.f + a * (1.f - s))));
  db = dropped(m, stays, dy * u);
}

template <typename T, bool ROWS>
__global__ void __launch_bounds__(kThreads)
gate_dropout_fwd_kernel(const T* a, const T* b, T* y, int64_t nvec, int64_t n, const Rows rw,
                        const __grid_constant__ DropMask mask) {
  constexpr int N = VecN<T>::N, K = kVecsGate;
  const int64_t v0 = (int64_t)blockIdx.x * (kThreads * K) + threadIdx.x;
  grid_dependents_go();
  grid_dependency_wait();
  uint4 ra[K], rb[K];
#pragma unroll
  for (int k = 0; k < K; ++k)
    if (v0 + k * kThreads < nvec) {
      const int64_t o = operand_vec<ROWS>(v0 + k * kThreads, rw);
      ra[k] = *(reinterpret_cast<const uint4*>(a) + o);
      rb[k] = *(reinterpret_cast<const uint4*>(b) + o);
    }
  Keep<N> keep[K];                                       // while the loads are on their way
#pragma unroll
  for (int k = 0; k < K; ++k) keep[k] = keep_of<N>(mask, (uint64_t)(v0 + k * kThreads));
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int64_t v = v0 + k * kThreads;
    if (v < nvec) {
      float fa[N], fb[N], fy[N];
      unpack<T>(ra[k], fa);
      unpack<T>(rb[k], fb);
#pragma unroll
      for (int i = 0; i < N; ++i) fy[i] = gate_fwd_one<T>(mask, keep[k](i), fa[i], fb[i]);
      reinterpret_cast<uint4*>(y)[v] = pack<T>(fy);
    }
  }
  if (blockIdx.x == 0 && threadIdx.x < (int)(n - nvec * N)) {
    const int64_t i = nvec * N + threadIdx.x;
    y[i] = Cvt<T>::from_f(gate_fwd_one<T>(mask, keep_one(mask, (uint64_t)i), Cvt<T>::to_f(a[i]), Cvt<T>::to_f(b[i])));
  }
}

template <typename T, bool ROWS>
__global__ void __launch_bounds__(kThreads)
gate_dropout_bwd_kernel(const T* a, const T* b, const T* dy, T* da, T* db,
                        int64_t nvec, int64_t n, const Rows rw, const __grid_constant__ DropMask mask) {
  constexpr int N = VecN<T>::N, K = kVecsGate;
  const int64_t v0 = (int64_t)blockIdx.x * (kThreads * K) + threadIdx.x;
  grid_dependents_go();
  grid_dependency_wait();
  uint4 ra[K], rb[K], rg[K];
#pragma unroll
  for (int k = 0; k < K; ++k)
    if (v0 + k * kThreads < nvec) {
      const int64_t o = operand_vec<ROWS>(v0 + k * kThreads, rw);
      ra[k] = *(reinterpret_cast<const uint4*>(a) + o);
      rb[k] = *(reinterpret_cast<const uint4*>(b) + o);
      rg[k] = *(reinterpret_cast<const uint4*>(dy) + v0 + k * kThreads);
    }
  Keep<N> keep[K];                                       // while the loads are on their way
#pragma unroll
  for (int k = 0; k < K; ++k) keep[k] = keep_of<N>(mask, (uint64_t)(v0 + k * kThreads));
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int64_t v = v0 + k * kThreads;
    if (v < nvec) {
      float fa[N], fb[N], fg[N], oa[N], ob[N];
      unpack<T>(ra[k], fa);
      unpack<T>(rb[k], fb);
      unpack<T>(rg[k], fg);
#pragma unroll
      for (int i = 0; i < N; ++i) gate_bwd_one<T>(mask, keep[k](i), fa[i], fb[i], fg[i], oa[i], ob[i]);
      const int64_t o = operand_vec<ROWS>(v, rw);
      reinterpret_cast<uint4*>(da)[o] = pack<T>(oa);
      reinterpret_cast<uint4*>(db)[o] = pack<T>(ob);
    }
  }
  if (blockIdx.x == 0 && threadIdx.x < (int)(n - nvec * N)) {
    const int64_t i = nvec * N + threadIdx.x;
    float oa, ob;
    gate_bwd_one<T>(mask, keep_one(mask, (uint64_t)i), Cvt<T>::to_f(a[i]), Cvt<T>::to_f(b[i]), Cvt<T>::to_f(dy[i]), oa, ob);
    da[i] = Cvt<T>::from_f(oa);
    db[i] = Cvt<T>::from_f(ob);
  }
}

unsigned grid_for(int64_t nvec, int per_thread) {
  const int64_t per = (int64_t)kThreads * per_thread, blocks = (nvec + per - 1) / per;
  return (unsigned)(blocks < 1 ? 1 : blocks);
}
bool aligned16(const void* p) { return p && !(reinterpret_cast<uintptr_t>(p) & 15); }

int check_drop(int dtype, int64_t n, double p, const char* who) {
  if (dtype != ULM_F16 && dtype != ULM_BF16 && dtype != ULM_F32) return fail(ULM_ERR_ARG, "%s: bad dtype", who);
  if (n < 0) return fail(ULM_ERR_ARG, "%s: negative size", who);
  if (!drop_p_ok(p)) return fail(ULM_ERR_ARG, "%s: p must lie between 0 and 1", who);
  if (n / 4 / kThreads > 0x7ffffff0LL) return fail(ULM_ERR_TOO_LARGE, "%s: too many elements", who);
  return ULM_OK;
}

template <typename T>
int gate_launch(const ulm_swiglu_args* p, bool bwd, int64_t d, int64_t stride, const DropMask& mask, const char* who) {
  cudaStream_t st = (cudaStream_t)p->stream;
  const int64_t nvec = p->n / VecN<T>::N;
  const Rows rw{(uint32_t)(d / VecN<T>::N), stride / VecN<T>::N};
  const T *a = (const T*)p->a, *b = (const T*)p->b, *dy = (const T*)p->dy;
  T *y = (T*)p->y, *da = (T*)p->da, *db = (T*)p->db;
  const unsigned grid = grid_for(nvec, kVecsGate);
  if (bwd) return launch_dependent(who, d ? gate_dropout_bwd_kernel<T, true> : gate_dropout_bwd_kernel<T, false>, grid, kThreads, 0, st, a, b, dy, da, db, nvec, p->n, rw, mask);
  return launch_dependent(who, d ? gate_dropout_fwd_kernel<T, true> : gate_dropout_fwd_kernel<T, false>, grid, kThreads, 0, st, a, b, y, nvec, p->n, rw, mask);
}

}  // namespace
}  // namespace ulm

extern "C" int ulm_dropout(const void* x, void* y, int64_t n, int32_t dtype, double p, uint64_t seed, void* stream) {
  using namespace ulm;
  const char* who = "ulm_dropout";
  if (int rc = check_drop(dtype, n, p, who)) return rc;
  if (n == 0) return ULM_OK;
  if (!aligned16(x) || !aligned16(y)) return fail(ULM_ERR_ARG, "%s: x and y must be non-null and 16-byte aligned", who);
  const DropMask mask = make_drop_mask(p, seed);
  cudaStream_t st = (cudaStream_t)stream;
  auto go = [&](auto t) {
    using T = decltype(t);
    const int64_t nvec = n / VecN<T>::N;
    return launch_dependent(who, dropout_kernel<T>, grid_for(nvec, kVecsDrop<T>), kThreads, 0, st, (const T*)x, (T*)y, nvec, n, mask);
  };
  return dtype == ULM_F16 ? go(__half()) : dtype == ULM_BF16 ? go(__nv_bfloat16()) : go(float());
}

extern "C" int ulm_swiglu_dropout(const ulm_swiglu_args* a, int32_t backward, int64_t d, int64_t row_stride, double p, uint64_t seed) {
  using namespace ulm;
  const char* who = "ulm_swiglu_dropout";
  if (!a) return fail(ULM_ERR_ARG, "%s: null args", who);
  if (int rc = check_drop(a->dtype, a->n, p, who)) return rc;
  if (d) {
    const int64_t vec = a->dtype == ULM_F32 ? 4 : 8;
    if (d < 0 || d % vec || row_stride % vec || row_stride < d || a->n % d) return fail(ULM_ERR_ARG, "%s: rows and their stride must be whole 16-byte vectors", who);
    if (a->n / vec > 0xffffffffLL) return fail(ULM_ERR_TOO_LARGE, "%s: too many elements", who);
  }
  if (a->n == 0) return ULM_OK;
  if (!aligned16(a->a) || !aligned16(a->b) || (backward ? !aligned16(a->dy) || !aligned16(a->da) || !aligned16(a->db) : !aligned16(a->y)))
    return fail(ULM_ERR_ARG, "%s: %s must be non-null and 16-byte aligned", who, backward ? "a, b, dy, da, db" : "a, b, y");
  const DropMask mask = make_drop_mask(p, seed);
  if (a->dtype == ULM_F16) return gate_launch<__half>(a, backward, d, row_stride, mask, who);
  if (a->dtype == ULM_BF16) return gate_launch<__nv_bfloat16>(a, backward, d, row_stride, mask, who);
  return gate_launch<float>(a, backward, d, row_stride, mask, who);
}
