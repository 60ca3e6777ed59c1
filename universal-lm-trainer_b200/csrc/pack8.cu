// Activations kept in 8 bits between forward and backward (sm_100a): a tensor by itself, and the operands of the feed-forward gate.
//
//   pack    codes and exponents of x (pack8.cuh);  unpack: x~
//   gate    y = keep ? c a s b : 0, s = sigmoid(a), and a, b in 8 bits
//           backward, of a~ and b~ alone: g = keep ? c dy : 0;  da = g b~ s (1 + a~ (1 - s)),  db = g a~ s;  y~ = keep ? c a~ s b~ : 0 again, which the
//           product behind the gate needs for its weight's gradient and which therefore is not kept either
//
// keep: the mask of philox.cuh over y's elements, or none.  Blocks go by an element's row-major index, whatever the rows.
//
// What bounds them: HBM.  The gate moves 8 1/16 bytes an element forward and back (10 1/16 with y~), where 16-bit operands would be 6 and 10
// (12 with the y they would keep); a step keeps 2 1/16 of its 6 bytes an element.
// A grid that covers the tensor once, 16-byte vectors, every load of a thread before its first use; the lanes of a block of
// 32 elements exchange its largest magnitude.
#include "pack8.cuh"
#include "philox.cuh"

namespace ulm {
namespace {

constexpr int kThreads = 256;
// 16-byte vectors of the operands a thread takes.  us at 32768 x 2048 bf16 (bytes moved at the copy rate: pack 31, the gate 83 each way), 1 / 2 / 4: pack
// 68 / 36 / 30, unpack 68 / 31 / 32, the gate's forward 92 / 85 / 81; its backward in rows of a projection 79.5 / 81 / 85 (fp16 79 / 90 / 85), with
// dropout, whose masks are formed while the loads are on their way, 124 / 111 / 119, in fp32 (8192 x 2048) 46 / 41 / 43.
constexpr int kVecsPack = 4, kVecsFwd = 4;
template <typename T, bool DROP> constexpr int kVecsBwd = sizeof(T) == 4 || DROP ? 2 : 1;

template <typename T>
__global__ void __launch_bounds__(kThreads)
pack8_kernel(const T* x, int8_t* codes, uint8_t* exps, int64_t nvec, int64_t n) {
  constexpr int N = VecN<T>::N, K = kVecsPack, S = kBlock8 / N;
  const int64_t v0 = (int64_t)blockIdx.x * (kThreads * K) + threadIdx.x;
  grid_dependents_go();
  grid_dependency_wait();
  uint4 r[K];
#pragma unroll
  for (int k = 0; k < K; ++k) r[k] = v0 + k * kThreads < nvec ? *(reinterpret_cast<const uint4*>(x) + v0 + k * kThreads) : make_uint4(0, 0, 0, 0);
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int64_t v = v0 + k * kThreads;
    const uint32_t most = block_magnitude<T>(magnitude<T>(r[k])), byte = exponent_byte(most);
    if (v < nvec) {
      float2 f[N / 2];
      unpack_pairs<T>(r[k], f);
      store_codes<T>(codes, v, f, per_step(byte), rounds_past(most));
      if (threadIdx.x % S == 0) exps[v / S] = (uint8_t)byte;
    }
  }
  if (blockIdx.x == 0 && threadIdx.x < 32 && nvec * N < n) {
    const int64_t i = nvec * N + threadIdx.x;
    const float f = i < n ? Cvt<T>::to_f(x[i]) : 0.f;
    const uint32_t byte = tail_exponent(f);
    if (i < n) codes[i] = tail_code(f, byte);
    if (threadIdx.x == 0) exps[nvec / S] = (uint8_t)byte;
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
unpack8_kernel(const int8_t* codes, const uint8_t* exps, T* x, int64_t nvec, int64_t n) {
  constexpr int N = VecN<T>::N, K = kVecsPack, S = kBlock8 / N;
  const int64_t v0 = (int64_t)blockIdx.x * (kThreads * K) + threadIdx.x;
  grid_dependents_go();
  grid_dependency_wait();
  Codes<T> c[K];
  uint32_t byte[K];
#pragma unroll
  for (int k = 0; k < K; ++k)
    if (v0 + k * kThreads < nvec) {
      c[k] = load_codes<T>(codes, v0 + k * kThreads);
      byte[k] = exps[(v0 + k * kThreads) / S];
    }
#pragma unroll
  for (int k = 0; k < K; ++k)
    if (v0 + k * kThreads < nvec) {
      float2 f[N / 2];
      values_of<T>(c[k], byte[k], f);
      reinterpret_cast<uint4*>(x)[v0 + k * kThreads] = pack_pairs<T>(f);
    }
  if (blockIdx.x == 0 && threadIdx.x < (int)(n - nvec * N)) {
    const int64_t i = nvec * N + threadIdx.x;
    x[i] = Cvt<T>::from_f(tail_value(codes[i], exps[nvec / S]));
  }
}

// sigmoid_silu of a pair; 16-bit tensors: the same operations, two at a time
template <typename T>
__device__ __forceinline__ void sigmoid_silu2(float2 a, float2& s, float2& u) {
  if constexpr (sizeof(T) == 4) {
    sigmoid_silu<T>(a.x, s.x, u.x);
    sigmoid_silu<T>(a.y, s.y, u.y);
  } else {
    const float2 t = mul2(a, both(-1.4426950408889634f));
    float2 e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(t.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(t.y));
    const float2 d = add2(both(1.f), e);
    asm("rcp.approx.f32 %0, %1;" : "=f"(s.x) : "f"(d.x));
    asm("rcp.approx.f32 %0, %1;" : "=f"(s.y) : "f"(d.y));
    u = mul2(a, s);
  }
}
__device__ __forceinline__ float2 dropped(const DropMask& m, bool stays_x, bool stays_y, float2 v) { return make_float2(dropped(m, stays_x, v.x), dropped(m, stays_y, v.y)); }

struct Gate8 { int8_t* codes_a; int8_t* codes_b; uint8_t* exps_a; uint8_t* exps_b; };

template <typename T, bool ROWS, bool DROP>
__global__ void __launch_bounds__(kThreads)
gate8_fwd_kernel(const T* a, const T* b, T* y, const Gate8 kept, int64_t nvec, int64_t n, const Rows rw, const __grid_constant__ DropMask mask) {
  constexpr int N = VecN<T>::N, K = kVecsFwd, S = kBlock8 / N;
  const int64_t v0 = (int64_t)blockIdx.x * (kThreads * K) + threadIdx.x;
  grid_dependents_go();
  grid_dependency_wait();
  uint4 ra[K], rb[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    ra[k] = rb[k] = make_uint4(0, 0, 0, 0);
    if (v0 + k * kThreads < nvec) {
      const int64_t o = operand_vec<ROWS>(v0 + k * kThreads, rw);
      ra[k] = *(reinterpret_cast<const uint4*>(a) + o);
      rb[k] = *(reinterpret_cast<const uint4*>(b) + o);
    }
  }
  Keep<N> keep[K];                                       // while the loads are on their way
  if constexpr (DROP) {
#pragma unroll
    for (int k = 0; k < K; ++k) keep[k] = keep_of<N>(mask, (uint64_t)(v0 + k * kThreads));
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int64_t v = v0 + k * kThreads;
    const uint32_t most_a = block_magnitude<T>(magnitude<T>(ra[k])), most_b = block_magnitude<T>(magnitude<T>(rb[k]));
    const uint32_t byte_a = exponent_byte(most_a), byte_b = exponent_byte(most_b);
    if (v < nvec) {
      float2 fa[N / 2], fb[N / 2], fy[N / 2];
      unpack_pairs<T>(ra[k], fa);
      unpack_pairs<T>(rb[k], fb);
      store_codes<T>(kept.codes_a, v, fa, per_step(byte_a), rounds_past(most_a));
      store_codes<T>(kept.codes_b, v, fb, per_step(byte_b), rounds_past(most_b));
      if (threadIdx.x % S == 0) {
        kept.exps_a[v / S] = (uint8_t)byte_a;
        kept.exps_b[v / S] = (uint8_t)byte_b;
      }
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        float2 s, u;
        sigmoid_silu2<T>(fa[i], s, u);
        fy[i] = mul2(u, fb[i]);
        if constexpr (DROP) fy[i] = dropped(mask, keep[k](2 * i), keep[k](2 * i + 1), fy[i]);
      }
      reinterpret_cast<uint4*>(y)[v] = pack_pairs<T>(fy);
    }
  }
  if (blockIdx.x == 0 && threadIdx.x < 32 && nvec * N < n) {
    const int64_t i = nvec * N + threadIdx.x, o = operand_element<T, ROWS>(i, rw);
    const float fa = i < n ? Cvt<T>::to_f(a[o]) : 0.f, fb = i < n ? Cvt<T>::to_f(b[o]) : 0.f;
    const uint32_t byte_a = tail_exponent(fa), byte_b = tail_exponent(fb);
    if (i < n) {
      kept.codes_a[i] = tail_code(fa, byte_a);
      kept.codes_b[i] = tail_code(fb, byte_b);
      float s, u;
      sigmoid_silu<T>(fa, s, u);
      y[i] = Cvt<T>::from_f(DROP ? dropped(mask, keep_one(mask, (uint64_t)i), u * fb) : u * fb);
    }
    if (threadIdx.x == 0) {
      kept.exps_a[nvec / S] = (uint8_t)byte_a;
      kept.exps_b[nvec / S] = (uint8_t)byte_b;
    }
  }
}

template <typename T, bool DROP>
__device__ __forceinline__ void gate8_bwd_one(const DropMask& m, bool stays, float a, float b, float dy, float& da, float& db, float& y) {
  float s, u;
  sigmoid_silu<T>(a, s, u);
  da = dy * b * (s * (1.f + a * (1.f - s)));
  db = dy * u;
  y = u * b;
  if constexpr (DROP) {
    da = dropped(m, stays, da);
    db = dropped(m, stays, db);
    y = dropped(m, stays, y);
  }
}

template <typename T, bool ROWS, bool DROP>
__global__ void __launch_bounds__(kThreads)
gate8_bwd_kernel(const Gate8 kept, const T* dy, T* da, T* db, T* y, int64_t nvec, int64_t n, const Rows rw, const __grid_constant__ DropMask mask) {
  constexpr int N = VecN<T>::N, K = kVecsBwd<T, DROP>, S = kBlock8 / N;
  const int64_t v0 = (int64_t)blockIdx.x * (kThreads * K) + threadIdx.x;
  grid_dependents_go();
  grid_dependency_wait();
  Codes<T> ca[K], cb[K];
  uint32_t ea[K], eb[K];
  uint4 rg[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int64_t v = v0 + k * kThreads;
    if (v < nvec) {
      ca[k] = load_codes<T>(kept.codes_a, v);
      cb[k] = load_codes<T>(kept.codes_b, v);
      rg[k] = *(reinterpret_cast<const uint4*>(dy) + v);
      ea[k] = kept.exps_a[v / S];
      eb[k] = kept.exps_b[v / S];
    }
  }
  Keep<N> keep[K];                                       // while the loads are on their way
  if constexpr (DROP) {
#pragma unroll
    for (int k = 0; k < K; ++k) keep[k] = keep_of<N>(mask, (uint64_t)(v0 + k * kThreads));
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int64_t v = v0 + k * kThreads;
    if (v < nvec) {
      float2 fa[N / 2], fb[N / 2], fg[N / 2], oy[N / 2];
      values_of<T>(ca[k], ea[k], fa);
      values_of<T>(cb[k], eb[k], fb);
      unpack_pairs<T>(rg[k], fg);
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        float2 s, u;
        sigmoid_silu2<T>(fa[i], s, u);
        oy[i] = mul2(u, fb[i]);
        // a's and b's places take their gradients: da = g b s (1 + a (1 - s)), db = g u
        fa[i] = mul2(mul2(fg[i], fb[i]), mul2(s, fma2(fa[i], fma2(s, both(-1.f), both(1.f)), both(1.f))));
        fb[i] = mul2(fg[i], u);
        if constexpr (DROP) {
          const bool x = keep[k](2 * i), z = keep[k](2 * i + 1);
          fa[i] = dropped(mask, x, z, fa[i]);
          fb[i] = dropped(mask, x, z, fb[i]);
          oy[i] = dropped(mask, x, z, oy[i]);
        }
      }
      const int64_t o = operand_vec<ROWS>(v, rw);
      reinterpret_cast<uint4*>(da)[o] = pack_pairs<T>(fa);
      reinterpret_cast<uint4*>(db)[o] = pack_pairs<T>(fb);
      if (y) reinterpret_cast<uint4*>(y)[v] = pack_pairs<T>(oy);
    }
  }
  if (blockIdx.x == 0 && threadIdx.x < (int)(n - nvec * N)) {
    const int64_t i = nvec * N + threadIdx.x, o = operand_element<T, ROWS>(i, rw);
    float oa, ob, oy;
    gate8_bwd_one<T, DROP>(mask, DROP ? keep_one(mask, (uint64_t)i) : true, tail_value(kept.codes_a[i], kept.exps_a[nvec / S]),
                           tail_value(kept.codes_b[i], kept.exps_b[nvec / S]), Cvt<T>::to_f(dy[i]), oa, ob, oy);
    da[o] = Cvt<T>::from_f(oa);
    db[o] = Cvt<T>::from_f(ob);
    if (y) y[i] = Cvt<T>::from_f(oy);
  }
}

unsigned grid_for(int64_t nvec, int per_thread) {
  const int64_t per = (int64_t)kThreads * per_thread, blocks = (nvec + per - 1) / per;
  return (unsigned)(blocks < 1 ? 1 : blocks);
}
bool aligned16(const void* p) { return p && !(reinterpret_cast<uintptr_t>(p) & 15); }
// vectors of the whole blocks
template <typename T> int64_t whole_vecs(int64_t n) { return n / kBlock8 * (kBlock8 / VecN<T>::N); }

int check_size(int dtype, int64_t n, const char* who) {
  if (dtype != ULM_F16 && dtype != ULM_BF16 && dtype != ULM_F32) return fail(ULM_ERR_ARG, "%s: bad dtype", who);
  if (n < 0) return fail(ULM_ERR_ARG, "%s: negative size", who);
  if (n / 4 / kThreads > 0x7ffffff0LL) return fail(ULM_ERR_TOO_LARGE, "%s: too many elements", who);
  return ULM_OK;
}

int check_gate(const ulm_swiglu8_args* a, const char* who) {
  if (!a) return fail(ULM_ERR_ARG, "%s: null args", who);
  if (int rc = check_size(a->dtype, a->n, who)) return rc;
  if (!drop_p_ok(a->p)) return fail(ULM_ERR_ARG, "%s: p must lie between 0 and 1", who);
  if (a->d) {
    const int64_t vec = a->dtype == ULM_F32 ? 4 : 8;
    if (a->d < 0 || a->d % vec || a->row_stride % vec || a->row_stride < a->d || a->n % a->d) return fail(ULM_ERR_ARG, "%s: rows and their stride must be whole 16-byte vectors", who);
    if (a->n / vec > 0xffffffffLL) return fail(ULM_ERR_TOO_LARGE, "%s: too many elements", who);
  }
  if (a->n && (!aligned16(a->codes_a) || !aligned16(a->codes_b) || !a->exps_a || !a->exps_b)) return fail(ULM_ERR_ARG, "%s: codes must be non-null and 16-byte aligned, exponents non-null", who);
  return ULM_OK;
}

template <typename T, bool DROP>
int gate8_launch(const ulm_swiglu8_args* p, bool bwd, const char* who) {
  cudaStream_t st = (cudaStream_t)p->stream;
  const int64_t nvec = whole_vecs<T>(p->n);
  const Rows rw = make_rows(p->d / VecN<T>::N, p->row_stride / VecN<T>::N);
  const Gate8 kept{p->codes_a, p->codes_b, p->exps_a, p->exps_b};
  const DropMask mask = make_drop_mask(p->p, p->seed);
  const T *a = (const T*)p->a, *b = (const T*)p->b, *dy = (const T*)p->dy;
  T *y = (T*)p->y, *da = (T*)p->da, *db = (T*)p->db;
  if (bwd)
    return launch_dependent(who, p->d ? gate8_bwd_kernel<T, true, DROP> : gate8_bwd_kernel<T, false, DROP>, grid_for(nvec, kVecsBwd<T, DROP>), kThreads, 0, st, kept, dy, da, db, y, nvec, p->n, rw, mask);
  return launch_dependent(who, p->d ? gate8_fwd_kernel<T, true, DROP> : gate8_fwd_kernel<T, false, DROP>, grid_for(nvec, kVecsFwd), kThreads, 0, st, a, b, y, kept, nvec, p->n, rw, mask);
}
template <typename T>
int gate8_launch(const ulm_swiglu8_args* p, bool bwd, const char* who) {
  return p->p > 0 ? gate8_launch<T, true>(p, bwd, who) : gate8_launch<T, false>(p, bwd, who);
}
int gate8(const ulm_swiglu8_args* p, bool bwd, const char* who) {
  return p->dtype == ULM_F16 ? gate8_launch<__half>(p, bwd, who) : p->dtype == ULM_BF16 ? gate8_launch<__nv_bfloat16>(p, bwd, who) : gate8_launch<float>(p, bwd, who);
}

}  // namespace
}  // namespace ulm

extern "C" int64_t ulm_pack8_blocks(int64_t n) { return n < 1 ? 0 : (n + ulm::kBlock8 - 1) / ulm::kBlock8; }

extern "C" int ulm_pack8(const void* x, int8_t* codes, uint8_t* exps, int64_t n, int32_t dtype, void* stream) {
  using namespace ulm;
  const char* who = "ulm_pack8";
  if (int rc = check_size(dtype, n, who)) return rc;
  if (n == 0) return ULM_OK;
  if (!aligned16(x) || !aligned16(codes) || !exps) return fail(ULM_ERR_ARG, "%s: x and codes must be non-null and 16-byte aligned, exponents non-null", who);
  auto go = [&](auto t) {
    using T = decltype(t);
    const int64_t nvec = whole_vecs<T>(n);
    return launch_dependent(who, pack8_kernel<T>, grid_for(nvec, kVecsPack), kThreads, 0, (cudaStream_t)stream, (const T*)x, codes, exps, nvec, n);
  };
  return dtype == ULM_F16 ? go(__half()) : dtype == ULM_BF16 ? go(__nv_bfloat16()) : go(float());
}

extern "C" int ulm_unpack8(const int8_t* codes, const uint8_t* exps, void* x, int64_t n, int32_t dtype, void* stream) {
  using namespace ulm;
  const char* who = "ulm_unpack8";
  if (int rc = check_size(dtype, n, who)) return rc;
  if (n == 0) return ULM_OK;
  if (!aligned16(x) || !aligned16(codes) || !exps) return fail(ULM_ERR_ARG, "%s: x and codes must be non-null and 16-byte aligned, exponents non-null", who);
  auto go = [&](auto t) {
    using T = decltype(t);
    const int64_t nvec = whole_vecs<T>(n);
    return launch_dependent(who, unpack8_kernel<T>, grid_for(nvec, kVecsPack), kThreads, 0, (cudaStream_t)stream, codes, exps, (T*)x, nvec, n);
  };
  return dtype == ULM_F16 ? go(__half()) : dtype == ULM_BF16 ? go(__nv_bfloat16()) : go(float());
}

extern "C" int ulm_swiglu8_fwd(const ulm_swiglu8_args* a) {
  using namespace ulm;
  const char* who = "ulm_swiglu8_fwd";
  if (int rc = check_gate(a, who)) return rc;
  if (a->n == 0) return ULM_OK;
  if (!aligned16(a->a) || !aligned16(a->b) || !aligned16(a->y)) return fail(ULM_ERR_ARG, "%s: a, b, y must be non-null and 16-byte aligned", who);
  return gate8(a, false, who);
}

extern "C" int ulm_swiglu8_bwd(const ulm_swiglu8_args* a) {
  using namespace ulm;
  const char* who = "ulm_swiglu8_bwd";
  if (int rc = check_gate(a, who)) return rc;
  if (a->n == 0) return ULM_OK;
  if (!aligned16(a->dy) || !aligned16(a->da) || !aligned16(a->db) || (a->y && !aligned16(a->y))) return fail(ULM_ERR_ARG, "%s: dy, da, db must be non-null and 16-byte aligned", who);
  return gate8(a, true, who);
}
