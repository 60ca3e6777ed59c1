// Rotary positions of any width, pairing and frequency, without tables (sm_100a).
//
//   (y_i, y_j) = f (x_i cos a - x_j sin a, x_j cos a + x_i sin a),  a = 2 pi (position * turns_i),  backward: a -> -a
//
// for the R / 2 pairs (i, j) of a head's first R columns: j = i + R / 2, or neighbours (interleaved).  The other D - R pass through.
// turns_i is the share of a full turn per position as a 64-bit fixed-point fraction, so that position * turns_i modulo 2^64 is the
// exact share of a turn at any position, of any sign: no large angle is ever formed and none is rounded.  The angle is reduced to an
// eighth of a turn on either side of a quarter in integers, and sine and cosine are the Taylor polynomials there (first
// terms left out: x^11 / 11! < 1.8e-9 and x^12 / 12! < 1.2e-10 for |x| <= pi / 4).  Products and sums fp32, one rounding at the store.
//
// What bounds it: HBM; every element is read once and written once.  A thread owns the same columns of up to kHeads heads of one
// position: the angles depend on position and column alone, and their 25 instructions each are shared by those heads.
#include "common.cuh"

namespace ulm {
namespace {

constexpr int kThreads = 128;

// V elements that lie on a multiple of A
template <typename T, int V, int A> struct alignas(sizeof(T) * A) Vec { T v[V]; };

struct Side { const void* in; void* out; int64_t in_sb, in_sh, in_ss, out_sb, out_sh, out_ss; int heads, chunks; };
struct RotaryParams {
  Side side[2];
  const uint64_t* turns;
  const void* positions;                                 // null: 0, 1, 2, ..
  int64_t pos_sb, pos_ss;
  int S, R, D, turning, units, per_position;             // units: of a head, `turning` of them turn; per_position: threads
  unsigned tasks;
  int pos_32;
  float factor, sign;                                    // sign: -1 backward
};

// cos and sin of `share` / 2^64 turns, times f; the sine also times sign
__device__ __forceinline__ void turn(uint64_t share, float f, float sign, float& c, float& s) {
  const uint32_t top = (uint32_t)(share >> 32), quarter = (top + 0x20000000u) >> 30;
  const int rest = (int)(top - (quarter << 30));         // [-2^29, 2^29): an eighth of a turn either way
  // x = rest 2 pi / 2^32 rounded once: the integer in two floats, the factor in two
  const float hi = __int2float_rn(rest), lo = __int2float_rn(rest - __float2int_rn(hi));
  constexpr double kUnit = 6.283185307179586476925 / 4294967296.0;
  constexpr float u_hi = (float)kUnit, u_lo = (float)(kUnit - (double)u_hi);
  const float x = fmaf(hi, u_hi, fmaf(hi, u_lo, lo * u_hi)), z = x * x;
  float sp = fmaf(z, 1.f / 362880.f, -1.f / 5040.f), cp = fmaf(z, -1.f / 3628800.f, 1.f / 40320.f);
  sp = fmaf(z, sp, 1.f / 120.f);
  cp = fmaf(z, cp, -1.f / 720.f);
  sp = fmaf(z, sp, -1.f / 6.f);
  cp = fmaf(z, cp, 1.f / 24.f);
  sp = fmaf(z * x, sp, x);
  cp = fmaf(z, fmaf(z, cp, -0.5f), 1.f);
  const float a = quarter & 1 ? sp : cp, b = quarter & 1 ? cp : sp;
  c = (quarter + 1) & 2 ? -f * a : f * a;                // quarters 1 and 2: the cosine is negative
  s = quarter & 2 ? -f * sign * b : f * sign * b;        // 2 and 3: the sine
}

template <typename T, int V, int A, bool INTER>
__global__ void __launch_bounds__(kThreads)
rotary_kernel(const __grid_constant__ RotaryParams p) {
  constexpr int kHeads = INTER ? 8 : 4;                  // 8 vectors a thread either way
  const unsigned task = blockIdx.x * kThreads + threadIdx.x;
  grid_dependents_go();
  grid_dependency_wait();
  if (task >= p.tasks) return;
  const unsigned at = task / (unsigned)p.per_position, r = task - at * (unsigned)p.per_position;
  const int chunk = (int)(r / (unsigned)p.units), unit = (int)(r - (unsigned)chunk * (unsigned)p.units);
  const int b = (int)(at / (unsigned)p.S), s = (int)(at - (unsigned)b * (unsigned)p.S);
  const bool second = chunk >= p.side[0].chunks;
  const Side& d = p.side[second];
  const int h0 = (second ? chunk - p.side[0].chunks : chunk) * kHeads, nh = d.heads - h0;
  const T* in = static_cast<const T*>(d.in) + b * d.in_sb + s * d.in_ss + h0 * d.in_sh;
  T* out = static_cast<T*>(d.out) + b * d.out_sb + s * d.out_ss + h0 * d.out_sh;
  using W = Vec<T, V, A>;
  if (unit >= p.turning) {                               // columns that pass through
    const int col = p.R + (unit - p.turning) * V;
    if constexpr (A < V) {                               // a head of an odd number of columns ends inside the last unit
#pragma unroll
      for (int i = 0; i < kHeads; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (i < nh && col + j < p.D) out[i * d.out_sh + col + j] = in[i * d.in_sh + col + j];
      return;
    }
    W w[kHeads];
#pragma unroll
    for (int i = 0; i < kHeads; ++i)
      if (i < nh) w[i] = *reinterpret_cast<const W*>(in + i * d.in_sh + col);
#pragma unroll
    for (int i = 0; i < kHeads; ++i)
      if (i < nh) *reinterpret_cast<W*>(out + i * d.out_sh + col) = w[i];
    return;
  }
  const int col = unit * V, half = p.R >> 1;
  W lo[kHeads], hi[INTER ? 1 : kHeads];
#pragma unroll
  for (int i = 0; i < kHeads; ++i)
    if (i < nh) {
      lo[i] = *reinterpret_cast<const W*>(in + i * d.in_sh + col);
      if constexpr (!INTER) hi[i] = *reinterpret_cast<const W*>(in + i * d.in_sh + col + half);
    }
  uint64_t position = (uint64_t)s;                       // negative positions wrap, as the product does
  if (p.positions) {
    const int64_t o = b * p.pos_sb + s * p.pos_ss;
    position = p.pos_32 ? (uint64_t)(int64_t)static_cast<const int32_t*>(p.positions)[o] : (uint64_t)static_cast<const int64_t*>(p.positions)[o];
  }
  constexpr int kPairs = INTER ? V / 2 : V;
  float cs[kPairs], sn[kPairs];
#pragma unroll
  for (int j = 0; j < kPairs; ++j) turn(position * p.turns[unit * kPairs + j], p.factor, p.sign, cs[j], sn[j]);
#pragma unroll
  for (int i = 0; i < kHeads; ++i)
    if (i < nh) {
#pragma unroll
      for (int j = 0; j < kPairs; ++j) {
        T& ta = INTER ? lo[i].v[2 * j] : lo[i].v[j];
        T& tb = INTER ? lo[i].v[2 * j + 1] : hi[INTER ? 0 : i].v[j];
        const float xa = Cvt<T>::to_f(ta), xb = Cvt<T>::to_f(tb);
        ta = Cvt<T>::from_f(fmaf(xa, cs[j], -(xb * sn[j])));
        tb = Cvt<T>::from_f(fmaf(xb, cs[j], xa * sn[j]));
      }
      *reinterpret_cast<W*>(out + i * d.out_sh + col) = lo[i];
      if constexpr (!INTER) *reinterpret_cast<W*>(out + i * d.out_sh + col + half) = hi[i];
    }
}

template <typename T, bool INTER>
int launch(const RotaryParams& p, int V, cudaStream_t st, const char* who) {
  const unsigned grid = (p.tasks + kThreads - 1) / kThreads;
  auto go = [&](auto kern) { return launch_dependent(who, kern, grid, kThreads, 0, st, p); };
  if constexpr (sizeof(T) == 2)
    if (V == 8) return go(rotary_kernel<T, 8, 8, INTER>);
  if (V == 4) return go(rotary_kernel<T, 4, 4, INTER>);
  if (V == 2) return go(rotary_kernel<T, 2, 2, INTER>);
  if constexpr (INTER) return go(rotary_kernel<T, 2, 1, INTER>);
  else return go(rotary_kernel<T, 1, 1, INTER>);
}

}  // namespace
}  // namespace ulm

extern "C" int ulm_rotary(const ulm_rotary_args* a) {
  using namespace ulm;
  const char* who = "ulm_rotary";
  if (!a) return fail(ULM_ERR_ARG, "%s: null args", who);
  if (a->dtype != ULM_F16 && a->dtype != ULM_BF16 && a->dtype != ULM_F32) return fail(ULM_ERR_ARG, "%s: bad dtype", who);
  if (a->B < 0 || a->S < 0 || a->Hq < 0 || a->Hk < 0 || a->D < 0) return fail(ULM_ERR_ARG, "%s: negative size", who);
  if (a->R <= 0 || a->R % 2 || a->R > a->D) return fail(ULM_ERR_ARG, "%s: the turning columns must be an even number from 2 to the head's width", who);
  if (a->pos_kind < 0 || a->pos_kind > 2) return fail(ULM_ERR_ARG, "%s: bad pos_kind", who);
  if (a->B == 0 || a->S == 0 || (a->Hq == 0 && a->Hk == 0)) return ULM_OK;
  if ((a->Hq && (!a->q || !a->qo)) || (a->Hk && (!a->k || !a->ko)) || !a->turns || (a->pos_kind && !a->positions)) return fail(ULM_ERR_ARG, "%s: null tensor", who);
  const int es = a->dtype == ULM_F32 ? 4 : 2;
  // elements a vector: they divide what turns and what does not, and every head of every tensor starts on a whole one
  int V = 16 / es;
  auto fits = [&](int v) {
    const int64_t t[12] = {a->q_sb, a->q_sh, a->q_ss, a->qo_sb, a->qo_sh, a->qo_ss, a->k_sb, a->k_sh, a->k_ss, a->ko_sb, a->ko_sh, a->ko_ss};
    const void* ptr[4] = {a->q, a->qo, a->k, a->ko};
    if ((a->interleaved ? a->R : a->R / 2) % v || (a->D - a->R) % v) return false;
    for (int i = 0; i < 12; ++i)
      if ((i < 6 ? a->Hq : a->Hk) && t[i] % v) return false;
    for (int i = 0; i < 4; ++i)
      if ((i < 2 ? a->Hq : a->Hk) && reinterpret_cast<uintptr_t>(ptr[i]) % (uintptr_t)(v * es)) return false;
    return true;
  };
  while (V > 1 && !fits(V)) V /= 2;
  if (!fits(V)) return fail(ULM_ERR_ARG, "%s: tensors must lie on whole elements", who);
  if (reinterpret_cast<uintptr_t>(a->turns) % 8 || (a->pos_kind && reinterpret_cast<uintptr_t>(a->positions) % (a->pos_kind == 1 ? 4 : 8)))
    return fail(ULM_ERR_ARG, "%s: turns and positions must lie on whole elements", who);
  RotaryParams p{};
  const int per = a->interleaved ? 8 : 4;
  p.side[0] = {a->q, a->qo, a->q_sb, a->q_sh, a->q_ss, a->qo_sb, a->qo_sh, a->qo_ss, a->Hq, (a->Hq + per - 1) / per};
  p.side[1] = {a->k, a->ko, a->k_sb, a->k_sh, a->k_ss, a->ko_sb, a->ko_sh, a->ko_ss, a->Hk, (a->Hk + per - 1) / per};
  p.turns = reinterpret_cast<const uint64_t*>(a->turns);
  p.positions = a->pos_kind ? a->positions : nullptr;
  p.pos_sb = a->pos_sb; p.pos_ss = a->pos_ss; p.pos_32 = a->pos_kind == 1;
  p.S = a->S; p.R = a->R; p.D = a->D;
  const int step = a->interleaved && V == 1 ? 2 : V;     // a thread has whole pairs
  p.turning = (a->interleaved ? a->R : a->R / 2) / step;
  p.units = p.turning + (a->D - a->R + step - 1) / step;
  const int64_t per_position = (int64_t)p.units * (p.side[0].chunks + p.side[1].chunks);
  const int64_t positions = (int64_t)a->B * a->S;
  if (per_position > 0x7fffffffLL || positions > 0xfffffff0LL / per_position) return fail(ULM_ERR_TOO_LARGE, "%s: too many elements", who);
  p.per_position = (int)per_position;
  p.tasks = (unsigned)(positions * per_position);
  p.factor = a->factor; p.sign = a->backward ? -1.f : 1.f;
  cudaStream_t st = (cudaStream_t)a->stream;
  auto go = [&](auto t) {
    using T = decltype(t);
    return a->interleaved ? launch<T, true>(p, V, st, who) : launch<T, false>(p, V, st, who);
  };
  return a->dtype == ULM_F16 ? go(__half()) : a->dtype == ULM_BF16 ? go(__nv_bfloat16()) : go(float());
}
