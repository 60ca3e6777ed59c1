// Rotary positions of any width, pairing and frequency, without tables (sm_100a).
//
//   (y_i, y_j) = f (x_i cos a - x_j sin a, x_j cos a + x_i sin a),  a = 2 pi (position * turns_i),  backward: a -> -a
//
// for the R / 2 pairs (i, j) of a head's first R columns: j = i + R / 2, or neighbours (interleaved).  The other D - R pass through.
// turns_i is the share of a full turn per position as a 64-bit fixed-point fraction, so that position * turns_i modulo 2^64 is the
// share of a turn at any position, of any sign, without an error beyond turns_i's own: no large angle is ever formed.  It is reduced to an
// eighth of a turn on either side of a quarter in integers, cut to 2^-58 of a turn, and rounded once, to fp32: a sine is good
// relative to itself, also a slow pair's near position 0.  Sine and cosine are the Taylor polynomials there (first
// terms left out: x^11 / 11! < 1.8e-9 and x^12 / 12! < 1.2e-10 for |x| <= pi / 4).  Products and sums fp32, one rounding at the store.
//
// What bounds it: HBM; every element is read once and written once.  A thread owns the same columns of up to kHeads heads of one
// position: the angles depend on position and column alone, and their 25 instructions each are shared by those heads.
#include "common.cuh"

namespace ulm {
namespace {

constexpr int kThreads = 128;
constexpr int kMaxTile = 16, kTileBytes = 16384;         // positions and bytes of a CTA that works on whole rows (8 and 32 KB: no faster)
constexpr int kRowsBelow = 4;                            // which it does where vectors of what turns have at most so many bytes
constexpr unsigned kGroup = kThreads;                    // positions; a multiple of kThreads

// V elements that lie on a multiple of A
template <typename T, int V, int A> struct alignas(sizeof(T) * A) Vec { T v[V]; };

struct Side { const void* in; void* out; int64_t in_sb, in_sh, in_ss, out_sb, out_sh, out_ss; int heads, chunks; };
struct RotaryParams {
  Side side[2];
  const uint64_t* turns;
  const void* positions;                                 // null: 0, 1, 2, ..
  int64_t pos_sb, pos_ss;
  unsigned turning, passing, chunks;                     // units of a head that turn and that pass through; groups of heads of both tensors
  unsigned turn_tasks, per_group, count;                 // threads of a group of positions: for what turns, in all; positions
  int S, R, D, pos_32, pass_wide;                        // pass_wide: whole 16-byte vectors whatever V is
  int tile;                                              // positions of a CTA that works on whole rows, or 0
  float factor, sign;                                    // sign: -1 backward
};

// negative positions wrap, as their product with a share of a turn does
__device__ __forceinline__ uint64_t position_of(const RotaryParams& p, int b, int s) {
  if (!p.positions) return (uint64_t)s;
  const int64_t o = b * p.pos_sb + s * p.pos_ss;
  return p.pos_32 ? (uint64_t)(int64_t)static_cast<const int32_t*>(p.positions)[o] : (uint64_t)static_cast<const int64_t*>(p.positions)[o];
}

// cos and sin of `share` / 2^64 turns, times f; the sine also times sign
__device__ __forceinline__ void turn(uint64_t share, float f, float sign, float& c, float& s) {
  const uint32_t top = (uint32_t)(share >> 32), quarter = (top + 0x20000000u) >> 30;
  const int rest = (int)(top - (quarter << 30));         // [-2^29, 2^29): an eighth of a turn either way, and the lower word behind it
  // the nearest multiple of 64, which an fp32 number holds, and 32 bits below it, of which the first six are the rest's: a slow pair
  // near position 0 turns by less than 2^-32, so that the lower word is all of its angle
  const float hi = __int2float_rn((rest + 32) & ~63), lo = __int2float_rn((int)__funnelshift_r((uint32_t)share, top, 6));
  // x = (hi + lo / 2^26) 2 pi / 2^32, rounded once: the factor in two floats
  constexpr double kUnit = 6.283185307179586476925 / 4294967296.0;
  constexpr float u_hi = (float)kUnit, u_lo = (float)(kUnit - (double)u_hi), u_26 = (float)(kUnit / 67108864.0);
  const float x = fmaf(hi, u_hi, fmaf(hi, u_lo, lo * u_26)), z = x * x;
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

// Heads a thread: 8 vectors of 16 bytes in flight where pairs lie apart, 4 where they are neighbours.  8x12x4096x64 bf16, 2 / 4 / 6 heads:
// apart 40.1 / 32.8 / 32.5 us (floor 30.7), neighbours 31.9 with 4, 33.1 with 6, 35.8 with 8; 12 heads leave a thread of 8 heads half empty.
// CTAs of 256 threads: 37.7 and 33.7.  What passes through in warps of its own: 1x(16+4)x32001x128 fp16, half of it turning, 64 -> 50.1 us
// (floor 50.0), as against both in one warp, which waited for memory twice.
constexpr int kHeads = 4;

// Seven CTAs on an SM are 72 registers; at 80, and so six, 8x12x4096x64 bf16 takes 34.4 us for 33.
template <typename T, int V, int A, bool INTER>
__global__ void __launch_bounds__(kThreads, 7)
rotary_kernel(const __grid_constant__ RotaryParams p) {
  constexpr int H = kHeads;
  grid_dependents_go();
  grid_dependency_wait();
  // of every kGroup positions first all that turns, then all that passes through: no warp has both, and the two halves of a
  // row of memory are asked for within a short time
  const unsigned task = blockIdx.x * kThreads + threadIdx.x, group = task / p.per_group, rest = task - group * p.per_group;
  const bool turns = rest < p.turn_tasks;
  const unsigned units = turns ? p.turning : p.passing, per_position = units * p.chunks, local = turns ? rest : rest - p.turn_tasks;
  const unsigned in_group = local / per_position, at = group * kGroup + in_group, r = local - in_group * per_position;
  if (at >= p.count) return;
  const int chunk = (int)(r / units), unit = (int)(r - (unsigned)chunk * units);
  const int b = (int)(at / (unsigned)p.S), s = (int)(at - (unsigned)b * (unsigned)p.S);
  const bool second = chunk >= p.side[0].chunks;
  const Side& d = p.side[second];
  const int h0 = (second ? chunk - p.side[0].chunks : chunk) * H, nh = d.heads - h0;
  const T* in = static_cast<const T*>(d.in) + b * d.in_sb + s * d.in_ss + h0 * d.in_sh;
  T* out = static_cast<T*>(d.out) + b * d.out_sb + s * d.out_ss + h0 * d.out_sh;
  using W = Vec<T, V, A>;
  if (!turns) {
    auto copy = [&](auto w0, int col) {
      using C = decltype(w0);
      C w[H];
#pragma unroll
      for (int i = 0; i < H; ++i)
        if (i < nh) w[i] = *reinterpret_cast<const C*>(in + i * d.in_sh + col);
#pragma unroll
      for (int i = 0; i < H; ++i)
        if (i < nh) *reinterpret_cast<C*>(out + i * d.out_sh + col) = w[i];
    };
    const int col = p.R + unit * V;
    if (p.pass_wide) copy(uint4(), p.R + unit * (int)(16 / sizeof(T)));
    else if (A == V || col + V <= p.D) copy(W(), col);
    else copy(T(), col);                                 // a head of an odd number of columns ends inside its last unit
    return;
  }
  const int col = unit * V, half = p.R >> 1;
  W lo[H], hi[INTER ? 1 : H];
#pragma unroll
  for (int i = 0; i < H; ++i)
    if (i < nh) {
      lo[i] = *reinterpret_cast<const W*>(in + i * d.in_sh + col);
      if constexpr (!INTER) hi[i] = *reinterpret_cast<const W*>(in + i * d.in_sh + col + half);
    }
  const uint64_t position = position_of(p, b, s);
  constexpr int kPairs = INTER ? V / 2 : V;
  float cs[kPairs], sn[kPairs];
#pragma unroll
  for (int j = 0; j < kPairs; ++j) turn(position * p.turns[unit * kPairs + j], p.factor, p.sign, cs[j], sn[j]);
#pragma unroll
  for (int i = 0; i < H; ++i)
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

// Where what turns is made of vectors of 4 bytes at most (R / 2 is a multiple of little, or R for neighbours) though the rows are whole 16-byte
// vectors: a CTA brings the rows of kHeads heads at p.tile positions into shared memory, turns them there element by element and stores
// them by whole vectors again.  us with the widest vectors that fit / this way (the bytes alone), 4 x 16 heads x 4096 positions fp16: 128 columns, 66 turn,
// halves 55 / 27 (20), 68 turn 32 / 27, 126 turn 49 / 36; 96 columns, 50 turn, halves 42 / 21 (15), neighbours 29 / 21; 13 x 4 heads x 10550 x 96, 2 turn,
// neighbours 108 / 37 (32).  With vectors of 8 bytes the direct way is the faster: 72 of 128 turn 23 / 30, fp32 36 of 80 28 / 29.
template <typename T, bool INTER>
__global__ void __launch_bounds__(kThreads)
rotary_rows_kernel(const __grid_constant__ RotaryParams p) {
  constexpr int H = kHeads, N = 16 / sizeof(T);
  extern __shared__ __align__(16) char mem[];            // [tile][H][D]
  __shared__ int64_t from[kMaxTile], to[kMaxTile];       // where a position's heads lie, in elements
  __shared__ uint64_t place[kMaxTile];
  T* rows = reinterpret_cast<T*>(mem);
  grid_dependents_go();
  grid_dependency_wait();
  const int chunk = (int)(blockIdx.x % p.chunks), tile = p.tile, tid = threadIdx.x;
  const unsigned first = blockIdx.x / p.chunks * (unsigned)tile;
  const bool second = chunk >= p.side[0].chunks;
  const Side& d = p.side[second];
  const int h0 = (second ? chunk - p.side[0].chunks : chunk) * H, nh = d.heads - h0 < H ? d.heads - h0 : H;
  const int held = p.count - first < (unsigned)tile ? (int)(p.count - first) : tile;       // positions
  if (tid < held) {
    const unsigned at = first + (unsigned)tid;
    const int b = (int)(at / (unsigned)p.S), s = (int)(at - (unsigned)b * (unsigned)p.S);
    from[tid] = b * d.in_sb + s * d.in_ss + h0 * d.in_sh;
    to[tid] = b * d.out_sb + s * d.out_ss + h0 * d.out_sh;
    place[tid] = position_of(p, b, s);
  }
  __syncthreads();
  // thread beside thread over the columns of the rows, counted on without divisions
  auto over = [&](int per_row, int rows, auto&& use) {
    const int hop_row = kThreads / per_row, hop = kThreads - hop_row * per_row;
    int row = tid / per_row, i = tid - row * per_row;
    while (row < rows) {
      use(row, i);
      row += hop_row; i += hop;
      if (i >= per_row) { i -= per_row; ++row; }
    }
  };
  const int inverse = 65536 / nh + 1;                    // row / nh is row * inverse / 65536: rows below kMaxTile H
  over(p.D / N, held * nh, [&](int row, int v) {
    const int at = row * inverse >> 16, h = row - at * nh;
    const uint32_t to_smem = (uint32_t)__cvta_generic_to_shared(rows + (at * H + h) * p.D + v * N);
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to_smem), "l"(static_cast<const T*>(d.in) + from[at] + h * d.in_sh + v * N) : "memory");
  });
  asm volatile("cp.async.commit_group;" ::: "memory");
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  const int pairs = p.R >> 1, second_of = INTER ? 1 : pairs;
  over(pairs, held, [&](int at, int pair) {
    float c, sn;
    turn(place[at] * p.turns[pair], p.factor, p.sign, c, sn);
    T* row = rows + at * H * p.D + (INTER ? 2 * pair : pair);
#pragma unroll
    for (int h = 0; h < H; ++h)
      if (h < nh) {
        T *a = row + h * p.D, *b = a + second_of;
        const float xa = Cvt<T>::to_f(*a), xb = Cvt<T>::to_f(*b);
        *a = Cvt<T>::from_f(fmaf(xa, c, -(xb * sn)));
        *b = Cvt<T>::from_f(fmaf(xb, c, xa * sn));
      }
  });
  __syncthreads();
  over(p.D / N, held * nh, [&](int row, int v) {
    const int at = row * inverse >> 16, h = row - at * nh;
    *reinterpret_cast<uint4*>(static_cast<T*>(d.out) + to[at] + h * d.out_sh + v * N) = *reinterpret_cast<const uint4*>(rows + (at * H + h) * p.D + v * N);
  });
}

template <typename T, bool INTER>
int launch(const RotaryParams& p, int V, cudaStream_t st, const char* who) {
  if (p.tile) {
    const unsigned blocks = (p.count + (unsigned)p.tile - 1) / (unsigned)p.tile * p.chunks;
    return launch_dependent(who, rotary_rows_kernel<T, INTER>, blocks, kThreads, (size_t)p.tile * kHeads * p.D * sizeof(T), st, p);
  }
  const unsigned grid = (p.count + kGroup - 1) / kGroup * (p.per_group / kThreads);
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
  const int wide = 16 / es;
  auto starts_on = [&](int v) {                          // every head of every tensor on a whole vector
    const int64_t t[12] = {a->q_sb, a->q_sh, a->q_ss, a->qo_sb, a->qo_sh, a->qo_ss, a->k_sb, a->k_sh, a->k_ss, a->ko_sb, a->ko_sh, a->ko_ss};
    const void* ptr[4] = {a->q, a->qo, a->k, a->ko};
    for (int i = 0; i < 12; ++i)
      if ((i < 6 ? a->Hq : a->Hk) && t[i] % v) return false;
    for (int i = 0; i < 4; ++i)
      if ((i < 2 ? a->Hq : a->Hk) && reinterpret_cast<uintptr_t>(ptr[i]) % (uintptr_t)(v * es)) return false;
    return true;
  };
  if (!starts_on(1)) return fail(ULM_ERR_ARG, "%s: tensors must lie on whole elements", who);
  // elements a vector: they divide what turns, and what does not
  const bool pass_wide = a->R % wide == 0 && (a->D - a->R) % wide == 0 && starts_on(wide);
  auto fits = [&](int v) { return (a->interleaved ? a->R : a->R / 2) % v == 0 && (pass_wide || (a->D - a->R) % v == 0) && starts_on(v); };
  int V = wide;
  while (V > 1 && !fits(V)) V /= 2;
  if (reinterpret_cast<uintptr_t>(a->turns) % 8 || (a->pos_kind && reinterpret_cast<uintptr_t>(a->positions) % (a->pos_kind == 1 ? 4 : 8)))
    return fail(ULM_ERR_ARG, "%s: turns and positions must lie on whole elements", who);
  RotaryParams p{};
  const int per = kHeads;
  p.side[0] = {a->q, a->qo, a->q_sb, a->q_sh, a->q_ss, a->qo_sb, a->qo_sh, a->qo_ss, a->Hq, (a->Hq + per - 1) / per};
  p.side[1] = {a->k, a->ko, a->k_sb, a->k_sh, a->k_ss, a->ko_sb, a->ko_sh, a->ko_ss, a->Hk, (a->Hk + per - 1) / per};
  p.turns = reinterpret_cast<const uint64_t*>(a->turns);
  p.positions = a->pos_kind ? a->positions : nullptr;
  p.pos_sb = a->pos_sb; p.pos_ss = a->pos_ss; p.pos_32 = a->pos_kind == 1;
  p.S = a->S; p.R = a->R; p.D = a->D;
  const int step = a->interleaved && V == 1 ? 2 : V;     // a thread has whole pairs
  p.turning = (unsigned)((a->interleaved ? a->R : a->R / 2) / step);
  p.pass_wide = pass_wide;
  p.passing = (unsigned)(pass_wide ? (a->D - a->R) / wide : (a->D - a->R + step - 1) / step);
  p.chunks = (unsigned)(p.side[0].chunks + p.side[1].chunks);
  // what passes through is where it belongs already
  if ((!a->Hq || a->q == a->qo) && (!a->Hk || a->k == a->ko)) p.passing = 0;
  const int64_t positions = (int64_t)a->B * a->S, per_position = (int64_t)(p.turning + p.passing) * p.chunks;
  if (per_position * kGroup > 0x7fffffffLL || positions > 0x7fffff00LL || (positions + kGroup) * per_position > 0xffffffffLL)
    return fail(ULM_ERR_TOO_LARGE, "%s: too many elements", who);
  p.count = (unsigned)positions;
  p.turn_tasks = (unsigned)(kGroup * p.turning * p.chunks);
  p.per_group = (unsigned)(kGroup * per_position);
  // whole rows: where vectors are at most kRowsBelow bytes though the rows are made of whole ones, and a few rows fit 16 KB
  const int64_t row_bytes = (int64_t)a->D * es;
  if (V * es <= kRowsBelow && a->D % wide == 0 && starts_on(wide) && kHeads * row_bytes <= kTileBytes)
    p.tile = (int)(kTileBytes / (kHeads * row_bytes) < kMaxTile ? kTileBytes / (kHeads * row_bytes) : kMaxTile);
  p.factor = a->factor; p.sign = a->backward ? -1.f : 1.f;
  cudaStream_t st = (cudaStream_t)a->stream;
  auto go = [&](auto t) {
    using T = decltype(t);
    return a->interleaved ? launch<T, true>(p, V, st, who) : launch<T, false>(p, V, st, who);
  };
  return a->dtype == ULM_F16 ? go(__half()) : a->dtype == ULM_BF16 ? go(__nv_bfloat16()) : go(float());
}
