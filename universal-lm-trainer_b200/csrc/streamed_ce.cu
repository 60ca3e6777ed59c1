// lm head + softmax cross-entropy over a large vocabulary in pieces of the vocabulary, with its gradient, without the logits
// (sm_100a).
//
//   z = H W^T (fp32 accumulators, never stored),  l_r = ln sum_c exp z[r,c],  loss_r = l_r - z[r, target_r]
//   G[r,c] = exp(z[r,c] - l_r) - [c = target_r]          (0 on ignored rows)
//   dH = g G W,   dW = g G^T H                           g: one factor for all rows, in device memory
//
// Forward: one pass over the vocabulary that keeps a running maximum and sum per row, and the target's logit.  Backward, for
// one piece of the vocabulary at a time: z again, G of the piece in 16 bits into a workspace [rows, piece], then the two
// products that read it; dH is summed over the pieces in fp32.  So 8 rows V d flops where keeping the logits takes 6, and
// a workspace whose size does not depend on the vocabulary.
//
// G is the only rounding before the results': to 16 bits, which the tensor cores take, with fp32 sums of exact
// products behind it.  fp16 would lose probabilities below 2^-24, so its G is held times 2^14 (|G| <= 1) and the factor taken
// back in the fp32 epilogue.  z is not rounded to 16 bits.
//
// All four products run through one main loop: persistent pairs of CTAs of 320 threads, one CTA per SM (warps 0-7 epilogue, warp
// 8 one-lane TMA producer, warp 9 of the pair's first CTA one-lane tcgen05.mma issuer), output tiles of 256 x 256, M256 x
// N256 x K16 instructions over both CTAs, six stages of 128x64 + 128x64 operands a CTA in 128-byte-swizzled shared memory, two
// accumulators of 256 TMEM columns so that a tile's epilogue runs under the next one's products.  H and W are stored with d contiguous and G with the vocabulary
// contiguous, so dH reads W, and dW reads both G and H, as MN-major operands: rows of 64-element atoms, no transposed copies.
// What bounds it from widths of 512 on: the tensor pipe, active 87-94 % of the cycles, and the clock that the power limit leaves.
// 32768 x 768 x 32000 bf16, forward and backward: 4.4 ms in short runs, 5.0-5.5 ms under lasting load, by the GPU (1160-1280 TFLOP/s of the
// products that are formed; library GEMMs of the same shapes 1120-1190).  One CTA a product instead of a pair: 5.69 ms where the pair
// took 5.48.  Narrower: the exponentials, 256 x 128 of them a CTA and tile, and G's way through memory (written once, read twice, at 6 TB/s);
// the products' column tiles are 256 wide whatever the width, the rest zeros; 32768 x 64 x 32000 2.3 ms.
// Waits are bounded (status bit and clean exit on expiry), like the attention kernels'.
#include "lmhead_tiles.cuh"
#include "tc.cuh"

#include <algorithm>

namespace ulm {
namespace {

using namespace tc;

enum Mode { kStats, kGrad, kProducts };                  // statistics; G; dW = G^T H and dH = G W
enum Product { kColGrad, kRowGrad, kNumProducts };       // dW, dH

constexpr int kPairM = 2 * LM_BM;                         // rows of a pair's output tile
constexpr int kPairs = kNumSMs / 2;
constexpr int kStages = 6;
constexpr int kBRows = LM_BN / 2;                        // columns of B that each CTA of a pair holds
constexpr uint32_t kATile = LM_BM * LM_BK * 2;           // 16 KB
constexpr uint32_t kBTile = kBRows * LM_BK * 2;          // 16 KB
constexpr uint32_t kStage = kATile + kBTile;             // of one CTA
constexpr uint32_t kAtom = 64 * 64 * 2;                  // one MN-major box: 64 (MN) x 64 (K)
constexpr uint32_t kStaging = 32 * 128;                  // a warp's 32 rows x 128 bytes of output
constexpr int kEpiWarps = 8;
constexpr int kThreads = (kEpiWarps + 2) * 32;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int64_t kSlot = (int64_t)kPairM * LM_BN;       // floats of one partial tile

template <typename T> struct Fmt { static constexpr int idesc = 0, g_shift = 14; };
template <> struct Fmt<__nv_bfloat16> { static constexpr int idesc = 1, g_shift = 0; };

struct Ctl {
  uint64_t full[kStages], empty[kStages], acc_full[2], acc_free[2];
  uint32_t tmem_base;
  int abort;
  uint32_t fail_bits;
};
constexpr size_t kCtlBytes = 1024;
static_assert(sizeof(Ctl) <= kCtlBytes, "control block");
constexpr size_t smem_bytes(int mode) { return 1024 + (size_t)kStages * kStage + (mode == kStats ? 0 : kEpiWarps * (size_t)kStaging) + kCtlBytes; }
static_assert(smem_bytes(kGrad) <= 227 * 1024, "shared memory");

// One launch's work.  Items are numbered and dealt round the CTAs.
//   statistics: 256 rows x a group of column tiles, whose statistics stay in registers;
//   G: one tile each, rows fastest, so that all CTAs read one stretch of W;
//   products: dW's and dH's `whole` tiles, then of each the `rest` that would not fill a round of the SMs, cut into `split`
//   stretches of the inner dimension; every stretch leaves its fp32 tile in a slot, and a second kernel adds up a tile's slots
//   in order.  Both products in one launch: one set-up and one drain less, and a launch or two of
//   the host's time (forward and backward, replayed as a graph: 7 x 768 x 32000 72 -> 69.5 us, x 2560 40 -> 32; the largest calls 0.5 %
//   slower).
struct Work {
  int n_mt, n_nt, n_kb, group;
  int whole, rest, split;
};
struct Item { int mt, nt, count, kb0, kb1, slot, product; };

// How the accumulators leave: out = factor * acc (+ prev).  A whole tile goes through shared memory and a TMA store, or where an
// fp32 out is its own prev a TMA addition (one to each element: no order to depend on); where a 16-bit out adds an fp32 prev,
// straight from the registers.  A cut tile's parts go to their slots, fp32 and without factor, and out by the join kernel.
struct Out {
  const float *factor_dev, *factor2_dev;
  float factor;
  const float* prev;
  void* out;
  int64_t ld, rows;                                      // of out and prev
  int cols, is_f32;
  float* slots;
};
// Bytes of A that the CTAs of a pair load per k-block, and of B each; the K16 steps of a k-block.  Where all rows fit one CTA's
// half tile, boxes end with them and the other CTA loads no A; an inner dimension of less than one k-block ends with its
// last step.  Zeros past a tensor's end cost a load more than data does: 7 rows, forward 25 -> 21 us.
struct Load {
  uint32_t a_bytes[2], b_bytes;
  int k_steps;
};
struct Products {
  Work w[kNumProducts];
  Out out[kNumProducts];
  Load load[kNumProducts];
  int slot0[kNumProducts];
};
// A and B, of the second product too; what is written; the slots
struct alignas(64) Maps { CUtensorMap a[kNumProducts], b[kNumProducts], out[kNumProducts], slots; };

struct Params {
  Work w;                                                // statistics and G
  Load load;
  int64_t rows;
  int V, v0;                                             // vocabulary; first column of the piece
  const int64_t* target;
  int64_t ignore_index;
  float *part_m, *part_s, *z_target;                     // statistics
  uint32_t* done;
  const float* lse;                                      // G
  int g_cols;                                            // the workspace's columns
  Products products;
  uint32_t* status;
};

template <int MODE>
__host__ __device__ inline int n_items(const Params& p) {
  if (MODE == kStats) return p.w.n_mt * ((p.w.n_nt + p.w.group - 1) / p.w.group);
  if (MODE == kGrad) return p.w.n_mt * p.w.n_nt;
  const Work *c = &p.products.w[kColGrad], *r = &p.products.w[kRowGrad];
  return c->whole + r->whole + c->rest * c->split + r->rest * r->split;
}
template <int MODE>
__device__ __forceinline__ Item item_of(const Params& p, int q) {
  Item it{0, 0, 1, 0, p.w.n_kb, -1, 0};
  if constexpr (MODE == kStats) {
    const int g = q / p.w.n_mt;
    it.mt = q - g * p.w.n_mt;
    it.nt = g * p.w.group;
    it.count = min(p.w.group, p.w.n_nt - it.nt);
  } else if constexpr (MODE == kGrad) {
    it.nt = q / p.w.n_mt;
    it.mt = q - it.nt * p.w.n_mt;
  } else {
    const Work *c = &p.products.w[kColGrad], *r = &p.products.w[kRowGrad];
    int part = -1;
    if (q >= c->whole) {
      q -= c->whole;
      it.product = kRowGrad;
      if (q >= r->whole) {
        part = q - r->whole;
        if (part < c->rest * c->split) it.product = kColGrad;
        else part -= c->rest * c->split;
      }
    }
    const Work& w = p.products.w[it.product];
    int t = q;
    it.kb1 = w.n_kb;
    if (part >= 0) {
      const int s = part / w.rest, j = part - s * w.rest;
      t = w.whole + j;
      it.kb0 = (int)((int64_t)w.n_kb * s / w.split);
      it.kb1 = (int)((int64_t)w.n_kb * (s + 1) / w.split);
      if (w.split > 1) it.slot = p.products.slot0[it.product] + j * w.split + s;
    }
    it.mt = t / w.n_nt;                                  // the column tiles of one row tile side by side: they share its A panel in L2
    it.nt = t - it.mt * w.n_nt;
  }
  return it;
}

__device__ __forceinline__ float out_factor(const Out& o) { return *o.factor_dev * (o.factor2_dev ? *o.factor2_dev : 1.f) * o.factor; }

// 128 bytes of a row of a warp's block into shared memory, lane = row, as the 128-byte swizzle has them: 16-byte chunk c at chunk
// position c ^ (lane & 7); then one TMA store or addition of the block to (col, row) of `map`.  Whole warp.
template <bool ADD>
__device__ __forceinline__ void store_block(const CUtensorMap* map, uint8_t* block, int lane, const uint32_t (&u)[32], int col, int row, int z = 0) {
  if (lane == 0) bulk_wait_read0();                      // the warp's previous store must have read the block
  __syncwarp();
  uint8_t* line = block + lane * 128;
#pragma unroll
  for (int c = 0; c < 8; ++c)
    *reinterpret_cast<uint4*>(line + ((c ^ (lane & 7)) << 4)) = make_uint4(u[4 * c], u[4 * c + 1], u[4 * c + 2], u[4 * c + 3]);
  fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) {
    if (ADD) tma_add_4d(map, block, col, row, z, 0); else tma_store_4d(map, block, col, row, z, 0);
    bulk_commit();
  }
}
// 64 fp32 columns as two blocks
template <bool ADD>
__device__ __forceinline__ void store_f32(const CUtensorMap* map, uint8_t* block, int lane, const uint32_t (&acc)[64], float factor, int col, int cols, int row) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (col + 32 * h >= cols) break;
    uint32_t u[32];
#pragma unroll
    for (int c = 0; c < 32; ++c) u[c] = __float_as_uint(factor * __uint_as_float(acc[32 * h + c]));
    store_block<ADD>(map, block, lane, u, col + 32 * h, row);
  }
}

// 64 accumulator columns of one row plus fp32 values, rounded to 16 bits
template <typename T>
__device__ __forceinline__ void add_and_round(const Out& o, float factor, int64_t row, int col, const uint32_t (&acc)[64]) {
  if (row >= o.rows) return;
#pragma unroll
  for (int c = 0; c < 64; c += 8) {
    if (col + c < o.cols) {                              // the width is whole vectors of 8
      const int64_t at = row * o.ld + col + c;
      const float4 a = *reinterpret_cast<const float4*>(o.prev + at), b = *reinterpret_cast<const float4*>(o.prev + at + 4);
      float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] += factor * __uint_as_float(acc[c + j]);
      *reinterpret_cast<uint4*>(static_cast<T*>(o.out) + at) =
          make_uint4(Cvt<T>::pack2(v[0], v[1]), Cvt<T>::pack2(v[2], v[3]), Cvt<T>::pack2(v[4], v[5]), Cvt<T>::pack2(v[6], v[7]));
    }
  }
}

template <typename T, int MODE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
streamed_ce_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Params p) {
  constexpr bool kBmn = MODE == kProducts;               // and A too in dW
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* stages = base;                                             // [stage][A tile | B tile]
  uint8_t* staging = base + (size_t)kStages * kStage;                 // [epilogue warp] one block each
  Ctl* ctl = reinterpret_cast<Ctl*>(staging + (MODE == kStats ? 0 : kEpiWarps * (size_t)kStaging));
  volatile int* abort_flag = &ctl->abort;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int items = n_items<MODE>(p);
  const uint32_t rank = cluster_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

  // full and acc_free are awaited in the CTA of rank 0, which issues the products: its full counts the bytes of both CTAs,
  // its acc_free an arrival of every epilogue warp of both
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) { mbar_init(&ctl->full[s], 1); mbar_init(&ctl->empty[s], 1); }
    for (int b = 0; b < 2; ++b) { mbar_init(&ctl->acc_full[b], 1); mbar_init(&ctl->acc_free[b], 2 * kEpiWarps); }
    ctl->abort = 0;
    ctl->fail_bits = 0;
    fence_mbar_init();
  }
  if (warp == kEpiWarps + 1) { tmem_alloc_pair(&ctl->tmem_base, 512); tmem_relinquish_pair(); }
  fence_before_sync();
  __syncthreads();
  cluster_sync();                                        // the other CTA's barriers are set up before anything signals them
  fence_after_sync();
  grid_dependents_go();
  grid_dependency_wait();
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, ctl->tmem_base, 0);   // warp-uniform

  if (MODE == kStats && blockIdx.x == 0 && threadIdx.x == 0) *p.done = 0u;
  if (warp == kEpiWarps) {
    // ---------------- TMA producer ----------------
    if (elect_one()) {
      for (int i = 0; i < (MODE == kProducts ? (int)kNumProducts : 1); ++i)
        if (MODE != kProducts || p.products.w[i].n_kb) { tma_prefetch_desc(&maps.a[i]); tma_prefetch_desc(&maps.b[i]); }
      uint32_t it = 0;                                   // k-blocks issued so far, over all tiles
      bool ok = true;
      for (int q = pair; ok && q < items; q += pairs) {
        const Item im = item_of<MODE>(p, q);
        const Load& load = MODE == kProducts ? p.products.load[im.product] : p.load;
        const CUtensorMap *tmA = &maps.a[im.product], *tmB = &maps.b[im.product];
        for (int t = 0; ok && t < im.count; ++t) {
          const int m0 = im.mt * kPairM + (int)rank * LM_BM, n0 = (im.nt + t) * LM_BN + (int)rank * kBRows;
          for (int kb = im.kb0; kb < im.kb1; ++kb, ++it) {
            const uint32_t s = it % kStages;
            if (it >= (uint32_t)kStages && !mbar_wait(&ctl->empty[s], ((it / kStages) - 1) & 1, abort_flag)) {
              atomicOr(&ctl->fail_bits, (uint32_t)ULM_STATUS_TIMEOUT_MMA);
              ok = false;
              break;
            }
            uint8_t* a = stages + (size_t)s * kStage;
            uint8_t* b = a + kATile;
            const int k0 = kb * LM_BK;
            if (rank == 0) mbar_expect_tx(&ctl->full[s], load.a_bytes[0] + load.a_bytes[1] + 2 * load.b_bytes);
            const uint32_t full = peer_smem(&ctl->full[s], 0);
            // W's rows are vocabulary columns, counted from the piece's first; G's blocks of 64 columns are its third dimension
            if constexpr (MODE == kProducts) {
              if (im.product == kColGrad) {
#pragma unroll
                for (int i = 0; i < LM_BM / 64; ++i) tma_load_4d_pair(a + i * kAtom, tmA, full, 0, k0, (m0 >> 6) + i, 0);
              } else if (load.a_bytes[rank]) {
                tma_load_4d_pair(a, tmA, full, 0, m0, kb, 0);
              }
              const int row = im.product == kColGrad ? k0 : p.v0 + k0;
#pragma unroll
              for (int i = 0; i < kBRows / 64; ++i) tma_load_4d_pair(b + i * kAtom, tmB, full, n0 + 64 * i, row, 0, 0);
            } else {
              if (load.a_bytes[rank]) tma_load_4d_pair(a, tmA, full, k0, m0, 0, 0);
              tma_load_4d_pair(b, tmB, full, k0, p.v0 + n0, 0, 0);
            }
          }
        }
      }
    }
  } else if (warp == kEpiWarps + 1) {
    // ---------------- MMA issuer: rank 0 for both ----------------
    if (rank == 0 && elect_one()) {
      constexpr uint64_t kStepK = 32 >> 4, kStepMN = 2048 >> 4;      // 16 elements of the inner dimension on
      uint32_t it = 0, tt = 0;                           // k-blocks / tiles so far
      bool ok = true;
      for (int q = pair; ok && q < items; q += pairs) {
        const Item im = item_of<MODE>(p, q);
        const bool a_mn = MODE == kProducts && im.product == kColGrad;
        const uint32_t idesc = a_mn ? make_idesc(Fmt<T>::idesc, kPairM, LM_BN, kBmn, 1) : make_idesc(Fmt<T>::idesc, kPairM, LM_BN, kBmn, 0);
        const uint64_t step_a = a_mn ? kStepMN : kStepK;
        const int k_steps = a_mn ? p.products.load[kColGrad].k_steps : LM_BK / 16;
        for (int t = 0; ok && t < im.count; ++t, ++tt) {
          const uint32_t b = tt & 1;
          // the accumulator still holds tile tt-2 until the epilogue warps have read it
          if (tt >= 2 && !mbar_wait<true>(&ctl->acc_free[b], ((tt >> 1) - 1) & 1, abort_flag)) { atomicOr(&ctl->fail_bits, (uint32_t)ULM_STATUS_TIMEOUT_SOFTMAX); ok = false; break; }
          fence_after_sync();
          for (int kb = im.kb0; kb < im.kb1; ++kb, ++it) {
            const uint32_t s = it % kStages;
            if (!mbar_wait(&ctl->full[s], (it / kStages) & 1, abort_flag)) { atomicOr(&ctl->fail_bits, (uint32_t)ULM_STATUS_TIMEOUT_LOAD); ok = false; break; }
            fence_after_sync();
            const uint32_t sa = smem_u32(stages + (size_t)s * kStage);
            const uint64_t da = a_mn ? make_sdesc_sw128_mn(sa, kAtom) : make_sdesc_sw128(sa);
            const uint64_t db = kBmn ? make_sdesc_sw128_mn(sa + kATile, kAtom) : make_sdesc_sw128(sa + kATile);
#pragma unroll
            for (int kk = 0; kk < LM_BK / 16; ++kk)
              if (MODE != kProducts || kk < k_steps) mma_ss_pair(tmem_base + b * LM_BN, da + kk * step_a, db + kk * (kBmn ? kStepMN : kStepK), idesc, (kb > im.kb0 || kk > 0) ? 1u : 0u);
            mma_commit_pair(&ctl->empty[s]);             // the stage is free in both CTAs once these MMAs have read it
          }
          if (ok) mma_commit_pair(&ctl->acc_full[b]);
        }
      }
    }
  } else {
    // ---------------- epilogue ----------------
    const int half = warp >> 2;                          // columns [128 half, 128 half + 128) of the tile
    const int r = ((warp & 3) << 5) | lane;              // row within the tile == TMEM lane
    const uint32_t t_row = tmem_base + ((uint32_t)((warp & 3) * 32) << 16);
    [[maybe_unused]] uint8_t* my_staging = staging + (size_t)warp * kStaging;
    [[maybe_unused]] float factor = 0.f;
    if constexpr (MODE == kProducts) factor = out_factor(p.products.out[kColGrad]);         // the same for both
    uint32_t tt = 0;
    bool ok = true;
    // the row's target column and, for G, its log-sum-exp; asked for an item ahead
    struct Row { int64_t target; float lse; };
    auto row_of = [&](int q) {
      Row w{-1, 0.f};
      if constexpr (MODE == kStats || MODE == kGrad) {
        const int64_t row = (int64_t)item_of<MODE>(p, q < items ? q : pair).mt * kPairM + rank * LM_BM + r;
        if (row < p.rows) {
          w.target = p.target[row];
          if (w.target == p.ignore_index || w.target >= p.V) w.target = -1;
          if constexpr (MODE == kGrad) w.lse = p.lse[row];
        }
      }
      return w;
    };
    [[maybe_unused]] Row next = row_of(pair);
    for (int q = pair; ok && q < items; q += pairs) {
      const Item im = item_of<MODE>(p, q);
      const int64_t grow = (int64_t)im.mt * kPairM + rank * LM_BM + r;
      [[maybe_unused]] const int row0 = (int)grow - lane;                        // the warp's first row
      [[maybe_unused]] float m = -INFINITY, ssum = 0.f;  // base-2 domain: m = max(z) * log2e
      [[maybe_unused]] const int tgt = next.target >= 0 ? (int)next.target : -1;
      [[maybe_unused]] const float lse = next.lse;
      if constexpr (MODE == kStats || MODE == kGrad) next = row_of(q + pairs);
      for (int t = 0; ok && t < im.count; ++t, ++tt) {
        const uint32_t b = tt & 1;
        const bool waited = __all_sync(0xffffffffu, mbar_wait(&ctl->acc_full[b], (tt >> 1) & 1, abort_flag));
        if (!waited && lane == 0) atomicOr(&ctl->fail_bits, (uint32_t)ULM_STATUS_TIMEOUT_MMA);
        if (!waited) { ok = false; break; }              // the whole warp; nothing below waits for another one
        fence_after_sync();
        const int col_tile = (im.nt + t) * LM_BN;
        // the thread's 128 columns at once, and the accumulator goes back before any of them is worked on
        uint32_t both[128];
#pragma unroll
        for (int c = 0; c < 128; c += 32) tmem_ld32(t_row + b * LM_BN + half * 128 + c, *reinterpret_cast<uint32_t(*)[32]>(&both[c]));
        tmem_wait_ld();
        fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive_peer(peer_smem(&ctl->acc_free[b], 0));
#pragma unroll
        for (int pass = 0; pass < 2; ++pass) {
          const int c_blk = half * 128 + pass * 64;      // first column of this pass within the tile
          uint32_t (&acc)[64] = *reinterpret_cast<uint32_t(*)[64]>(&both[64 * pass]);
          if constexpr (MODE == kStats) {
            const int col0 = col_tile + c_blk;
            if (col0 + 64 > p.V) {
#pragma unroll
              for (int c = 0; c < 64; ++c)
                if (col0 + c >= p.V) acc[c] = __float_as_uint(-INFINITY);
            }
            if ((unsigned)(tgt - col0) < 64u) {          // one block of one thread holds the row's target
              float z = 0.f;
#pragma unroll
              for (int c = 0; c < 64; ++c) z = tgt - col0 == c ? __uint_as_float(acc[c]) : z;
              p.z_target[grow] = z;
            }
            // four chains each for maximum and sum: two warps a scheduler do not hide the latency of one
            float mq[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int c = 0; c < 64; c += 2) mq[c >> 1 & 3] = fmax3(mq[c >> 1 & 3], __uint_as_float(acc[c]), __uint_as_float(acc[c + 1]));
            const float mx = fmax3(fmaxf(mq[0], mq[1]), mq[2], mq[3]);
            const float m_new = fmaxf(m, mx * kLog2e);
            if (m_new > -INFINITY) {
              ssum *= ex2(m - m_new);                    // 2^(-inf) = 0 on the first block
              const uint64_t log2e2 = f2_pack(kLog2e, kLog2e), nm2 = f2_pack(-m_new, -m_new);
              uint64_t sq[4] = {f2_pack(0.f, 0.f), f2_pack(0.f, 0.f), f2_pack(0.f, 0.f), f2_pack(0.f, 0.f)};
#pragma unroll
              for (int c = 0; c < 64; c += 2) {
                float e0, e1;
                f2_unpack(f2_fma(f2_pack(__uint_as_float(acc[c]), __uint_as_float(acc[c + 1])), log2e2, nm2), e0, e1);
                sq[c >> 1 & 3] = f2_add(sq[c >> 1 & 3], f2_pack(ex2(e0), ex2(e1)));
              }
              float s0, s1;
              f2_unpack(f2_add(f2_add(sq[0], sq[1]), f2_add(sq[2], sq[3])), s0, s1);
              ssum += s0 + s1;
              m = m_new;
            } else {                                     // nothing but -inf, or NaN, which fmaxf passes over
#pragma unroll
              for (int c = 0; c < 64; ++c)
                if (__uint_as_float(acc[c]) != __uint_as_float(acc[c])) ssum = __uint_as_float(acc[c]);
            }
          } else if constexpr (MODE == kGrad) {
            const int col0 = p.v0 + col_tile + c_blk;
            const float shift = (float)Fmt<T>::g_shift - lse * kLog2e;           // of the exponent
            const uint64_t log2e2 = f2_pack(kLog2e, kLog2e), shift2 = f2_pack(shift, shift);
            uint32_t pk[32];
            // p - 1 of the target, which may be far below an ulp of p: from the exponent by itself, without the rounding of lse log2e that
            // the other columns' share, and not as a difference
            float g_target = 0.f;
            if ((unsigned)(tgt - col0) < 64u) {
              float z = 0.f;
#pragma unroll
              for (int c = 0; c < 64; ++c) z = tgt - col0 == c ? __uint_as_float(acc[c]) : z;
              const float hi = lse * kLog2e, lo = fmaf(lse, kLog2e, -hi);
              g_target = (float)(1 << Fmt<T>::g_shift) * expm1f((fmaf(z, kLog2e, -hi) - lo) * kLn2);
            }
#pragma unroll
            for (int c = 0; c < 64; c += 2) {
              float g0, g1;
              f2_unpack(f2_fma(f2_pack(__uint_as_float(acc[c]), __uint_as_float(acc[c + 1])), log2e2, shift2), g0, g1);
              acc[c] = __float_as_uint(ex2(g0));
              acc[c + 1] = __float_as_uint(ex2(g1));
            }
            if ((unsigned)(tgt - col0) < 64u) {
#pragma unroll
              for (int c = 0; c < 64; ++c)
                if (tgt - col0 == c) acc[c] = __float_as_uint(g_target);
            }
#pragma unroll
            for (int c = 0; c < 64; c += 2) pk[c >> 1] = tgt >= 0 ? Cvt<T>::pack2(__uint_as_float(acc[c]), __uint_as_float(acc[c + 1])) : 0u;
            if (col0 + 64 > p.V) {                       // the workspace's columns past the vocabulary are zero
#pragma unroll
              for (int c = 0; c < 64; c += 2) {
                if (col0 + c >= p.V) pk[c >> 1] = 0u;
                else if (col0 + c + 1 >= p.V) pk[c >> 1] &= 0xffffu;
              }
            }
            if (col_tile + c_blk < p.g_cols && row0 < p.rows) store_block<false>(&maps.out[0], my_staging, lane, pk, 0, row0, (col_tile + c_blk) >> 6);
          } else {
            const int col = col_tile + c_blk;
            const Out& out = p.products.out[im.product];
            const CUtensorMap* tmOut = &maps.out[im.product];
            if (im.slot >= 0) {
              if (row0 < out.rows) store_f32<false>(&maps.slots, my_staging, lane, acc, 1.f, c_blk, LM_BN, im.slot * kPairM + (int)rank * LM_BM + (warp & 3) * 32);
            } else if (col < out.cols && row0 < out.rows) {
              if (out.is_f32 && out.prev) {
                store_f32<true>(tmOut, my_staging, lane, acc, factor, col, out.cols, row0);
              } else if (out.is_f32) {
                store_f32<false>(tmOut, my_staging, lane, acc, factor, col, out.cols, row0);
              } else if (out.prev) {
                add_and_round<T>(out, factor, grow, col, acc);
              } else {
                uint32_t pk[32];
#pragma unroll
                for (int c = 0; c < 64; c += 2) pk[c >> 1] = Cvt<T>::pack2(factor * __uint_as_float(acc[c]), factor * __uint_as_float(acc[c + 1]));
                store_block<false>(tmOut, my_staging, lane, pk, col, row0);
              }
            }
          }
        }
      }
      if constexpr (MODE == kStats) {
        if (!ok) break;
        if (grow < p.rows) {                             // [row][group][half]: the finishing kernel merges a row's pairs
          const int64_t o = (grow * ((p.w.n_nt + p.w.group - 1) / p.w.group) + im.nt / p.w.group) * 2 + half;
          p.part_m[o] = m;
          p.part_s[o] = ssum;
        }
      }
    }
    if (MODE != kStats && lane == 0) bulk_wait0();       // our stores must be complete before the CTA ends
  }

  fence_before_sync();
  __syncthreads();
  // Some warp has given up: this CTA's copies and products in flight land before the pair's shared memory and TMEM go away.  The
  // copies' barrier is rank 0's and may lack the other CTA's half, so it is time that is waited for: a thousand times what a load
  // takes.  Here, where no warp can issue or give up any more: the producer may have issued its last copies before another warp gave up.
  if (*abort_flag && threadIdx.x == 0) {
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 1000000ull) {}
  }
  __syncwarp();
  cluster_sync();                                        // neither CTA leaves while the other's products or arrivals may reach it
  if (warp == kEpiWarps + 1) tmem_dealloc_pair(tmem_base, 512);
  if (threadIdx.x == 0 && ctl->fail_bits && p.status) atomicOr(p.status, ctl->fail_bits);
}

// The tiles that were cut: out = factor * (sum of the tile's slots, in order) (+ prev).  A CTA takes eight rows of a tile, a
// thread eight columns.
template <typename T>
__global__ void __launch_bounds__(256)
streamed_ce_join_kernel(const Products p) {
  grid_dependents_go();
  grid_dependency_wait();
  const int of_dw = p.w[kColGrad].split > 1 ? p.w[kColGrad].rest : 0;
  const int which = (int)blockIdx.x < of_dw ? kColGrad : kRowGrad, j = (int)blockIdx.x - (which == kColGrad ? 0 : of_dw);
  const Work& w = p.w[which];
  const Out& o = p.out[which];
  const int t = w.whole + j, mt = t / w.n_nt, nt = t - mt * w.n_nt;
  const int r = blockIdx.y * 8 + (threadIdx.x >> 5), c = (threadIdx.x & 31) * 8;
  const int64_t row = (int64_t)mt * kPairM + r;
  const int col = nt * LM_BN + c;
  if (row >= o.rows || col >= o.cols) return;
  const float* s = o.slots + (p.slot0[which] + (int64_t)j * w.split) * kSlot + r * LM_BN + c;
  const float factor = out_factor(o);
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = 0.f;
#pragma unroll 8
  for (int k = 0; k < w.split; ++k, s += kSlot) {
    const float4 a = *reinterpret_cast<const float4*>(s), b = *reinterpret_cast<const float4*>(s + 4);
    v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
    v[4] += b.x; v[5] += b.y; v[6] += b.z; v[7] += b.w;
  }
  const int64_t at = row * o.ld + col;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = factor * v[i] + (o.prev ? o.prev[at + i] : 0.f);
  if (o.is_f32) {
    float4* q = reinterpret_cast<float4*>(static_cast<float*>(o.out) + at);
    q[0] = make_float4(v[0], v[1], v[2], v[3]);
    q[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    *reinterpret_cast<uint4*>(static_cast<T*>(o.out) + at) =
        make_uint4(Cvt<T>::pack2(v[0], v[1]), Cvt<T>::pack2(v[2], v[3]), Cvt<T>::pack2(v[4], v[5]), Cvt<T>::pack2(v[6], v[7]));
  }
}

// lse[r] from the per-group (max, sum) pairs, loss[r] = lse[r] - z_target[r] (0 on ignored rows; loss holds z_target on entry): a
// warp per row.  For the loss the target's logit is formed once more here, by fp32 fused multiply-adds, and takes the place of the tensor
// core's in the sum and in the difference: their additions round towards zero, 1e-6 of a logit at d = 1024 (-1.8e-5 +- 0.3e-5 at
// 17, -0.3e-5 at d = 128), which stays in the mean (loss against 64 bits, d = 1024: 1.0e-6 -> 0.45e-6).  2 d bytes of H and W a row.  The CTA that finishes last adds up the rows' losses, in fp64 and a fixed order: mean = sum / n and inv = 1 / n,
// n = *denom_dev, denom if that is positive, or the number of targets that are not ignore_index (at least 1).
struct Mean {
  const float* denom_dev;
  float denom;
  float *mean, *inv;
  uint32_t* done;                                        // CTAs that have finished: zeroed by the statistics kernel
};
struct Operands { const void *h, *w; int64_t h_stride, w_stride; int d; };
template <typename T>
__global__ void __launch_bounds__(256)
streamed_ce_finish_kernel(const float* part_m, const float* part_s, int n_parts, const int64_t* target,
                          int64_t ignore_index, int V, float* lse, float* loss, int64_t rows, const Operands op, const Mean mean) {
  __shared__ double s_sum[8];
  __shared__ int s_n[8];
  __shared__ uint32_t s_before;
  grid_dependents_go();
  grid_dependency_wait();
  const int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (r < rows) {
    const int64_t t = target[r];
    const float z_tensor = loss[r];
    const bool counts = t != ignore_index && t >= 0 && t < V;
    float m = -INFINITY, s = 0.f;
#pragma unroll 4
    for (int i = lane; i < n_parts; i += 32) {
      const float mi = part_m[r * n_parts + i], si = part_s[r * n_parts + i], mn = fmaxf(m, mi);
      // a group of nothing but -inf has the sum 0; of NaN, NaN
      s = (m > -INFINITY ? s * exp2f(m - mn) : s) + (mi > -INFINITY ? si * exp2f(mi - mn) : si);
      m = mn;
    }
    const float lane_m = m;
    m = warp_max(m);
    s = warp_sum(lane_m > -INFINITY ? s * exp2f(lane_m - m) : s);
    float z = 0.f;
    if (counts) {
      const T *h = static_cast<const T*>(op.h) + r * op.h_stride, *w = static_cast<const T*>(op.w) + t * op.w_stride;
      float z0 = 0.f, z1 = 0.f;
      for (int k = lane * 8; k < op.d; k += 256) {
        const uint4 a = *reinterpret_cast<const uint4*>(h + k), b = *reinterpret_cast<const uint4*>(w + k);
        const uint32_t au[4] = {a.x, a.y, a.z, a.w}, bu[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 x = Cvt<T>::unpack2(au[j]), y = Cvt<T>::unpack2(bu[j]);
          z0 = fmaf(x.x, y.x, z0);
          z1 = fmaf(x.y, y.y, z1);
        }
      }
      z = warp_sum(z0 + z1);
    }
    if (lane == 0) {
      // the log-sum-exp of the very logits that the backward forms again: the target's probability is their ratio, and what
      // it lacks of 1 may be far below the two logits' difference.  In fp64 up to one rounding
      lse[r] = (float)(((double)m + (double)log2f(s)) / (double)kLog2e);
      if (counts) s += exp2f(fmaf(z, kLog2e, -m)) - exp2f(fmaf(z_tensor, kLog2e, -m));
      const float log2_s = log2f(s);
      // lse - z, with the large parts subtracted first and exactly: their difference is as small as the loss
      const float l = (fmaf(-z, kLog2e, m) + log2_s) * kLn2;
      loss[r] = !counts || l < 0.f ? 0.f : l;             // the sum may round below its largest term; NaN stays
    }
  }
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) s_before = atomicAdd(mean.done, 1u);
  __syncthreads();
  if (s_before != gridDim.x - 1) return;
  __threadfence();
  double sum = 0.;
  int n = 0;
  const bool count = !mean.denom_dev && !(mean.denom > 0.f);
#pragma unroll 4
  for (int64_t i = threadIdx.x; i < rows; i += 256) {
    sum += __ldcg(loss + i);
    if (count) n += target[i] != ignore_index;
  }
  sum = warp_sum(sum);
  n = __reduce_add_sync(0xffffffffu, n);
  if (lane == 0) { s_sum[threadIdx.x >> 5] = sum; s_n[threadIdx.x >> 5] = n; }
  __syncthreads();
  if (threadIdx.x) return;
  for (int w = 1; w < 8; ++w) { sum += s_sum[w]; n += s_n[w]; }
  const float d = mean.denom_dev ? *mean.denom_dev : count ? (float)(n > 0 ? n : 1) : mean.denom;
  *mean.mean = (float)(sum / d);
  *mean.inv = 1.f / d;
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
// The rest tiles' split: the fewest rounds over the SMs, in k-blocks, an item's own cost (fill, epilogue, its slot's way
// through memory) being worth about 12 of them; stretches of at least 4 k-blocks.
Work product_work(int64_t m, int64_t n, int64_t k) {
  Work w{};
  w.n_mt = (int)((m + kPairM - 1) / kPairM);
  w.n_nt = (int)((n + LM_BN - 1) / LM_BN);
  w.n_kb = (int)((k + LM_BK - 1) / LM_BK);
  const int64_t tiles = (int64_t)w.n_mt * w.n_nt;
  w.whole = (int)(tiles / kPairs * kPairs);
  w.rest = (int)(tiles - w.whole);
  w.split = 1;
  int64_t best = INT64_MAX;
  for (int s = 1; s <= 64 && w.rest && (s == 1 || w.n_kb / s >= 4); ++s) {
    const int64_t rounds = ((int64_t)w.rest * s + kPairs - 1) / kPairs, cost = rounds * ((w.n_kb + s - 1) / s + 12) + (s > 1 ? 12 : 0);
    if (cost < best) { best = cost; w.split = s; }
  }
  return w;
}
int n_slots(const Work& w) { return w.split > 1 ? w.rest * w.split : 0; }

template <typename T, int MODE>
int launch(const Maps& maps, const Params& p, int device, cudaStream_t st, const char* who) {
  static std::atomic<bool> attr_set[kMaxDevices];
  auto kern = streamed_ce_kernel<T, MODE>;
  if (int rc = ensure_smem_attr(kern, smem_bytes(MODE), device, attr_set, who)) return rc;
  const int items = n_items<MODE>(p), grid = 2 * (items < kPairs ? items : kPairs);
  return launch_dependent(who, kern, grid, kThreads, smem_bytes(MODE), st, maps, p);
}
// Both products and, where tiles were cut, their sums
template <typename T>
int launch_products(Maps& maps, Params& p, float* slots, int dtype, int device, cudaStream_t st, const char* who) {
  Products& m = p.products;
  int rc, joined = 0, n = 0;
  int64_t most_rows = 0;
  for (int i = 0; i < kNumProducts; ++i) {
    Out& o = m.out[i];
    m.slot0[i] = n;
    o.slots = slots;
    if (!o.out) continue;
    if ((rc = encode_matrix_map(&maps.out[i], o.out, o.is_f32 ? (int)ULM_F32 : dtype, o.rows, o.cols, o.ld, 32, who))) return rc;
    if (m.w[i].split > 1) {
      n += n_slots(m.w[i]);
      joined += m.w[i].rest;
      if (o.rows > most_rows) most_rows = o.rows;
    }
  }
  if (n && (rc = encode_matrix_map(&maps.slots, slots, ULM_F32, (int64_t)n * kPairM, LM_BN, LM_BN, 32, who))) return rc;
  rc = launch<T, kProducts>(maps, p, device, st, who);
  if (rc || !joined) return rc;
  return launch_dependent(who, streamed_ce_join_kernel<T>, dim3(joined, (unsigned)((most_rows < kPairM ? most_rows : kPairM) + 7) / 8), 256, 0, st, m);
}

int check_args(const ulm_streamed_ce_args* a, const char* who) {
  if (!a) return fail(ULM_ERR_ARG, "%s: null args", who);
  if (a->dtype != ULM_F16 && a->dtype != ULM_BF16) return fail(ULM_ERR_ARG, "%s: dtype must be fp16 or bf16", who);
  if (a->rows < 0 || a->V <= 0 || a->d <= 0 || a->d % 8) return fail(ULM_ERR_ARG, "%s: need rows >= 0, V > 0, d a positive multiple of 8", who);
  // tile numbers and TMA coordinates are 32-bit
  if (a->rows > (1 << 30) || a->V > (1 << 30) || a->d > (1 << 20)) return fail(ULM_ERR_TOO_LARGE, "%s: too many rows or columns", who);
  if (((a->rows + 127) / 128) * (((int64_t)a->V + 255) / 256) > 0x7fffffffLL) return fail(ULM_ERR_TOO_LARGE, "%s: too many output tiles", who);
  if (a->rows == 0) return ULM_OK;
  if (!a->h || !a->w || !a->target || !a->lse) return fail(ULM_ERR_ARG, "%s: null tensor", who);
  return ULM_OK;
}
bool ok_out(const void* p, int64_t stride, int d) { return !(reinterpret_cast<uintptr_t>(p) & 15) && stride % 8 == 0 && stride >= d; }

// rows of a box of A where A's rows are the tensor's: all there are, if they fit
int a_box(int64_t rows) { return rows < LM_BM ? (int)(rows + 7) / 8 * 8 : LM_BM; }
// K16 steps of dW's k-blocks, which go over the rows
int col_steps(int64_t rows) { return rows < LM_BK ? (int)(rows + 15) / 16 : LM_BK / 16; }
Load load_of(int64_t rows, bool col_grad) {
  Load l;
  l.k_steps = col_grad ? col_steps(rows) : LM_BK / 16;
  l.a_bytes[0] = col_grad ? kATile / 4 * l.k_steps : (uint32_t)a_box(rows) * LM_BK * 2;
  l.a_bytes[1] = !col_grad && rows <= LM_BM ? 0u : l.a_bytes[0];
  l.b_bytes = col_grad ? kBTile / 4 * l.k_steps : kBTile;
  return l;
}

Params common_params(const ulm_streamed_ce_args* a) {
  Params p{};
  p.rows = a->rows; p.V = a->V; p.target = a->target; p.ignore_index = a->ignore_index; p.status = a->status_dev;
  p.load = load_of(a->rows, false);
  return p;
}

Work stats_work(int64_t rows, int V, int d) {
  Work w{};
  w.n_mt = (int)((rows + kPairM - 1) / kPairM);
  w.n_nt = (V + LM_BN - 1) / LM_BN;
  w.n_kb = (d + LM_BK - 1) / LM_BK;
  w.group = lm_group_tiles(w.n_mt, w.n_nt, kPairs);
  return w;
}

template <typename T>
int forward(const ulm_streamed_ce_args* a, int device, const char* who) {
  Maps maps{};
  if (int rc = encode_matrix_map(&maps.a[0], a->h, a->dtype, a->rows, a->d, a->h_stride, a_box(a->rows), who)) return rc;
  if (int rc = encode_matrix_map(&maps.b[0], a->w, a->dtype, a->V, a->d, a->w_stride, kBRows, who)) return rc;
  Params p = common_params(a);
  p.w = stats_work(a->rows, a->V, a->d);
  const int parts = 2 * ((p.w.n_nt + p.w.group - 1) / p.w.group);
  p.part_m = a->scratch; p.part_s = a->scratch + a->rows * parts; p.z_target = a->loss;
  p.done = reinterpret_cast<uint32_t*>(a->scratch + 2 * a->rows * parts);
  cudaStream_t st = (cudaStream_t)a->stream;
  if (int rc = launch<T, kStats>(maps, p, device, st, who)) return rc;
  const Mean mean{a->denom_dev, a->denom, a->mean, a->inv, p.done};
  const Operands op{a->h, a->w, a->h_stride, a->w_stride, a->d};
  return launch_dependent(who, streamed_ce_finish_kernel<T>, (unsigned)((a->rows + 7) / 8), 256, 0, st, p.part_m, p.part_s, parts, a->target, a->ignore_index, a->V,
                          a->lse, a->loss, a->rows, op, mean);
}

// G's workspace: blocks of 64 columns, [block][row][64], so that every box that is stored or loaded is one stretch of memory.
// As a row-major matrix, whose boxes are 128-byte pieces of far-apart rows, the whole op took 0.5 % longer (32768 x 768 x 32000).
int64_t g_blocks(int64_t piece) { return (piece + 63) / 64; }

template <typename T>
int backward(const ulm_streamed_ce_args* a, const ulm_streamed_ce_grads* g, int device, const char* who) {
  cudaStream_t st = (cudaStream_t)a->stream;
  Maps logits{}, products{};                             // H and W for z; G and H, G and W for the products: K-major and MN-major boxes
  int rc;
  const int steps = 16 * col_steps(a->rows), box = a_box(a->rows);
  if ((rc = encode_matrix_map(&logits.a[0], a->h, a->dtype, a->rows, a->d, a->h_stride, box, who))) return rc;
  if ((rc = encode_matrix_map(&logits.b[0], a->w, a->dtype, a->V, a->d, a->w_stride, kBRows, who))) return rc;
  if ((rc = encode_matrix_map(&products.b[kColGrad], a->h, a->dtype, a->rows, a->d, a->h_stride, steps, who))) return rc;
  if ((rc = encode_matrix_map(&products.b[kRowGrad], a->w, a->dtype, a->V, a->d, a->w_stride, 64, who))) return rc;
  for (int64_t v0 = 0; v0 < a->V; v0 += g->piece) {
    const int64_t n = a->V - v0 < g->piece ? a->V - v0 : g->piece;
    auto g_map = [&](CUtensorMap* m, int box_rows) {
      return encode_bhsd_map(m, g->workspace, a->dtype, 1, (int)g_blocks(n), (int)a->rows, 0, a->rows * 64, 64, box_rows, who);
    };
    if ((rc = g_map(&logits.out[0], 32)) || (rc = g_map(&products.a[kColGrad], steps)) || (rc = g_map(&products.a[kRowGrad], box))) return rc;
    Params p = common_params(a);
    p.v0 = (int)v0;
    p.lse = a->lse;
    p.g_cols = (int)g_blocks(n) * 64;
    p.w = stats_work(a->rows, (int)n, a->d);
    if ((rc = launch<T, kGrad>(logits, p, device, st, who))) return rc;
    Products& m = p.products;
    for (Out& o : m.out) {
      o.factor_dev = g->factor_dev;
      o.factor2_dev = g->factor2_dev;
      o.factor = 1.f / (float)(1 << Fmt<T>::g_shift);
      o.cols = a->d;
    }
    if (g->dw) {
      m.w[kColGrad] = product_work(n, a->d, a->rows);
      m.load[kColGrad] = load_of(a->rows, true);
      Out& o = m.out[kColGrad];
      o.ld = g->dw_stride; o.rows = n; o.is_f32 = g->dw_f32;
      o.out = g->dw_f32 ? (void*)((float*)g->dw + v0 * g->dw_stride) : (void*)((T*)g->dw + v0 * g->dw_stride);
      o.prev = g->dw_add ? (const float*)o.out : nullptr;
    }
    if (g->dh) {
      const bool first = v0 == 0, last = v0 + n >= a->V;
      m.w[kRowGrad] = product_work(a->rows, a->d, n);
      m.load[kRowGrad] = load_of(a->rows, false);
      Out& o = m.out[kRowGrad];
      o.ld = a->d; o.rows = a->rows; o.is_f32 = !last;   // dh and dh_sum are dense
      o.out = last ? g->dh : (void*)g->dh_sum;
      o.prev = first ? nullptr : g->dh_sum;
    }
    if ((rc = launch_products<T>(products, p, g->slots, a->dtype, device, st, who))) return rc;
  }
  return ULM_OK;
}

}  // namespace
}  // namespace ulm

extern "C" int64_t ulm_streamed_ce_scratch(int64_t rows, int32_t V, int32_t d) {
  if (rows <= 0 || V <= 0 || d <= 0) return 0;
  const ulm::Work w = ulm::stats_work(rows, V, d);
  return rows * 4 * ((w.n_nt + w.group - 1) / w.group) + 1;
}

extern "C" int64_t ulm_streamed_ce_workspace(int64_t rows, int32_t V, int64_t piece) {
  return rows * 64 * ulm::g_blocks(piece < V ? piece : V);
}

extern "C" int64_t ulm_streamed_ce_slots(int64_t rows, int32_t V, int32_t d, int64_t piece, int32_t want_dh, int32_t want_dw) {
  using namespace ulm;
  if (rows <= 0 || V <= 0 || d <= 0 || piece <= 0) return 0;
  int64_t most = 0;
  const int64_t tail = V % piece ? V % piece : piece;    // the pieces have two sizes at most
  for (int64_t n : {piece < V ? piece : (int64_t)V, tail < V ? tail : (int64_t)V})
    most = std::max<int64_t>(most, (want_dw ? n_slots(product_work(n, d, rows)) : 0) + (want_dh ? n_slots(product_work(rows, d, n)) : 0));
  return most * kSlot;
}

extern "C" int ulm_streamed_ce_fwd(const ulm_streamed_ce_args* a) {
  using namespace ulm;
  const char* who = "ulm_streamed_ce_fwd";
  int rc = check_args(a, who);
  if (rc || a->rows == 0) return rc;
  if (!a->loss || !a->scratch || !a->mean || !a->inv) return fail(ULM_ERR_ARG, "%s: null tensor", who);
  DeviceScope scope(a->h, who);
  if (scope.rc) return scope.rc;
  return a->dtype == ULM_BF16 ? forward<__nv_bfloat16>(a, scope.device, who) : forward<__half>(a, scope.device, who);
}

extern "C" int ulm_streamed_ce_bwd(const ulm_streamed_ce_args* a, const ulm_streamed_ce_grads* g) {
  using namespace ulm;
  const char* who = "ulm_streamed_ce_bwd";
  int rc = check_args(a, who);
  if (rc) return rc;
  if (!g) return fail(ULM_ERR_ARG, "%s: null grads", who);
  if (g->piece <= 0 || g->piece % LM_BN) return fail(ULM_ERR_ARG, "%s: piece must be a positive multiple of %d columns", who, LM_BN);
  if (a->rows == 0 || (!g->dh && !g->dw)) return ULM_OK;
  if (!g->factor_dev || !g->workspace || (g->dh && g->piece < a->V && !g->dh_sum)) return fail(ULM_ERR_ARG, "%s: null tensor", who);
  if (!g->slots && ulm_streamed_ce_slots(a->rows, a->V, a->d, g->piece, g->dh != nullptr, g->dw != nullptr) > 0) return fail(ULM_ERR_ARG, "%s: null slots", who);
  if ((g->dw && !ok_out(g->dw, g->dw_stride, a->d)) || (g->dh && !ok_out(g->dh, a->d, a->d)) || (reinterpret_cast<uintptr_t>(g->dh_sum) & 15) ||
      (reinterpret_cast<uintptr_t>(g->slots) & 15))
    return fail(ULM_ERR_ARG, "%s: gradients must be 16-byte aligned, dw's row stride a multiple of 8 and at least d", who);
  if (g->dw_add && !g->dw_f32) return fail(ULM_ERR_ARG, "%s: only an fp32 dw can be added to", who);
  DeviceScope scope(a->h, who);
  if (scope.rc) return scope.rc;
  return a->dtype == ULM_BF16 ? backward<__nv_bfloat16>(a, g, scope.device, who) : backward<__half>(a, g, scope.device, who);
}
