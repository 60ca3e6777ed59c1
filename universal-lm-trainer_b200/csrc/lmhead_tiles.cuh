// How the lm-head products are cut into output tiles of 128 rows x 256 vocabulary columns, and those into work items.
#pragma once

#include "common.cuh"

namespace ulm {
namespace {

constexpr int LM_BM = 128, LM_BN = 256, LM_BK = 64;
constexpr int kLmGroupTiles = 25;                      // column tiles per work item (upper bound)

// Column tiles per work item: the count whose rounds of items over the workers (SMs, or pairs of them) take the fewest tile times, an item's own
// cost (pipeline fill, statistics) being worth about a quarter of a tile.  At 32768 x 32000 that is 5 (220 tile times,
// 216 ideal; the fixed 25 of before took 225); with 2048 rows x 4096 columns, 1 instead of 16: 256 items on 148 SMs
// where 16 SMs had one each.
inline int lm_group_tiles(int64_t n_rb, int64_t n_ct, int workers) {
  int best = 1;
  int64_t best_cost = INT64_MAX;
  for (int want = 1; want <= kLmGroupTiles; ++want) {
    const int64_t groups = (n_ct + want - 1) / want, tiles = (n_ct + groups - 1) / groups;
    const int64_t cost = ((n_rb * groups + workers - 1) / workers) * (4 * tiles + 1);
    if (cost < best_cost) { best_cost = cost; best = (int)tiles; }
  }
  return best;
}

inline int lm_group_tiles(int64_t rows, int V) { return lm_group_tiles((rows + LM_BM - 1) / LM_BM, ((int64_t)V + LM_BN - 1) / LM_BN, kNumSMs); }

struct LmItems {
  int n_rb, n_ct, n_groups, group_tiles;
  __host__ __device__ LmItems(int64_t rows, int V, int tiles) {
    n_rb = (int)((rows + LM_BM - 1) / LM_BM);
    n_ct = (V + LM_BN - 1) / LM_BN;
    group_tiles = tiles;
    n_groups = (n_ct + tiles - 1) / tiles;
  }
  __host__ __device__ int n_items() const { return n_rb * n_groups; }
  // all CTAs are on one column group at a time: its W tiles are read from L2 by everyone
  __device__ void decode(int idx, int& rb, int& g, int& ct0, int& nct) const {
    g = idx / n_rb;
    rb = idx - g * n_rb;
    ct0 = g * group_tiles;
    nct = n_ct - ct0 < group_tiles ? n_ct - ct0 : group_tiles;
  }
};

}  // namespace
}  // namespace ulm
