// Which output tiles each pair of CTAs of linear_pair.cu makes, in which order. Computed from the sizes alone (no counters in memory),
// so launches share nothing; plain arithmetic, which the host's compiler takes as well.
//
// Tiles have HALVES * 256 rows (j) x 256 columns (i). With HALVES == 1 a launch takes one product or two (the backward pass): the tiles
// of the product with the longer r, product 0, come first; pairs that get one tile of it less than others start on product 1
// meanwhile, and the rest of its tiles are dealt out in turn. With HALVES == 2 there is one product. A launch of one product has
// it as product 1. Tiles of product 1 that would not fill a round of pairs are cut into smaller ones.
#pragma once

#include <algorithm>
#include <cstdint>

#ifdef __CUDACC__
#define TVB_SCHEDULE_CALL __host__ __device__
#else
#define TVB_SCHEDULE_CALL
#endif

namespace tvb {

constexpr int kHalfJ = 256, kTileI = 256;

// One product's part: its output is J x I in tiles_j x tiles_i tiles, with `blocks` steps of r each.
struct PairExtent {
  int I, J, blocks, tiles, tiles_i, tiles_j;
};

struct PairPlan {
  int extra;        // tiles of product 1 that a pair with fewer tiles of product 0 takes first
  int light_first;  // which pairs come first when the rest of product 1 is dealt out
  int whole;        // tiles of product 1 that are not cut; the others become cut tiles of 256 rows x cut_cols columns
  int cut_cols;
};

struct PairTile {
  int product, row, col, cols, halves;
};

// The plan for `pairs` pairs; returns how many of them to launch. (HALVES == 2: e0 is empty.)
template <int HALVES>
int plan_pairs(const PairExtent& e0, const PairExtent& e1, int pairs, PairPlan* plan) {
  *plan = PairPlan{};
  int light = 0;
  if (HALVES == 1 && e0.tiles % pairs != 0) {
    const int a = e0.blocks, b = e1.blocks;
    light = pairs - e0.tiles % pairs;
    plan->extra = (2 * a + b) / (2 * b);  // a / b, rounded
    plan->light_first = static_cast<int64_t>(plan->extra) * b < a;
    plan->extra = std::min(plan->extra, (e1.tiles + light - 1) / light);  // (no more than there are)
  }
  // Tiles of product 1 beyond whole rounds of pairs: a round of tiles as they are, or rounds of smaller ones. Relative costs of a
  // step (512 or 256 rows x 256 columns, 256 x 128), by the bytes an SM stages: 48, 32 and 24 KB.
  const int early = static_cast<int>(std::min<int64_t>(static_cast<int64_t>(light) * plan->extra, e1.tiles)), rest = (e1.tiles - early) % pairs;
  const int64_t uncut = HALVES == 2 ? 48 : 32, half = (static_cast<int64_t>(HALVES) * rest + pairs - 1) / pairs * 32,
                quarter = (2ll * HALVES * rest + pairs - 1) / pairs * 24;
  plan->cut_cols = kTileI;
  plan->whole = e1.tiles;
  if (rest != 0 && std::min(half, quarter) < uncut) {
    plan->whole -= rest;
    plan->cut_cols = half <= quarter ? kTileI : kTileI / 2;
  }
  const int per_cut = HALVES * kTileI / plan->cut_cols;
  const int64_t tiles = static_cast<int64_t>(e0.tiles) + plan->whole + static_cast<int64_t>(e1.tiles - plan->whole) * per_cut;
  return static_cast<int>(std::min<int64_t>(pairs, tiles));
}

// Walks the tiles of one pair: its tiles of product 0, its share of product 1, its share of what was cut.
template <int HALVES>
struct PairSchedule {
  static constexpr int kTileJ = HALVES * kHalfJ, kBand = 16 / HALVES;  // (tile rows per band of the tile order)
  int pair, pairs, at, heavy, rank_among, order, stage;
  bool is_light;
  TVB_SCHEDULE_CALL PairSchedule(const PairPlan& plan, const PairExtent& e0, int pair_, int pairs_) : pair(pair_), pairs(pairs_) {
    if constexpr (HALVES == 1) {
      heavy = e0.tiles % pairs;  // pairs 0 ... heavy - 1 have one tile of product 0 more than the others
      is_light = heavy != 0 && pair >= heavy;
      rank_among = is_light ? pair - heavy : pair;
      order = heavy != 0 && plan.light_first ? (is_light ? rank_among : pairs - heavy + pair) : pair;
      stage = 0;
    } else {
      order = pair;
      stage = 2;
    }
    at = pair;
  }
  TVB_SCHEDULE_CALL static void place(const PairExtent& d, int index, PairTile& t) {
    const int per_band = kBand * d.tiles_i, b = index / per_band, first = b * kBand;
    const int rows = d.tiles_j - first < kBand ? d.tiles_j - first : kBand;
    const int r = index - b * per_band;
    t.row = (first + r % rows) * kTileJ;
    t.col = r / rows * kTileI;
    t.cols = kTileI;
    t.halves = HALVES == 2 && t.row + kHalfJ < d.J ? 2 : 1;
  }
  TVB_SCHEDULE_CALL bool next(const PairPlan& plan, const PairExtent& e0, const PairExtent& e1, PairTile& t) {
    for (;;) {
      t.product = 1;
      if constexpr (HALVES == 1) {
        const int light = heavy != 0 ? pairs - heavy : 0, early = light * plan.extra;
        if (stage == 0) {
          if (at < e0.tiles) {
            t.product = 0;
            place(e0, at, t);
            at += pairs;
            return true;
          }
          stage = 1;
          at = rank_among;
        }
        if (stage == 1) {
          if (is_light && at < early && at < plan.whole) {
            place(e1, at, t);
            at += light;
            return true;
          }
          stage = 2;
          at = early + order;
        }
      }
      if (stage == 2) {
        if (at < plan.whole) {
          place(e1, at, t);
          at += pairs;
          return true;
        }
        stage = 3;
        at = order;
      }
      const int per_half = kTileI / plan.cut_cols, per_tile = HALVES * per_half;
      const int index = plan.whole + at / per_tile, sub = at % per_tile;
      if (index >= e1.tiles) return false;
      at += pairs;
      place(e1, index, t);
      t.row += sub / per_half * kHalfJ;
      t.col += sub % per_half * plan.cut_cols;
      t.cols = plan.cut_cols;
      t.halves = 1;
      if (t.row < e1.J && t.col < e1.I) return true;  // (a cut tile may lie outside altogether)
    }
  }
};

}  // namespace tvb
