// The choice of tiles of the matrix-core GEMMs on lists of 64-, 128- and 256-row
// tiles (host side).
#pragma once

#include "mfma_tile.h"

namespace astrai_moe {
namespace {

// Which tiles a GEMM takes on a list of 128- or 256-row tiles: the list's own
// with 256 columns (gate/up: 128 of each), or, where those leave compute units
// idle, 128 rows by 128 columns, and on a 256-row list also 128 by 256.
// (64-row lists: 64 by 128.)
enum class Tiles { kList, kHalves, kNarrow, kNarrowHalves, kNarrowMid };

// A GEMM of few tiles takes rounds of its compute units times a tile's K steps,
// however few the tiles of the last round: 1.4 us a step of a 256 x 256 tile,
// 1.07 of 128 x 256, 0.83 of 64 x 256, 0.71 of 128 x 128, 0.55 of 64 x 128
// (measured; the small tiles pay more per flop). The others are taken where
// this promises a tenth under even routing and loses no more than a twentieth up
// to a skewed one, since a few row tiles more can cost a whole round of the
// smaller tiles (D 4096, F 14336, 8 experts, top-2, 256 tokens, 128-row list: a
// layer 559 us against 609 evenly routed, and 670 against 601 skewed); only within
// kFewRounds rounds of the list's own tiles, past which the shares are even and
// the memory system decides. A last round that the 256-row down GEMM splits
// along K (SplitWalk) counts the share of a round that its slices take and their
// reduction.
// Measured, us, a down GEMM of the list's tiles / the ones taken:
// - 8 experts, top-2, D 1000, F 2664, 130 to 375 rows an expert 50 / 31 to 58 /
//   33, and 9 of 500 rows 59 / 50 (halves); D 512, F 1024, 130 to 768 rows 23 / 14
//   to 26 / 15 (gate/up 17 / 13 to 19 / 14.5);
// - 16 experts, top-4, D 704, F 576, 64 to 512 rows 12 / 10 to 21 / 17 (gate/up
//   21 / 17.5 at 130 to 256); D 2048, F 1408, 64 rows 27 / 20, 130 37 / 29 (halves),
//   256 (a third more row tiles than places in a round) 42 / 44 if taken;
// - one expert, D 4096, F 14336, 512 rows 180 / 127, 1024 191 / 141; D 2048, F 5632,
//   1500 rows 81 / 55, 300 rows (64-row list) 73 / 35.
constexpr double kFewRounds = 2.0;
struct Pick {
  Tiles tiles;
  double us_per_step;  // rounds times a step's time
};
Pick pick_tiles(const RowCounts& rows, int block_m, int64_t k, int64_t n, bool gate_up) {
  const bool big = block_m == kMfmaBigBM;
  const double cu = cu_count(), step = big ? 1.4 : block_m == kMfmaMid2BM ? 1.07 : 0.83;
  const double wide = (double)ceil_div(n, gate_up ? 128 : 256), narrow = (double)ceil_div(n, gate_up ? 64 : 128);
  const double least = (double)rows.total() / block_m * wide;  // (bounds the counting below)
  if (block_m < kMfmaMidBM || least > kFewRounds * cu) return {Tiles::kList, std::ceil(least / cu) * step};
  const RowTileCount count = count_row_tiles(rows, block_m);
  // times by the number of row tiles; 128-row halves of a 256-row tile: one
  // without a second half still takes its place in the walk
  const double halves = big ? 2.0 : 1.0, narrow_step = block_m == kMfmaMidBM ? 0.55 : 0.71;
  const bool split = big && !gate_up && splits_tail(k);
  auto own = [&](double row_tiles) {
    if (split) {
      const int64_t tiles = std::llround(row_tiles * wide), g = std::min<int64_t>(std::llround(count.most * wide), cu);
      const int64_t left = g > 0 ? tiles % g : 0;
      const int64_t slices = left > 0 && 2 * left <= g ? std::min<int64_t>(g / left, k_steps(k) / kSplitMinSteps) : 1;
      if (slices >= 2) return ((double)(tiles / g) + 1.0 / (double)slices) * step + kSplitReduceUs / k_steps(k);
    }
    return std::ceil(row_tiles * wide / cu) * step;
  };
  auto wide_halves = [&](double row_tiles) { return std::ceil(halves * row_tiles * wide / cu) * 1.07; };
  auto narrow_tiles = [&](double row_tiles) { return std::ceil(halves * row_tiles * narrow / cu) * narrow_step; };
  const double t_own = own(count.even);
  if (count.even * wide > kFewRounds * cu) return {Tiles::kList, t_own};
  auto gains = [&](auto time) {
    if (!(time(count.even) < 0.9 * t_own)) return false;
    const double by = std::max(1.0, (count.skewed - count.even) / 64.0);
    for (double r = std::floor(count.even) + 1.0; r <= count.skewed; r += by)
      if (time(r) > 1.05 * own(r)) return false;
    return true;
  };
  const double t_wide = wide_halves(count.even), t_narrow = narrow_tiles(count.even);
  const bool take_wide = big && gains(wide_halves);
  if ((!take_wide || t_narrow <= t_wide) && gains(narrow_tiles))
    return {big ? Tiles::kNarrowHalves : block_m == kMfmaMid2BM ? Tiles::kNarrow : Tiles::kNarrowMid, t_narrow};
  if (take_wide) return {Tiles::kHalves, t_wide};
  return {Tiles::kList, t_own};
}

}  // namespace
}  // namespace astrai_moe
