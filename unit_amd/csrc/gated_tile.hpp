// The tiles of the gated products: those of grouped_tile.hpp, in forms whose waves have an even number of column blocks.
#pragma once
#include "gated_mixed.hpp"
#include "gated_split.hpp"

namespace unit {

// Which tile (rows x columns of h, each of which is a row of the gate's and of the up projection's weight).  us, bf16 unless said otherwise,
// measured on both sides of each line (* the one taken; single runs side by side: another card is off by up to a tenth, both sides alike):
//   NARROW  64 x 32, two sets of waves that share the k-steps: one round of it.  Few tiles wait for their stages, each CU for its own: smaller
//           ones are more of them.
//             20 x 2048 -> 4096:           NARROW *9.5, SMALL 12.9    100 x 2048 -> 4096 (256 tiles): NARROW *10.2, SMALL 13.3
//             150 x 2048 -> 4096 (384):    NARROW 14.0, SMALL *13.1   700 x 1024 -> 1024 (352):       NARROW 9.4, SMALL *8.5
//   FEW     32 x 64, two sets: up to 16 rows a group
//             1000 x 1024 -> 1024 over 64: FEW *51.0, SMALL 52.9      300 over 16: FEW 15.7, SMALL *12.5
//   LARGE   256 x 128, one a CU: 128 rows a group, at least half of the CUs get one, 256 columns of reduction and 2^32 products in all
//   ROUND   192 x 128        } in the place of LARGE, whichever an estimate of the rounds says (large_tiles below):
//   MIXED   LARGE and WIDE   }   (us kept in 16 bits, LARGE, ROUND, MIXED with remainders of up to 128 and of up to 255 rows by WIDE)
//             8192 x 1024 -> 1024 over 16: 62.6, 62.1, *47.6, 47.7    16384 x 1024 -> 1024 over 32: 103, 115, *100, 106
//             6000 x 768 -> 1536 over 8: 47.1, 41.2, 48.3, *39.4      2200 x 2048 -> 4096: 97.6, 81.4, 97.4, *74.7
//             3000 x 1024 -> 2048: 31.3, *28.3, 31.1, 31.9            5000 x 1536 -> 1536: *46.4, 64.2, 46.2, 55.3
//   WIDE    128 x 64, two sets, one a CU: most of one round of it, 128 rows a group, and 2 KiB of reduction
//             1500 x 1024 -> 1024 (192 tiles): WIDE *11.8, MIDDLE 12.4, SMALL 13.0   500 x 2048 -> 4096 (256): WIDE *22.2, MIDDLE 22.6
//             1000 x 512 -> 2048 (256):    WIDE 11.5, MIDDLE *8.9     1000 x 1024 -> 1024 (128): WIDE 11.1, SMALL *9.0
//             2200 x 4096 -> 512 (144):    WIDE *27.5, SMALL 34.6     1000 x 1024 -> 1024 over 16: WIDE 22.3, SMALL *15.3
//   MIDDLE  128 x 64, two a CU: 192 tiles and as many rows a group
//             1000 x 512 -> 2048:          MIDDLE *8.9, SMALL 10.5    3000 x 1024 -> 1024 over 64: MIDDLE 63.9, SMALL *53.9
//   SMALL   64 x 64, two a CU
// Environment: UNIT_AMD_GATED_TILE=1..8 pins one, in the order below; UNIT_AMD_GATED_MOST a remainder of MIXED.
enum GatedTile { GATED_NARROW, GATED_FEW, GATED_SMALL, GATED_WIDE, GATED_MIDDLE, GATED_LARGE, GATED_ROUND, GATED_MIXED };
struct GatedTiling {
  GatedTile tile;
  int most = 128;  // MIXED: rows of a remainder that goes by small tiles
};

// LARGE, ROUND or MIXED: the least of their estimates.  A tile costs a start with its results, and its stages of 64 elements; tiles are dealt to
// 256 CUs, large ones first.  A group ends anywhere in a large tile.  Of 42 problems of 2200 to 16384 rows the one that it takes is 1.3 % slower
// than the best on average, 13 % at most (LARGE or ROUND alone: 7.7 and 30).  What is kept does not enter: it would change no choice of those,
// and h has the same bits with it and without.
inline GatedTiling large_tiles(const GatedParams &p, long groups) {
  const double stages = p.k / 64.0, large = 4 + 1.62 * stages, wide = 2 + 0.45 * stages;
  const long cols = (p.n + 127) / 128, wide_cols = (p.n + 63) / 64;
  const auto dealt = [](double front, double tf, double back, double tb) {
    const double rounds = (double)(long)(front / 256), left = front - 256 * rounds;
    const double filled = left > 0.01 ? (256 - left) * (long)(tf / tb) : 0, rest = back > filled ? back - filled : 0;
    return (left > 0.01 ? rounds + 1 : rounds) * tf + (double)(long)((rest + 255.99) / 256) * tb;
  };
  const auto rows_in = [&](int x) { return groups == 1 ? (double)((p.rows + x - 1) / x) : (double)p.rows / x + groups / 2.0; };
  GatedTiling best{GATED_LARGE};
  double least = dealt(rows_in(256) * cols, large, 0, wide);
  const auto consider = [&](GatedTile tile, int most, double us) {
    if (us < least) least = us, best = {tile, most};
  };
  consider(GATED_ROUND, 0, dealt(rows_in(192) * cols, 0.78 * large, 0, wide));
  for (const int most : {128, 255}) {
    const int rest = p.rows % 256;  // of a single group; of many, a remainder is anything
    const double front = groups == 1 ? p.rows / 256 + (rest > most) : (double)p.rows / 256 - groups * (0.5 - (255 - most) / 256.0);
    const double back = groups == 1 ? (rest > most ? 0 : (rest + 127) / 128) : groups * (128 + 2.0 * (most - 128)) / 256;
    consider(GATED_MIXED, most, dealt(front * cols, large, back * wide_cols, wide));
  }
  return best;
}

inline GatedTiling gated_tile_size(const GatedParams &p) {
  if (const int pinned = tuning_override("UNIT_AMD_GATED_TILE")) {
    const int most = tuning_override("UNIT_AMD_GATED_MOST");
    return {static_cast<GatedTile>(pinned - 1), most > 0 && most < 256 ? most : 128};
  }
  const long rows = p.rows ? p.rows : 1, busy = p.groups < rows ? p.groups : rows, mean = (rows + busy - 1) / busy;
  const auto tiles = [&](int x, int y) { return (mean + x - 1) / x * ((p.n + y - 1) / y) * busy; };
  if (tiles(64, 32) <= 256) return {GATED_NARROW};
  if (mean <= 16) return {GATED_FEW};
  if (mean >= 128 && p.n >= 96 && p.k >= 256 && tiles(256, 128) >= 128 && mean * p.n * 2 * busy >= (1l << 32) / p.k) return large_tiles(p, busy);
  const long middle = tiles(128, 64);
  if (middle >= 140 && middle <= 256 && p.k >= 1024 && mean >= 128) return {GATED_WIDE};
  return {middle >= 192 && mean >= 192 ? GATED_MIDDLE : GATED_SMALL};
}

template <class Op, class Out, int GATE>
int run_gated_sizes(const char *what, const char *tag, const GatedParams &p, hipStream_t s) {
  if constexpr (GATE != GATE_GRAD)
    if (p.rows <= kSplitRows && !tuning_override("UNIT_AMD_GATED_TILE")) return run_gated_split<typename Op::half_t, Out, GATE>(what, tag, p, s);
  // LARGE keeps pre-activations of 16 bits in lines of 64 columns a wave: 16384 x 1024 -> 1024 over 32 107.4 us by 32 columns, 104.0 so
  constexpr int WX = GATE == GATE_KEEP ? 4 : 2;
  const GatedTiling t = gated_tile_size(p);
  switch (t.tile) {
    case GATED_NARROW: return run_grouped_tile<Op, FORWARD, Tile<64, 64, 128, 2, 1, false, 2>, 4, Out, GATE>(what, tag, p, s);
    case GATED_FEW: return run_grouped_tile<Op, FORWARD, Tile<32, 128, 128, 1, 2, false, 2>, 4, Out, GATE>(what, tag, p, s);
    case GATED_WIDE: return run_grouped_tile<Op, FORWARD, Tile<128, 128, 128, 2, 2, false, 2>, 3, Out, GATE>(what, tag, p, s);
    case GATED_MIDDLE: return run_grouped_tile<Op, FORWARD, Tile<128, 128, 64, 2, 2>, 4, Out, GATE>(what, tag, p, s);
    case GATED_LARGE: return run_grouped_tile<Op, FORWARD, Tile<256, 256, 128, WX, 8 / WX>, 2, Out, GATE>(what, tag, p, s);
    case GATED_ROUND: return run_grouped_tile<Op, FORWARD, Tile<192, 256, 128, 2, 4>, 2, Out, GATE>(what, tag, p, s);
    case GATED_MIXED:
      return run_gated_mixed<Op, Tile<256, 256, 128, WX, 8 / WX>, Tile<128, 128, 128, 2, 2, false, 2>, 3, Out, GATE>(what, tag, p, t.most, s);
    default: return run_grouped_tile<Op, FORWARD, Tile<64, 128, 128, 2, 2>, 3, Out, GATE>(what, tag, p, s);
  }
}

// GATE_GRAD writes the operands' type
template <class Op, class Out>
int run_gated_gate(const char *what, int gate, const char *tag, const GatedParams &p, hipStream_t s) {
  if (gate == GATE_KEEP) return run_gated_sizes<Op, Out, GATE_KEEP>(what, tag, p, s);
  if (gate == GATE_KEEP8) return run_gated_sizes<Op, Out, GATE_KEEP8>(what, tag, p, s);
  if (gate == GATE_GRAD) return run_gated_sizes<Op, typename Op::half_t, GATE_GRAD>(what, tag, p, s);
  return run_gated_sizes<Op, Out, GATE_ONLY>(what, tag, p, s);
}

}  // namespace unit
