// The tiles of the gated products: those of grouped_tile.hpp, in forms whose waves have an even number of column blocks.
#pragma once
#include "gated_split.hpp"

namespace unit {

// Which tile (rows x columns of h, each of which is a row of the gate's and of the up projection's weight).  us, bf16 unless said otherwise,
// measured on both sides of each line (* the one taken):
//   NARROW  64 x 32, two sets of waves that share the k-steps: one round of it.  Few tiles wait for their stages, each CU for its own: smaller
//           ones are more of them.
//             20 x 2048 -> 4096:           NARROW *9.5, SMALL 12.9    100 x 2048 -> 4096 (256 tiles): NARROW *10.2, SMALL 13.3
//             150 x 2048 -> 4096 (384):    NARROW 14.0, SMALL *13.1   700 x 1024 -> 1024 (352):       NARROW 9.4, SMALL *8.5
//   FEW     32 x 64, two sets: up to 16 rows a group
//             1000 x 1024 -> 1024 over 64: FEW *51.0, SMALL 52.9      300 over 16: FEW 15.7, SMALL *12.5
//   LARGE   256 x 128, one a CU: at least half of the CUs get one, 512 bytes of reduction and 2^32 products in all
//   ROUND   192 x 128: where its rounds are less work than LARGE's, a group ending in the middle of a tile on average
//             2200 x 2048 -> 4096:         LARGE 96.1, ROUND *80.9    8192 x 1024 -> 1024 over 16: LARGE 52.5, ROUND *46.3
//             16384 x 1024 -> 1024 over 32: LARGE *92.5, ROUND 105.7  4096 x 2048 -> 4096: LARGE *114.5, ROUND 129.1
//   WIDE    128 x 64, two sets, one a CU: most of one round of it, 128 rows a group, and 2 KiB of reduction
//             1500 x 1024 -> 1024 (192 tiles): WIDE *11.8, MIDDLE 12.4, SMALL 13.0   500 x 2048 -> 4096 (256): WIDE *22.2, MIDDLE 22.6
//             1000 x 512 -> 2048 (256):    WIDE 11.5, MIDDLE *8.9     1000 x 1024 -> 1024 (128): WIDE 11.1, SMALL *9.0
//             2200 x 4096 -> 512 (144):    WIDE *27.5, SMALL 34.6     1000 x 1024 -> 1024 over 16: WIDE 22.3, SMALL *15.3
//   MIDDLE  128 x 64, two a CU: 192 tiles and as many rows a group
//             1000 x 512 -> 2048:          MIDDLE *8.9, SMALL 10.5    3000 x 1024 -> 1024 over 64: MIDDLE 63.9, SMALL *53.9
//   SMALL   64 x 64, two a CU
// Environment: UNIT_AMD_GATED_TILE=1..7 pins one, in the order below.
enum GatedTile { GATED_NARROW, GATED_FEW, GATED_SMALL, GATED_WIDE, GATED_MIDDLE, GATED_LARGE, GATED_ROUND };
inline GatedTile gated_tile_size(const GatedParams &p) {
  if (const int pinned = tuning_override("UNIT_AMD_GATED_TILE")) return static_cast<GatedTile>(pinned - 1);
  const long rows = p.rows ? p.rows : 1, busy = p.groups < rows ? p.groups : rows, mean = (rows + busy - 1) / busy;
  const auto tiles = [&](int x, int y) { return (mean + x - 1) / x * ((p.n + y - 1) / y) * busy; };
  if (tiles(64, 32) <= 256) return GATED_NARROW;
  if (mean <= 16) return GATED_FEW;
  if (mean >= 192 && p.n >= 96 && p.k >= 256 && tiles(256, 128) >= 128 && mean * p.n * 2 * busy >= (1l << 32) / p.k) {
    // rounds of row tiles, half a tile more for each group that may end in one
    const auto rounds = [&](int x) { return (((2 * rows + x - 1) / x + (busy > 1 ? busy : 0) + 1) / 2 * ((p.n + 127) / 128) + 255) / 256 * x; };
    return 10 * rounds(192) < 9 * rounds(256) ? GATED_ROUND : GATED_LARGE;
  }
  const long middle = tiles(128, 64);
  if (middle >= 140 && middle <= 256 && p.k >= 1024 && mean >= 128) return GATED_WIDE;
  return middle >= 192 && mean >= 192 ? GATED_MIDDLE : GATED_SMALL;
}

template <class Op, class Out, int GATE>
int run_gated_sizes(const char *what, const char *tag, const GatedParams &p, hipStream_t s) {
  if constexpr (GATE != GATE_GRAD)
    if (p.rows <= kSplitRows && !tuning_override("UNIT_AMD_GATED_TILE")) return run_gated_split<typename Op::half_t, Out, GATE>(what, tag, p, s);
  // LARGE keeps pre-activations of 16 bits in lines of 64 columns a wave: 16384 x 1024 -> 1024 over 32 107.4 us by 32 columns, 104.0 so
  constexpr int WX = GATE == GATE_KEEP ? 4 : 2;
  switch (gated_tile_size(p)) {
    case GATED_NARROW: return run_grouped_tile<Op, FORWARD, Tile<64, 64, 128, 2, 1, false, 2>, 4, Out, GATE>(what, tag, p, s);
    case GATED_FEW: return run_grouped_tile<Op, FORWARD, Tile<32, 128, 128, 1, 2, false, 2>, 4, Out, GATE>(what, tag, p, s);
    case GATED_WIDE: return run_grouped_tile<Op, FORWARD, Tile<128, 128, 128, 2, 2, false, 2>, 3, Out, GATE>(what, tag, p, s);
    case GATED_MIDDLE: return run_grouped_tile<Op, FORWARD, Tile<128, 128, 64, 2, 2>, 4, Out, GATE>(what, tag, p, s);
    case GATED_LARGE: return run_grouped_tile<Op, FORWARD, Tile<256, 256, 128, WX, 8 / WX>, 2, Out, GATE>(what, tag, p, s);
    case GATED_ROUND: return run_grouped_tile<Op, FORWARD, Tile<192, 256, 128, 2, 4>, 2, Out, GATE>(what, tag, p, s);
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
