// The tiles of the gated products: those of grouped_tile.hpp, in forms whose waves have an even number of column blocks.
#pragma once
#include "gated_split.hpp"

namespace unit {

// the tile that the product with both halves of the weight would take
inline int gated_tile_size(const GatedParams &p, bool mx) {
  GroupedParams both = p;
  both.n = 2 * p.n;
  return grouped_tile_size(both, FORWARD, mx);
}

template <class Op, class Out, int GATE>
int run_gated_sizes(const char *what, const char *tag, const GatedParams &p, hipStream_t s) {
  if constexpr (GATE != GATE_GRAD)
    if (p.rows <= kSplitRows && !tuning_override("UNIT_AMD_GROUPED_TILE")) 
      return run_gated_split<typename Op::half_t, Out, GATE>(what, tag, p, s);
  switch (gated_tile_size(p, false)) {
    case TILE_FEW: return run_grouped_tile<Op, FORWARD, Tile<32, 128, 128, 1, 2>, 3, Out, GATE>(what, tag, p, s);
    case TILE_SMALL: return run_grouped_tile<Op, FORWARD, Tile<64, 128, 128, 2, 2>, 3, Out, GATE>(what, tag, p, s);
    case TILE_MIDDLE: return run_grouped_tile<Op, FORWARD, Tile<128, 128, 64, 2, 2>, 4, Out, GATE>(what, tag, p, s);
    case TILE_ROUND: return run_grouped_tile<Op, FORWARD, Tile<192, 256, 128, 2, 4>, 2, Out, GATE>(what, tag, p, s);
    default: return run_grouped_tile<Op, FORWARD, Tile<256, 256, 128, 2, 4>, 2, Out, GATE>(what, tag, p, s);
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
