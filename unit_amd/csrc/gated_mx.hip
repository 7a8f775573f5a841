// MXFP4 gated products.
#include "grouped_split.hpp"

namespace unit {
namespace {

// the tile that the product with both halves of the weight would take
inline int gated_tile_size_mx(const GatedParams &p) {
  GroupedParams both = p;
  both.n = 2 * p.n;
  return grouped_tile_size(both, FORWARD, true);
}

template <class Out>
int run(const char *what, const GatedParams &p, hipStream_t s) {
  if (p.x_dtype == UNIT_F16) return run_grouped_split<_Float16, Out, GATE_ONLY>(what, p, s);
  if (p.x_dtype == UNIT_BF16) return run_grouped_split<__bf16, Out, GATE_ONLY>(what, p, s);
  const char *tag = "mxgated";
  switch (gated_tile_size_mx(p)) {
    case TILE_FEW: return run_grouped_tile<OpMx, FORWARD, Tile<32, 128, 128, 1, 2>, 2, Out, GATE_ONLY>(what, tag, p, s);
    case TILE_SMALL: return run_grouped_tile<OpMx, FORWARD, Tile<64, 128, 128, 2, 2>, 3, Out, GATE_ONLY>(what, tag, p, s);
    case TILE_MIDDLE: return run_grouped_tile<OpMx, FORWARD, Tile<128, 128, 128, 2, 2>, 2, Out, GATE_ONLY>(what, tag, p, s);
    default: return run_grouped_tile<OpMx, FORWARD, Tile<256, 256, 128, 2, 4>, 2, Out, GATE_ONLY>(what, tag, p, s);
  }
}

}  // namespace

// as grouped_mx_takes_floats: one launch for everything, where the chip holds its workgroups at once
bool gated_mx_takes_floats(const GroupedParams &p) {
  return (p.x_dtype == UNIT_F16 || p.x_dtype == UNIT_BF16) && p.k % 8 == 0 && reinterpret_cast<uintptr_t>(p.x) % 16 == 0 && grouped_split_pays(p, 2);
}

int run_gated_mx(const char *what, const GatedParams &p, int out_dtype, hipStream_t s) {
  if (out_dtype == UNIT_F32) return run<float>(what, p, s);
  return out_dtype == UNIT_F16 ? run<_Float16>(what, p, s) : run<__bf16>(what, p, s);
}

}  // namespace unit
