// MXFP4 products, grouped by expert or with one weight.
#include "grouped_split.hpp"

namespace unit {
namespace {

template <class Out>
int run(const char *what, const GroupedParams &p, hipStream_t s) {
  if (p.x_dtype == UNIT_F16) return run_grouped_split<_Float16, Out>(what, p, s);
  if (p.x_dtype == UNIT_BF16) return run_grouped_split<__bf16, Out>(what, p, s);
  const char *tag = "mxdense";
  switch (grouped_tile_size(p, FORWARD, true)) {
    case TILE_FEW: return run_grouped_tile<OpMx, FORWARD, Tile<32, 64, 128, 1, 2>, 2, Out>(what, tag, p, s);
    case TILE_SMALL: return run_grouped_tile<OpMx, FORWARD, Tile<64, 64, 128, 2, 2>, 3, Out>(what, tag, p, s);
    case TILE_MIDDLE: return run_grouped_tile<OpMx, FORWARD, Tile<128, 128, 128, 2, 2>, 2, Out>(what, tag, p, s);
    default: return run_grouped_tile<OpMx, FORWARD, Tile<256, 256, 128, 2, 4>, 2, Out>(what, tag, p, s);
  }
}

}  // namespace

// x in floats is taken where one launch for everything pays; the caller quantises it first elsewhere
bool grouped_mx_takes_floats(const GroupedParams &p) {
  return (p.x_dtype == UNIT_F16 || p.x_dtype == UNIT_BF16) && p.k % 8 == 0 && reinterpret_cast<uintptr_t>(p.x) % 16 == 0 && grouped_split_pays(p);
}

int run_grouped_mx(const char *what, const GroupedParams &p, int out_dtype, hipStream_t s) {
  if (out_dtype == UNIT_F32) return run<float>(what, p, s);
  return out_dtype == UNIT_F16 ? run<_Float16>(what, p, s) : run<__bf16>(what, p, s);
}

}  // namespace unit
