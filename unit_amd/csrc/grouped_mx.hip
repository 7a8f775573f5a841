// MXFP4 products, grouped by expert or with one weight.
#include "grouped_tile.hpp"

namespace unit {
namespace {

template <class Out>
int run(const char *what, const GroupedParams &p, hipStream_t s) {
  if (grouped_large(p, FORWARD)) return run_grouped_tile<OpMx, FORWARD, Tile<256, 256, 128, 2, 4>, 2, Out>(what, "mxdense", p, s);
  return run_grouped_tile<OpMx, FORWARD, Tile<128, 128, 128, 2, 2>, 2, Out>(what, "mxdense", p, s);
}

}  // namespace

int run_grouped_mx(const char *what, const GroupedParams &p, int out_dtype, hipStream_t s) {
  if (out_dtype == UNIT_F32) return run<float>(what, p, s);
  return out_dtype == UNIT_F16 ? run<_Float16>(what, p, s) : run<__bf16>(what, p, s);
}

}  // namespace unit
