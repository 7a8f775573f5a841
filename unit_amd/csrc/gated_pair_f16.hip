// fp16 gradients of gated products.
#include "gated_pair.hpp"

namespace unit {

int run_gated_pair_f16(const char *what, const GroupedParams &px, int dx_dtype, const GroupedParams &pw, int dw_dtype, const PairPlan &plan, hipStream_t s) {
  return run_gated_pair_types<OpHalf, _Float16>(what, "f16gatedpair", px, dx_dtype, pw, dw_dtype, plan, s);
}

}  // namespace unit
