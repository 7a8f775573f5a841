// fp16 products grouped by expert and their gradients.
#include "grouped_tile.hpp"

namespace unit {
namespace {

template <int DIR>
int run(const char *what, const char *tag, const GroupedParams &p, int out_dtype, hipStream_t s) {
  return out_dtype == UNIT_F32 ? run_grouped_sizes<OpHalf, DIR, float>(what, tag, p, s) : run_grouped_sizes<OpHalf, DIR, _Float16>(what, tag, p, s);
}

}  // namespace

int run_grouped_f16(const char *what, int dir, const GroupedParams &p, int out_dtype, hipStream_t s) {
  if (dir == FORWARD) return run<FORWARD>(what, "f16grouped", p, out_dtype, s);
  if (dir == GRAD_DATA) return run<GRAD_DATA>(what, "f16groupeddx", p, out_dtype, s);
  return run<GRAD_WEIGHT>(what, "f16groupeddw", p, out_dtype, s);
}

}  // namespace unit
