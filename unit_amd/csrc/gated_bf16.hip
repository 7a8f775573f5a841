// bf16 gated products.
#include "gated_tile.hpp"

namespace unit {

int run_gated_bf16(const char *what, int gate, const GatedParams &p, int out_dtype, hipStream_t s) {
  return out_dtype == UNIT_F32 && gate != GATE_GRAD ? run_gated_gate<OpBF16, float>(what, gate, "bf16gated", p, s) : run_gated_gate<OpBF16, __bf16>(what, gate, "bf16gated", p, s);
}

}  // namespace unit
