// Gated feed-forward products: h[r] = act(gate x[r]) * (up x[r]), the weight of a group being gate's N rows, then up's.
//
//   act(z) = z * sigmoid(c1 z + c3 z^3)     silu: c1 = 1, c3 = 0;  gelu_tanh: c1 = 2 sqrt(2 / pi), c3 = 0.044715 c1, since
//                                           (1 + tanh a) / 2 = sigmoid(2 a)
//   act'(z) = s + z s (1 - s) (c1 + 3 c3 z^2), s the sigmoid
//
// Both activations are one formula with two numbers, so that no kernel is built twice and none branches.
#pragma once
#include "grouped.hpp"
#include "mxfp8.hpp"

namespace unit {

struct Activation {
  float e1, e3, d1, d3;  // -log2(e) times c1 and c3: sigmoid = 1 / (1 + 2^(z (e1 + e3 z^2))); c1 and 3 c3
};
// false: no such activation
inline bool activation_of(int code, Activation *a) {
  if (code != UNIT_SILU && code != UNIT_GELU_TANH) return false;
  const double log2e = 1.4426950408889634, c = 1.5957691216057308;  // 2 sqrt(2 / pi)
  const double c1 = code == UNIT_SILU ? 1 : c, c3 = code == UNIT_SILU ? 0 : 0.044715 * c;
  *a = {(float)(-log2e * c1), (float)(-log2e * c3), (float)c1, (float)(3 * c3)};
  return true;
}

// z^2, bounded: its product with a c3 of 0 has to be 0, and the sigmoid is 0 or 1 long before
__device__ __forceinline__ float bounded_square(float z) { return fminf(z * z, 1e30f); }
__device__ __forceinline__ float act_share(const Activation &a, float z, float z2) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * fmaf(a.e3, z2, a.e1)));
}
__device__ __forceinline__ float act_value(const Activation &a, float z) { return z * act_share(a, z, bounded_square(z)); }
// act(z), and its derivative into *slope
__device__ __forceinline__ float act_both(const Activation &a, float z, float *slope) {
  const float z2 = bounded_square(z), s = act_share(a, z, z2), v = z * s;
  *slope = fmaf(v * (1.0f - s), fmaf(a.d3, z2, a.d1), s);
  return v;
}

// p.n: columns of h; the weight of a group has 2 * p.n rows
struct GatedParams : GroupedParams {
  Activation act;
  char *pre;         // kept pre-activations (rows, 2, N): the operands' type, or MXFP8 codes
  char *pre_scales;  // MXFP8
  const char *dh;    // GATE_GRAD: h's gradient (rows, N), of the operands' type
};

// What a kernel of the gated product writes: h, h and the pre-activations in the operands' type, h and them in MXFP8, or the gate's gradients
// dpre (rows, 2, N) in the place of h
enum Gate { GATE_NONE, GATE_ONLY, GATE_KEEP, GATE_KEEP8, GATE_GRAD };

// what a kernel of the product takes.  (The enumeration has a name and the condition none of it: in a kernel's mangled name an unnamed type is
// counted, and the host's count differs from the device's.)
template <int GATE>
using GateParams = std::conditional_t<(GATE != 0), GatedParams, GroupedParams>;

int run_gated_f16(const char *what, int gate, const GatedParams &p, int out_dtype, hipStream_t s);
int run_gated_bf16(const char *what, int gate, const GatedParams &p, int out_dtype, hipStream_t s);
int run_gated_mx(const char *what, const GatedParams &p, int out_dtype, hipStream_t s);

}  // namespace unit
