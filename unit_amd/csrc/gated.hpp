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
// How the two products of a gradient run (gated_pair.hpp): tiles of dx and of dw, and how many workgroups share the rows of a tile of dw.
//   PAIR_SMALL 64 x 64 (two sets of waves) and 128 x 128, two workgroups a CU    PAIR_WIDE 128 x 128 (two sets), one a CU
//   PAIR_ROUND 192 x 256 and 256 x 256                                           PAIR_LARGE 256 x 256
//   PAIR_TALL  128 x 256, two a CU, of several groups: the start and the results of one beside the stages of the other
// Chosen by an estimate: a tile costs a + b * (64-element stages), fitted to 20 forms of the launch on 28 problems; a launch takes its tiles over
// the workgroups that the chip holds, or its longest tile, whichever is more, and a quarter of the other.  Where the estimate is wrong it
// costs 3.5 % on average over those problems.  us, rows x K -> N over groups (* the one taken):
//   8192 x 1024 -> 2048 over 16: SMALL 250, WIDE 267, ROUND 191, LARGE 186, TALL *184   1000 x 1024 -> 1024 over 64: ROUND 153, LARGE 152, TALL *132
//   8192 x 1024 -> 1024 over 16: ROUND 102, LARGE 101, TALL *97                         200 x 512 -> 512 over 64: ROUND 32.5, LARGE 32.7, TALL *28.9
//   16384 x 512 -> 512, one group: LARGE *60.6, TALL 71.4                               3000 x 2048 -> 4096: SMALL 285, WIDE 241, ROUND *193, LARGE 203
//   1000 x 520 -> 776 over 12: SMALL *22.7, WIDE 30.2, ROUND 35.4, LARGE 35.7   2000 x 1024 -> 1024: SMALL 35.0, WIDE *28.0, ROUND 45.3
//   5000 x 768 -> 1536 over 4: SMALL 77.4, WIDE *74.5, ROUND 67.6, LARGE 75.7   (one of those where it is wrong)
// and of the splits, dense, at the best tiles for each:
//   16384 x 512 -> 512 1: 107, 4: 64, 16: *58    10000 x 256 -> 256 1: 66, 8: 26.0, 16: *27.1 (others 30)    8192 x 2048 -> 512 1: 90, 4: *77, 8: 99
//   8192 x 1024 -> 1024 1: 86, 4: *81, 8: 98     4096 x 1024 -> 2048 1: *79, 2: 93
// Environment: UNIT_AMD_GATED_PAIR=1..5 pins the tiles, UNIT_AMD_GATED_SPLITS the splits.
enum PairTiles { PAIR_SMALL, PAIR_WIDE, PAIR_ROUND, PAIR_LARGE, PAIR_TALL };
struct PairPlan {
  PairTiles tiles;
  int splits, split_rows;  // rows of a split: whole stages of 64
};
// both: 2 N; one_group: no sizes.  A function of these values alone: the workspace's size goes by it.
PairPlan gated_pair_plan(int rows, int groups, bool one_group, int both, int k);

// Whether dw of 16 bits goes past the caches: it would push out of the memory-side cache (256 MiB) what the call has yet to read, w above all,
// but what fits there is read back from it by the update that follows.  dw of 40 MiB, and either the pre-activations were computed from
// the rows first (w is read twice) or the call moves 280 MiB in all (moved: every operand, intermediate and result once).  Measured with an update
// of w by dw behind each call, us, through the caches and past them, * the one taken (rows x K -> N over groups; dw, moved):
//   pre kept   1000 x 512 -> 1024 over 64 (128 MiB, 268): *122.4, 125.7     700 x 960 -> 1024 over 32 (120, 249): *114.6, 117.7
//              6000 x 640 -> 1024 over 32 (80, 233): *119.4, 120.9          8192 x 384 -> 2048 over 16 (48, 268): *144.7, 146.4
//              4096 x 768 -> 2048 over 16 (96, 284): 170.7, *168.5          8192 x 512 -> 2048 over 16 (64, 304): 168.9, *167.9
//              3000 x 576 -> 512 over 128 (144, 309): 152.5, *145.2         4000 x 1024 -> 1024 over 64 (256, 567): 283, *273
//   in MXFP8   4096 x 832 -> 1024 over 32 (104, 263): *129.5, 129.6         4096 x 960 -> 1024 over 32 (120, 299): 139.3, *138.1
//   from rows  8192 x 256 -> 2048 over 16 (32 MiB): *123.5, 124.7           8192 x 384 -> 2048 over 16 (48): 169.3, *166.1
//              4096 x 768 -> 2048 over 16 (96): 205, *181                   4096 x 1024 -> 1024 over 32 (128): 181, *175
// Of 69 such pairs the choice is the slower one in six, by 2.2 % at most.  Timed without the update, calls from rows that move 265 to 320 MiB are up
// to 7 % slower past the caches, the others as above.
inline bool dw_past_caches(size_t dw_bytes, size_t moved, bool kept) { return dw_bytes >= (size_t)40 << 20 && (!kept || moved >= (size_t)280 << 20); }

// px: dpre, w, dx; pw: dpre, x, dw (splits > 1: float32 sums of each split, one behind the other)
int run_gated_pair_f16(const char *what, const GroupedParams &px, int dx_dtype, const GroupedParams &pw, int dw_dtype, const PairPlan &plan, hipStream_t s);
int run_gated_pair_bf16(const char *what, const GroupedParams &px, int dx_dtype, const GroupedParams &pw, int dw_dtype, const PairPlan &plan, hipStream_t s);
bool gated_mx_takes_floats(const GroupedParams &p);
int run_gated_mx(const char *what, const GatedParams &p, int out_dtype, hipStream_t s);

}  // namespace unit
