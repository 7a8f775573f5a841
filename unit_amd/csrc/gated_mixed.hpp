// Gated products by tiles of two sizes in one launch: a group's rows by 256 x 128 columns, but for a remainder of `most` rows or fewer, which goes
// by 128 x 64.  Groups that end inside a large tile cost a launch of few rounds a good part of one; small tiles come last and fill the
// CUs that the large ones leave.
#pragma once
#include "grouped_tile.hpp"

namespace unit {

struct MixedGrid {
  int front;                 // workgroups of large tiles, a multiple of the XCDs
  int front_nts, back_nts;   // column tiles of either
  int most;                  // rows of a remainder that goes by small tiles
};

template <class Op, class TF, class TB, int NB, class Out, int GATE>
__global__ __launch_bounds__(TF::NT, 2) void gated_mixed(GatedParams p, MixedGrid g) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lane = threadIdx.x & 63;
  if ((int)blockIdx.x < g.front) {
    const GroupTileOf t = find_tile<TF::BX, 8, FRONT_ROWS>(p, g.front_nts, (int)blockIdx.x, lane, g.most);
    if (!t.any) return;
    compute_tile<Op, FORWARD, TF, 2, Out, GATE>(p, lds, t.group, t.first, t.count, t.x0, t.high, t.nt * (TF::BY / 2));
  } else {
    const GroupTileOf t = find_tile<TB::BX, 8, BACK_ROWS>(p, g.back_nts, (int)blockIdx.x - g.front, lane, g.most);
    if (!t.any) return;
    compute_tile<Op, FORWARD, TB, NB, Out, GATE>(p, lds, t.group, t.first, t.count, t.x0, t.high, t.nt * (TB::BY / 2));
  }
}

template <class Op, class TF, class TB, int NB, class Out, int GATE>
int run_gated_mixed(const char *what, const char *tag, const GatedParams &p, int most, hipStream_t s) {
  constexpr int lds = 2 * TF::STAGE > NB * TB::STAGE ? 2 * TF::STAGE : NB * TB::STAGE;
  static_assert(lds <= kMaxLds && TF::NT == TB::NT && TF::BX == (int)kFront, "rings fit the LDS, workgroups are of one size");
  auto kern = gated_mixed<Op, TF, TB, NB, Out, GATE>;
  static thread_local unsigned long long allowed = 0;
  if (lds > 65536)
    if (int rc = allow_lds(what, reinterpret_cast<const void *>(kern), &allowed)) return rc;
  MixedGrid g;
  g.front_nts = ceil_div(p.n, TF::BY / 2), g.back_nts = ceil_div(p.n, TB::BY / 2);
  // at most: every group, and the rows of none, ends one row past the remainder that small tiles take; every one has such a remainder
  const long parts = p.sizes ? (p.groups + 1 < p.rows ? p.groups + 1 : p.rows) : 1;
  const long front = (((p.rows + parts * (long)(kFront - 1)) / kFront * g.front_nts + 7) + 7) / 8 * 8;
  const long back = parts * ceil_div(most, TB::BX) * g.back_nts + 7;
  if ((front + back) * TF::NT >= 1l << 32) return fail(UNIT_E_ARG, "%s: %ld tiles exceed one launch", what, front + back);
  g.front = (int)front, g.most = most;
  hipLaunchKernelGGL(kern, dim3((unsigned)(front + back)), dim3(TF::NT), lds, s, p, g);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(UNIT_E_LAUNCH, "%s: launch: %s", what, hipGetErrorString(e));
  set_variant("%s_x%d_y%d_x%d_y%d", tag, TF::BX, TF::BY, TB::BX, TB::BY);
  return UNIT_OK;
}

}  // namespace unit
