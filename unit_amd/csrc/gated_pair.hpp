// Both products of a gated product's gradients in one launch: dx[r] = w^T dpre[r] and dw = sum dpre[r] x[r]^T, which have dpre in common and
// nothing to wait for in each other.  Workgroups of the longer reduction come first, those of the other fill the CUs that the last round
// of the first leaves idle.  us with the gate's gradients in front, bf16, rows x K -> N over groups (two launches; one; single runs side by
// side: another card is off by up to a tenth, both alike):
//   8192 x 1024 -> 2048 over 16: 212, 181    8192 x 1024 -> 1024 over 16: 114, 97    4000 x 768 -> 768 over 32: 83, 57
//   1000 x 520 -> 776 over 12: 28.9, 23.3    300 x 1024 -> 1024: 20.2, 14.1          2000 x 1024 -> 1024: 41, 26
//
// One group of many rows and a small weight has few tiles of dw and a long way along each: its rows are then shared out to `splits`
// workgroups a tile, whose sums meet in the workspace in float32 and are added in their order.
#pragma once
#include "grouped_tile.hpp"

namespace unit {

struct PairGrid {
  int first;         // workgroups of the product that comes first
  int dx_first;
  int dx_nts;        // column tiles of dx
  int dw_nts, dw_xts;  // column and row tiles of a group's dw
  int dw_parts;        // groups, or splits of the only one
  int split_rows;      // rows of a split; 0: groups as they are
};

// TX, NX: tile and stages of dx; TW, NW: of dw
template <class Op, class TX, int NX, class TW, int NW, class OutX, class OutW>
__global__ __launch_bounds__(TX::NT, 2) void gated_pair(GroupedParams px, GroupedParams pw, PairGrid g) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lane = threadIdx.x & 63;
  const bool front = (int)blockIdx.x < g.first;
  const int bid = front ? (int)blockIdx.x : (int)blockIdx.x - g.first;
  if (front == (g.dx_first != 0)) {
    const GroupTileOf t = find_tile<TX::BX, 8>(px, g.dx_nts, bid, lane);
    if (!t.any) return;
    compute_tile<Op, GRAD_DATA, TX, NX, OutX>(px, lds, t.group, t.first, t.count, t.x0, t.high, t.nt * TX::BY);
  } else {
    const int turn = bid / (g.dw_nts * g.dw_xts), in = bid - turn * (g.dw_nts * g.dw_xts), x0 = in % g.dw_xts * TW::BX;
    if (turn >= g.dw_parts) return;  // the front is rounded up to a multiple of the XCDs
    int group = turn, first = turn * g.split_rows, count = min(pw.rows - first, g.split_rows);
    if (!g.split_rows) find_rows(pw, turn, lane, group, first, count);
    compute_tile<Op, GRAD_WEIGHT, TW, NW, OutW>(pw, lds, group, first, count, x0, min(pw.n - x0, TW::BX), in / g.dw_xts * TW::BY);
  }
}

template <class Op, class TX, int NX, class TW, int NW, class OutX, class OutW>
int run_gated_pair(const char *what, const char *tag, const GroupedParams &px, GroupedParams pw, const PairPlan &plan, hipStream_t s) {
  constexpr int lds = NX * TX::STAGE > NW * TW::STAGE ? NX * TX::STAGE : NW * TW::STAGE;
  static_assert(lds <= kMaxLds && TX::NT == TW::NT, "rings fit the LDS, workgroups are of one size");
  auto kern = gated_pair<Op, TX, NX, TW, NW, OutX, OutW>;
  static thread_local unsigned long long allowed = 0;
  if (lds > 65536)
    if (int rc = allow_lds(what, reinterpret_cast<const void *>(kern), &allowed)) return rc;
  PairGrid g;
  g.dx_nts = ceil_div(px.k, TX::BY);
  g.dw_nts = ceil_div(pw.k, TW::BY), g.dw_xts = ceil_div(pw.n, TW::BX);
  // at most: every group, and the rows of none, ends inside a tile; a multiple of the XCDs, so that both products are dealt to them alike
  if (plan.splits > 1) pw.groups = plan.splits;  // each with sums of its own
  g.dw_parts = pw.groups;
  const long parts = px.sizes ? (px.groups + 1 < px.rows ? px.groups + 1 : px.rows) : 1;
  const long dx = ((px.rows + parts * (TX::BX - 1)) / TX::BX * g.dx_nts + 7 + 7) / 8 * 8, dw = (long)g.dw_parts * g.dw_nts * g.dw_xts;
  g.split_rows = plan.splits > 1 ? plan.split_rows : 0;
  g.dx_first = px.n >= (pw.rows + g.dw_parts - 1) / g.dw_parts;
  if ((dx + dw) * TX::NT >= 1l << 32) return fail(UNIT_E_ARG, "%s: %ld tiles exceed one launch", what, dx + dw);
  g.first = (int)(g.dx_first ? dx : (dw + 7) / 8 * 8);
  const long wgs = g.dx_first ? dx + dw : g.first + dx;
  hipLaunchKernelGGL(kern, dim3((unsigned)wgs), dim3(TX::NT), lds, s, px, pw, g);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(UNIT_E_LAUNCH, "%s: launch: %s", what, hipGetErrorString(e));
  set_variant("%s_x%d_y%d_w%d_y%d", tag, TX::BX, TX::BY, TW::BX, TW::BY);
  return UNIT_OK;
}

template <class Op, class OutX, class OutW>
int run_gated_pair_sizes(const char *what, const char *tag, const GroupedParams &px, const GroupedParams &pw, const PairPlan &plan, hipStream_t s) {
  using L = Tile<256, 256, 128, 2, 4>;
  using W = Tile<128, 128, 128, 2, 2, false, 2>;
  switch (plan.tiles) {
    case PAIR_SMALL: return run_gated_pair<Op, Tile<64, 64, 128, 2, 1, false, 2>, 4, Tile<128, 128, 64, 2, 2>, 4, OutX, OutW>(what, tag, px, pw, plan, s);
    case PAIR_WIDE: return run_gated_pair<Op, W, 3, W, 3, OutX, OutW>(what, tag, px, pw, plan, s);
    case PAIR_ROUND: return run_gated_pair<Op, Tile<192, 256, 128, 2, 4>, 2, L, 2, OutX, OutW>(what, tag, px, pw, plan, s);
    case PAIR_TALL: return run_gated_pair<Op, Tile<128, 256, 64, 2, 2>, 3, Tile<128, 256, 64, 2, 2>, 3, OutX, OutW>(what, tag, px, pw, plan, s);
    default: return run_gated_pair<Op, L, 2, L, 2, OutX, OutW>(what, tag, px, pw, plan, s);
  }
}

// dx_dtype, dw_dtype: UNIT_F32 or the operands' type, Half
template <class Op, class Half>
int run_gated_pair_types(const char *what, const char *tag, const GroupedParams &px, int dx_dtype, const GroupedParams &pw, int dw_dtype, const PairPlan &plan, hipStream_t s) {
  if (dx_dtype == UNIT_F32)
    return dw_dtype == UNIT_F32 ? run_gated_pair_sizes<Op, float, float>(what, tag, px, pw, plan, s) : run_gated_pair_sizes<Op, float, Half>(what, tag, px, pw, plan, s);
  return dw_dtype == UNIT_F32 ? run_gated_pair_sizes<Op, Half, float>(what, tag, px, pw, plan, s) : run_gated_pair_sizes<Op, Half, Half>(what, tag, px, pw, plan, s);
}

}  // namespace unit
