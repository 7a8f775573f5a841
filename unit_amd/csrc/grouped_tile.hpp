// Tiled kernel of the grouped products: tiles of both operands go global -> LDS by direct loads into a ring of NSTAGE stages, every
// MFMA is followed by one slice of the step's other work, as in mma_dma_kernel (mma_dma.hpp); here a workgroup first finds the
// group its tile belongs to, operands may both be reduction-major, and all loads are bounded by buffer descriptors.
//
// Operand forms.  "rows": reduction-contiguous rows, in LDS as rows of BKB bytes with their 16-byte chunks XORed (swz), fragments
// read 16 bytes a lane.  "cols": reduction-major, (reduction, width) with the width contiguous; the tile lies in LDS as in memory,
// [reduction][width], and fragments come out of it with the LDS transposing read, two per fragment.
//   forward        X = x rows,  Y = w rows       out[row][n]
//   data gradient  X = dy rows, Y = w cols       dx[row][k]
//   weight gradient X = dy cols, Y = x cols      dw[n][k], the reduction runs over a group's rows
// Y is the first MFMA operand: the result's rows lie along the lanes, its columns along the accumulator registers, four consecutive ones
// in four registers, so that results leave 16 bytes at a time (through LDS, where they are put in order).
//
// Bounds.  A stage's descriptor begins at the stage's first byte and ends where the operand's valid rows end, so rows past a group's
// last (weight gradient) read as zeros, and rows past a tile's last valid one read as zeros or stay in the tensor.  A reduction that ends
// inside a stage of rows: lanes whose chunk lies past its end are sent out of the descriptor, on both sides, so that what
// lies behind (NaN, say) meets nothing.
#pragma once
#include "grouped.hpp"
#include "mma_dma.hpp"

namespace unit {

struct OpHalf {
  using acc_t = v16f;
  static constexpr bool kMx = false;
  static __device__ __forceinline__ acc_t mma(v4i x, v4i y, acc_t c) { return OpF16::mma(x, y, c); }
};
struct OpBF16 {
  using acc_t = v16f;
  static constexpr bool kMx = false;
  static __device__ __forceinline__ acc_t mma(v4i x, v4i y, acc_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8b, x), __builtin_bit_cast(v8b, y), c, 0, 0, 0);
  }
};
// 64 elements of 4 bits are 32 bytes like 16 of 16 bits: the tiling in bytes is the same.  S: which byte of the scale dwords
struct OpMx {
  using acc_t = v16f;
  static constexpr bool kMx = true;
  template <int S>
  static __device__ __forceinline__ acc_t mma(v4i x, v4i y, acc_t c, int sx, int sy) {
    const v8i x8 = {x[0], x[1], x[2], x[3]}, y8 = {y[0], y[1], y[2], y[3]};
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(x8, y8, c, 4, 4, S, sx, S, sy);
  }
};

// ------------------------------------------------------------------------------------------- rows -> groups -> tiles
__device__ __forceinline__ u32 scalar(u32 v) { return (u32)__builtin_amdgcn_readfirstlane((int)v); }
__device__ __forceinline__ u32 lane_value(u32 v, int l) { return (u32)__builtin_amdgcn_readlane((int)v, l); }

// inclusive sums over the 64 lanes, no larger than `top` (v <= top <= 2^30, so no addition wraps)
__device__ __forceinline__ u32 scan_upto(u32 v, u32 top) {
  auto add = [&](u32 o) { v = min(v + o, top); };
  add((u32)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, false));  // row_shr 1, 2, 4, 8: inside 16 lanes
  add((u32)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, false));
  add((u32)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, false));
  add((u32)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, false));
  add((u32)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false));  // row_bcast 15: lane 15 to rows 1, 47 to 3
  add((u32)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false));  // row_bcast 31
  return v;
}

// Where the groups begin and end, in rows and in tiles of BM rows: sums of sizes over the lanes, lane l for group l of the chunk of 64
// at hand.  Every wave does this by itself.
template <int BM>
struct GroupScan {
  u32 rows0, tiles0;      // rows and tiles of the chunks before
  u32 start, end, tend;   // this lane's group: first row, end of rows, end of tiles
  u32 rows_in, tiles_in;  // rows and tiles of all groups
  int chunks;

  __device__ __forceinline__ void chunk(const GroupedParams &p, int c, int lane) {
    const int g = c * 64 + lane;
    const u32 size = g < p.groups ? (u32)group_size(p, g) : 0;
    end = min(rows0 + scan_upto(size, (u32)p.rows), (u32)p.rows);
    start = (u32)__builtin_amdgcn_update_dpp((int)rows0, (int)end, 0x138, 0xf, 0xf, false);  // the lane before's; lane 0: rows0
    tend = tiles0 + scan_upto((end - start + BM - 1) / BM, 1u << 30);
  }
  __device__ __forceinline__ void run(const GroupedParams &p, int lane) {
    rows0 = tiles0 = 0;
    chunks = (p.groups + 63) / 64;
    for (int c = 0; c < chunks; ++c) {
      if (c) rows0 = lane_value(end, 63), tiles0 = lane_value(tend, 63);
      chunk(p, c, lane);
    }
    rows_in = lane_value(end, 63), tiles_in = lane_value(tend, 63);
  }
  // tiles of all rows, those of no group included
  __device__ __forceinline__ u32 total(const GroupedParams &p) const { return tiles_in + ((u32)p.rows - rows_in + BM - 1) / BM; }
  // the group of row tile m < total(): itself (p.groups: none), its rows, and how many tiles lie before them
  __device__ __forceinline__ void find(const GroupedParams &p, u32 m, int lane, int &group, int &first, int &count, u32 &before) {
    if (m >= tiles_in) {
      group = p.groups, first = (int)rows_in, count = p.rows - (int)rows_in, before = tiles_in;
      return;
    }
    int c = 0;
    if (chunks > 1) {
      rows0 = tiles0 = 0;
      for (;; ++c) {
        chunk(p, c, lane);
        if (lane_value(tend, 63) > m) break;
        rows0 = lane_value(end, 63), tiles0 = lane_value(tend, 63);
      }
    }
    const int l = __builtin_ctzll(__ballot(tend > m));  // ends never decrease: the first group that ends behind m
    group = c * 64 + l;
    first = (int)lane_value(start, l);
    count = (int)lane_value(end, l) - first;
    before = l ? lane_value(tend, l - 1) : tiles0;
  }
};

struct GroupTileOf {
  int group;         // p.groups: rows of no group
  int first, count;  // the group's rows
  int x0, high;      // the tile's rows: first (of the group's), how many
  int nt;            // tile of the columns
  bool any;          // the workgroup has a tile
};

// The tile of workgroup `bid`.  The number of tiles is known here only, so the host launches what any sizes can need and the rest
// ends at once.  Workgroups are dealt round-robin to the eight XCDs: those of one XCD take consecutive tiles, which walk a group in
// panels of PH row tiles, column tile after column tile, so that the XCD's L2 holds the panel's rows and sees each weight tile once
// a panel.
template <int BM, int PH>
__device__ __forceinline__ GroupTileOf find_tile(const GroupedParams &p, int nts, int bid, int lane) {
  GroupTileOf t;
  GroupScan<BM> scan;
  scan.run(p, lane);
  const u32 total = scan.total(p) * (u32)nts;
  const u32 per = total / 8, rem = total % 8, xcd = (u32)bid % 8, idx = (u32)bid / 8;
  const u32 logical = xcd * per + min(xcd, rem) + idx;
  t.any = idx < per + (xcd < rem ? 1u : 0u);
  if (!t.any) return t;
  u32 before;
  scan.find(p, scalar(logical / (u32)nts), lane, t.group, t.first, t.count, before);  // a group is nts * (its row tiles)
  const u32 mts = ((u32)t.count + BM - 1) / BM, within = scalar(logical) - before * (u32)nts;
  const u32 panel = within / ((u32)nts * PH), in_panel = within - panel * ((u32)nts * PH);
  const u32 high = min(mts - panel * PH, (u32)PH);
  t.nt = (int)scalar(in_panel / high);
  const u32 mt = panel * PH + in_panel - (u32)t.nt * high;
  // as many tiles as BM asks for, of even heights in blocks of 32 rows; never beyond the end: (mts - 1) * BM < count
  const u32 even = scalar(((u32)t.count + 32 * mts - 1) / (32 * mts)) * 32;
  t.x0 = (int)scalar(mt * even);
  t.high = min(t.count - t.x0, (int)even);
  return t;
}

// The rows of the group whose turn it is: the longest first where a wave holds them all, so that the last workgroups have little to do,
// else as they come.
__device__ __forceinline__ void find_rows(const GroupedParams &p, int turn, int lane, int &group, int &first, int &count) {
  u32 rows0 = 0, end = 0, start = 0;
  const int last = p.groups <= 64 ? 0 : turn / 64;
  for (int c = 0; c <= last; ++c) {
    if (c) rows0 = lane_value(end, 63);
    const int i = c * 64 + lane;
    end = min(rows0 + scan_upto(i < p.groups ? (u32)group_size(p, i) : 0, (u32)p.rows), (u32)p.rows);
    start = (u32)__builtin_amdgcn_update_dpp((int)rows0, (int)end, 0x138, 0xf, 0xf, false);
  }
  int l = turn % 64;
  group = turn;
  if (p.groups <= 64) {
    const u32 size = end - start;
    int before = 0;  // how many have their turn before this lane's group
    for (int g = 0; g < p.groups; ++g) {
      const u32 other = lane_value(size, g);
      before += other > size || (other == size && g < lane);
    }
    group = l = __builtin_ctzll(__ballot(lane < p.groups && before == turn));
  }
  first = (int)lane_value(start, l);
  count = (int)lane_value(end, l) - first;
}

// ------------------------------------------------------------------------------------------- the kernel
__device__ __forceinline__ v4i bounded(const char *base, u32 bytes) {
  const unsigned long long b = (unsigned long long)base;
  v4i r;
  r[0] = (int)scalar((u32)b);
  r[1] = (int)scalar((u32)(b >> 32) & 0xffffu);
  r[2] = (int)scalar(bytes);
  r[3] = 0x00020000;
  return r;
}
constexpr u32 kOutside = 0xfffffff0u;  // past every descriptor

// XOR of the 16-byte chunk position inside a row of a "cols" tile, so that the four rows of a transposing read fall into
// different bank groups (rows of 128, 256 or 512 bytes)
template <int WIDTH>
__device__ __forceinline__ int cols_swz(int row) {
  static_assert(WIDTH == 64 || WIDTH == 128 || WIDTH == 256, "tile widths");
  return WIDTH == 64 ? 4 * ((row >> 1) & 1) : 4 * (row & 3);
}

// One tile: rows x0 .. x0 + high - 1 of the group's (weight gradient: rows of dw), columns y0 .. y0 + BY - 1.
template <class Op, int DIR, class T, int NSTAGE, class Out>
__device__ __forceinline__ void compute_tile(const GroupedParams &p, char *lds, int group, int first, int count, int x0, int high, int y0) {
  constexpr bool MX = Op::kMx, XT = DIR == GRAD_WEIGHT, YT = DIR != FORWARD;
  constexpr int KK = T::BKB / 32, CPR = T::CPR, NW = T::NT / 64, RPL = 64 / CPR;
  constexpr int KS = T::BKB / 2;                     // cols: reduction elements of a stage
  constexpr int XL = T::XBYTES / 1024 / NW, YL = T::YBYTES / 1024 / NW;
  constexpr int SCALES = MX ? (T::BX + T::BY) * 8 : 0, PIECES = MX ? (SCALES + 1023) / 1024 : 0, PIECE = PIECES ? PIECES : 1;
  constexpr int LPS = XL + YL + (MX ? 1 : 0);        // direct loads per wave and stage
  constexpr int STAGE = T::STAGE + PIECES * 1024;
  static_assert(XL * 1024 * NW == T::XBYTES && YL * 1024 * NW == T::YBYTES && KK % 2 == 0, "loads split evenly over the waves");
  static_assert(!MX || (T::BKB == 128 && PIECES <= NW && DIR == FORWARD), "a stage of MXFP4 is one dword of scales per row and half");

  const int t = threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int wx = wave / T::WY, wy = wave % T::WY, l32 = lane & 31, half = lane >> 5;  // waves of different rows share a SIMD
  // the row blocks there are, shared out evenly: this wave's first and how many
  const int high32 = (high + 31) / 32, block0 = (high32 * wx + T::WX - 1) / T::WX, blocks_x = (high32 * (wx + 1) + T::WX - 1) / T::WX - block0;
  const u32 ring = (u32)(uintptr_t)(lptr_t)lds;

  const int ys = DIR == FORWARD ? p.n : p.k;  // columns of the result
  const bool live = group < p.groups;

  // operand bases (of this tile's first row or column), bytes per row, and how many bytes lie behind the base
  const int K = DIR == FORWARD ? p.k : DIR == GRAD_DATA ? p.n : count;  // reduction elements
  const long xld = MX ? (long)mx_stages(p.k) * 128 : DIR == FORWARD ? 2l * p.k : 2l * p.n;
  const long yld = MX ? xld : 2l * p.k;
  const int kbytes = MX ? (int)xld : K * 2;
  const int nk = !live ? 0 : XT ? (count + KS - 1) / KS : YT ? (K + KS - 1) / KS : (kbytes + T::BKB - 1) / T::BKB;
  const char *xb, *yb;
  long xleft, yleft;
  if constexpr (XT) {
    xb = p.x + (long)first * xld + 2l * x0, xleft = (long)count * xld - 2l * x0;
    yb = p.y + (long)first * yld + 2l * y0, yleft = (long)count * yld - 2l * y0;
  } else {
    xb = p.x + (long)(first + x0) * xld, xleft = (long)high * xld;
    if constexpr (YT)
      yb = p.y + (long)group * p.n * yld + 2l * y0, yleft = (long)p.n * yld - 2l * y0;
    else
      yb = p.y + ((long)group * p.n + y0) * yld, yleft = (long)min(ys - y0, T::BY) * yld;
  }
  const long xstep = XT ? (long)KS * xld : T::BKB, ystep = YT ? (long)KS * yld : T::BKB;  // bytes from stage to stage

  // this lane's chunk of each load
  u32 xoff[XL], yoff[YL];
  auto offset = [&](auto cols, auto width, int load, long ld) __attribute__((always_inline)) {
    constexpr int W = decltype(width)::value;
    if constexpr (decltype(cols)::value) {
      constexpr int CPW = W / 8;
      const int row = load * (64 / CPW) + lane / CPW;
      return (u32)row * (u32)ld + (u32)(((lane % CPW) ^ cols_swz<W>(row)) << 4);
    } else {
      const int row = load * RPL + lane / CPR;
      return (u32)row * (u32)ld + (u32)(((lane % CPR) ^ swz<T::BKB>(row)) << 4);
    }
  };
#pragma unroll
  for (int i = 0; i < XL; ++i) xoff[i] = offset(std::integral_constant<bool, XT>{}, std::integral_constant<int, T::BX>{}, wave * XL + i, xld);
#pragma unroll
  for (int i = 0; i < YL; ++i) yoff[i] = offset(std::integral_constant<bool, YT>{}, std::integral_constant<int, T::BY>{}, wave * YL + i, yld);
  // MXFP4: the scales of a stage, X rows then Y rows, each [half][row] dwords, 64 pieces of four rows per load
  const char *sptr = nullptr;
  long sstep = 0;
  if constexpr (MX) {
    const int c = min((wave % PIECE) * 64 + lane, (T::BX + T::BY) / 2 - 1), cy = c - T::BX / 2;
    const long xrows = p.rows, yrows = (long)p.groups * p.n;
    if (c < T::BX / 2)
      sptr = reinterpret_cast<const char *>(p.xs + c / (T::BX / 4) * xrows + first + x0 + c % (T::BX / 4) * 4), sstep = xrows * 8;
    else
      sptr = reinterpret_cast<const char *>(p.ys + cy / (T::BY / 4) * yrows + (long)group * p.n + y0 + cy % (T::BY / 4) * 4), sstep = yrows * 8;
  }

  struct Source {
    v4i x, y;
  };
  // descriptors of stage kt
  auto source = [&](int kt) __attribute__((always_inline)) {
    const long xa = kt * xstep, ya = kt * ystep;
    auto clip = [](long v) { return (u32)min(v, 0xffffff00l); };
    return Source{bounded(xb + xa, clip(xleft - xa)), bounded(yb + ya, clip(yleft - ya))};
  };
  // load i of stage kt into ring buffer `slot`; last: the reduction may end inside the stage
  auto issue_one = [&](const Source &src, int kt, int slot, int i, auto last) __attribute__((always_inline)) {
    const u32 buf = ring + (u32)(slot * STAGE);
    auto inside = [&](u32 off, int j, bool cols, int n) {
      if (!decltype(last)::value || cols || MX) return off;
      const int row = (wave * n + j) * RPL + lane / CPR;
      const int at = kt * T::BKB + (((lane % CPR) ^ swz<T::BKB>(row)) << 4);
      return at < kbytes ? off : kOutside;
    };
    if (i < XL)
      dma_buffer_16(buf + (wave * XL + i) * 1024, inside(xoff[i], i, XT, XL), src.x, 0);
    else if (i < XL + YL)
      dma_buffer_16(buf + T::XBYTES + (wave * YL + (i - XL)) * 1024, inside(yoff[i - XL], i - XL, YT, YL), src.y, 0);
    else
      direct_load_16(sptr + kt * sstep, buf + T::STAGE + (wave % PIECE) * 1024);
  };

  typename Op::acc_t acc[T::TX][T::TY];
#pragma unroll
  for (int i = 0; i < T::TX; ++i)
#pragma unroll
    for (int j = 0; j < T::TY; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;

  // fragment addresses inside a stage, k-step 0
  const int xrow = block0 * 32 + l32, yrow = wy * (T::TY * 32) + l32;
  const int xsw = swz<T::BKB>(xrow), ysw = swz<T::BKB>(yrow);
  int xtr[T::TX], ytr[T::TY];
  {
    const int jrow = (lane & 15) >> 2, q = lane & 3, g16 = (lane >> 4) & 1;
    auto at = [&](int c, auto width) {
      constexpr int W = decltype(width)::value;
      return (8 * half + jrow) * (W * 2) + (((c + 2 * g16 + (q >> 1)) ^ cols_swz<W>(jrow)) << 4) + (q & 1) * 8;
    };
    if constexpr (XT) {
#pragma unroll
      for (int i = 0; i < T::TX; ++i) xtr[i] = at(block0 * 4 + i * 4, std::integral_constant<int, T::BX>{});
    }
    if constexpr (YT) {
#pragma unroll
      for (int j = 0; j < T::TY; ++j) ytr[j] = T::XBYTES + at(wy * (T::TY * 4) + j * 4, std::integral_constant<int, T::BY>{});
    }
  }
  auto transposed = [&](const char *src, int pitch) __attribute__((always_inline)) {
    typedef __attribute__((address_space(3))) v4s *trptr_t;
    typedef short v8s __attribute__((ext_vector_type(8)));
    const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((trptr_t)(src));
    const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((trptr_t)(src + 4 * pitch));
    return __builtin_bit_cast(v4i, (v8s)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  };
  v4i xf[2][T::TX], yf[2][T::TY];
  int sx[2][T::TX], sy[2][T::TY];  // MXFP4: scale dwords of this stage and of the next
  // fragment idx of a step's list: X0, Y0 .. Y(TY-1), X1 .. X(TX-1)
  auto load_one = [&](const char *stage, int kk, int s, int idx) __attribute__((always_inline)) {
    if (idx >= 1 && idx <= T::TY) {
      const int j = idx - 1;
      if constexpr (YT)
        yf[s][j] = transposed(stage + ytr[j] + kk * 16 * (T::BY * 2), T::BY * 2);
      else
        yf[s][j] = *reinterpret_cast<const v4i *>(stage + T::XBYTES + (yrow + j * 32) * T::BKB + (((2 * kk + half) ^ ysw) << 4));
      if (MX && kk == 0) sy[1][j] = *reinterpret_cast<const int *>(stage + T::STAGE + T::BX * 8 + half * (T::BY * 4) + (yrow + j * 32) * 4);
    } else {
      const int i = idx == 0 ? 0 : idx - T::TY;
      if constexpr (XT)
        xf[s][i] = transposed(stage + xtr[i] + kk * 16 * (T::BX * 2), T::BX * 2);
      else
        xf[s][i] = *reinterpret_cast<const v4i *>(stage + (xrow + i * 32) * T::BKB + (((2 * kk + half) ^ xsw) << 4));
      if (MX && kk == 0) sx[1][i] = *reinterpret_cast<const int *>(stage + T::STAGE + half * (T::BX * 4) + (xrow + i * 32) * 4);
    }
  };
  auto next_scales = [&]() __attribute__((always_inline)) {
    if constexpr (MX) {
#pragma unroll
      for (int i = 0; i < T::TX; ++i) sx[0][i] = sx[1][i];
#pragma unroll
      for (int j = 0; j < T::TY; ++j) sy[0][j] = sy[1][j];
    }
  };
  using yes = std::integral_constant<bool, true>;
  using no = std::integral_constant<bool, false>;
  // One k-step: MFMAs, each followed by its share of the next step's fragment reads and of the loads of a later stage.
  // NX: how many of its row blocks this wave has rows for; the others are left out.
  auto step = [&](auto nxc, auto kkc, const char *rd_stage, int rd_kk, const Source &src, int issue_kt, int slot, auto has_read, auto has_issue, auto last)
                  __attribute__((always_inline)) {
    constexpr int s = decltype(kkc)::value & 1, NX = decltype(nxc)::value, NM = NX * T::TY, NF = NX ? NX + T::TY : 0, PER = NM ? NM : 1;
    if constexpr (NX == 0 && decltype(has_issue)::value) {
#pragma unroll
      for (int f = 0; f < LPS; ++f) issue_one(src, issue_kt, slot, f, last);
    }
#pragma unroll
    for (int m = 0; m < NM; ++m) {
      const int i = m / T::TY, j = m % T::TY;
      if constexpr (MX)
        acc[i][j] = Op::template mma<decltype(kkc)::value>(yf[s][j], xf[s][i], acc[i][j], sy[0][j], sx[0][i]);
      else
        acc[i][j] = Op::mma(yf[s][j], xf[s][i], acc[i][j]);
      if constexpr (decltype(has_read)::value) {
#pragma unroll
        for (int f = m * NF / PER; f < (m + 1) * NF / PER; ++f) load_one(rd_stage, rd_kk, s ^ 1, f);
      }
      if constexpr (decltype(has_issue)::value) {
#pragma unroll
        for (int f = m * LPS / PER; f < (m + 1) * LPS / PER; ++f) issue_one(src, issue_kt, slot, f, last);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // One stage.  ISSUE: stage kt + NSTAGE exists and goes into the buffer that this stage frees; STEADY: NSTAGE - 1 younger stages are in
  // flight at the barrier; NEXT: stage kt + 1 exists; LAST: the stage that is fetched may hold the reduction's end.
  auto stage = [&](auto nxc, int kt, int slot, auto issue_next, auto steady, auto next, auto last) __attribute__((always_inline)) {
    const char *cur = lds + slot * STAGE;
    const char *nxt = lds + (slot + 1 == NSTAGE ? 0 : slot + 1) * STAGE;
    const Source none{};
    auto early = [&](auto kkc) __attribute__((always_inline)) { step(nxc, kkc, cur, decltype(kkc)::value + 1, none, 0, 0, yes{}, no{}, no{}); };
    early(std::integral_constant<int, 0>{});
    if constexpr (KK > 2) {
      early(std::integral_constant<int, 1>{});
      early(std::integral_constant<int, 2>{});
    }
    if constexpr (decltype(steady)::value)
      UNIT_WAIT_VMCNT((NSTAGE - 2) * LPS);
    else
      UNIT_WAIT_VMCNT(0);
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): this wave's reads of `cur` are done
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    Source src{};
    if constexpr (decltype(issue_next)::value) src = source(kt + NSTAGE);
    step(nxc, std::integral_constant<int, KK - 1>{}, nxt, 0, src, kt + NSTAGE, slot, next, issue_next, last);
    if constexpr (decltype(next)::value) next_scales();
  };

  if (nk > 0) {
#pragma unroll
    for (int s = 0; s < NSTAGE; ++s)
      if (s < nk) {
        const Source src = source(s);
#pragma unroll
        for (int i = 0; i < LPS; ++i) issue_one(src, s, s, i, yes{});
      }
    if (nk >= NSTAGE)
      UNIT_WAIT_VMCNT((NSTAGE - 1) * LPS);
    else
      UNIT_WAIT_VMCNT(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    auto loop = [&](auto nxc) __attribute__((always_inline)) {
      constexpr int NX = decltype(nxc)::value;
#pragma unroll
      for (int f = 0; f < (NX ? NX + T::TY : 0); ++f) load_one(lds, 0, 0, f);
      next_scales();
      int kt = 0;
      for (; kt + 2 * NSTAGE < nk; kt += NSTAGE) {  // fetches up to stage kt + 2 * NSTAGE - 1: never the last one
#pragma unroll
        for (int s = 0; s < NSTAGE; ++s) stage(nxc, kt + s, s, yes{}, yes{}, yes{}, no{});
      }
      for (; kt + NSTAGE < nk; ++kt) stage(nxc, kt, kt % NSTAGE, yes{}, yes{}, yes{}, yes{});
      for (; kt + 1 < nk; ++kt) stage(nxc, kt, kt % NSTAGE, no{}, no{}, yes{}, no{});
      stage(nxc, kt, kt % NSTAGE, no{}, no{}, no{}, no{});
    };
    // a wave without columns has no rows either
    const int blocks = y0 + wy * (T::TY * 32) < ys ? blocks_x : 0;
    if (blocks == T::TX)
      loop(std::integral_constant<int, T::TX>{});
    else if (blocks == 0)
      loop(std::integral_constant<int, 0>{});
    else if (T::TX > 2 && blocks == 3)
      loop(std::integral_constant<int, T::TX < 3 ? T::TX : 3>{});
    else if (T::TX > 2 && blocks == 2)
      loop(std::integral_constant<int, T::TX < 2 ? T::TX : 2>{});
    else
      loop(std::integral_constant<int, 1>{});
  }

  // Results, rounded once, here: each wave puts 32 rows of its columns in order in LDS of its own and writes them in runs of 16 bytes a lane.
  // (Straight from the registers, 2 bytes a lane: experts of 16384 x 1024 -> 2048 102.7 us, 96.2 like this.)
  constexpr int ES_OUT = (int)sizeof(Out), PITCH = T::TY * 32 * ES_OUT + 16, PER = 16 / ES_OUT, RUNS = T::TY * 32 / PER;  // elements per run, runs per row
  static_assert(NW * 32 * PITCH <= NSTAGE * STAGE, "the waves' rows fit the ring");
  __syncthreads();  // the ring is read out
  char *const rows = lds + wave * (32 * PITCH);
  const long out_row = (DIR == GRAD_WEIGHT ? (long)group * p.n : (long)first) + x0;
  const __amdgpu_buffer_rsrc_t out = __builtin_amdgcn_make_buffer_rsrc(p.out + out_row * ys * (long)sizeof(Out), 0, -1, 0x00020000);
  // Weight gradients in fp32 whose rows are whole lines go out with nt: as large as all operands together, they would push those out
  // of the memory-side cache (119 -> 115 us for both gradients of 8192 rows; results of 16 bits lose, forward 90 -> 97).
  const bool whole = ys % PER == 0, lines = ys % 32 == 0;
  typedef Out v4o __attribute__((ext_vector_type(4)));
#pragma unroll
  for (int i = 0; i < T::TX; ++i) {
    if (i >= blocks_x) break;
    const int xi = (block0 + i) * 32;
#pragma unroll
    for (int j = 0; j < T::TY; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        v4o v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (Out)acc[i][j][4 * r + e];
        *reinterpret_cast<v4o *>(rows + l32 * PITCH + (j * 32 + 8 * r + 4 * half) * ES_OUT) = v;
      }
#pragma unroll
    for (int k = 0; k < 32 * RUNS / 64; ++k) {
      const int row = (k * 64 + lane) / RUNS, c = (k * 64 + lane) % RUNS * PER, x = xi + row, y = y0 + wy * (T::TY * 32) + c;
      const v4u v = *reinterpret_cast<const v4u *>(rows + row * PITCH + c * ES_OUT);
      if (x >= high || y >= ys) continue;
      const u32 at = ((u32)x * (u32)ys + (u32)y) * (u32)ES_OUT;
      if (DIR == GRAD_WEIGHT && ES_OUT == 4 && lines) {
        store_result<kResultPolicy>(out, at, v);
      } else if (whole) {
        store_result<kRowPolicy>(out, at, v);
      } else if (y + PER <= ys) {  // rows begin on any element: the same 16 bytes, unaligned
        typedef u32 v4un __attribute__((ext_vector_type(4), aligned(2)));
        *reinterpret_cast<v4un *>(p.out + (out_row + x) * (long)ys * ES_OUT + (long)y * ES_OUT) = v;
      } else {
#pragma unroll
        for (int e = 0; e < PER; ++e)
          if (y + e < ys) {
            if constexpr (ES_OUT == 4)
              store_result<kRowPolicy>(out, at + e * 4, v[e]);
            else
              store_result<kRowPolicy>(out, at + e * 2, (unsigned short)(v[e / 2] >> (e % 2 * 16)));
          }
      }
    }
  }
}

template <class Op, int DIR, class T, int NSTAGE, class Out>
__global__ __launch_bounds__(T::NT, 2) void grouped_tile(GroupedParams p, int nts, int xts) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lane = threadIdx.x & 63;
  if constexpr (DIR == GRAD_WEIGHT) {
    // Consecutive workgroups, which go to the eight XCDs in turn, share a group: each XCD has its part of the long ones and of the
    // short ones (8192 rows over 16, 288 to 1220 each: 71 us with two groups an XCD, 64.5 like this).
    const int turn = (int)blockIdx.x / (nts * xts), in = (int)blockIdx.x - turn * (nts * xts), x0 = in % xts * T::BX;
    int group, first, count;
    find_rows(p, turn, lane, group, first, count);
    compute_tile<Op, DIR, T, NSTAGE, Out>(p, lds, group, first, count, x0, min(p.n - x0, T::BX), in / xts * T::BY);
  } else {
    const GroupTileOf g = find_tile<T::BX, 4>(p, nts, (int)blockIdx.x, lane);
    if (!g.any) return;
    compute_tile<Op, DIR, T, NSTAGE, Out>(p, lds, g.group, g.first, g.count, g.x0, g.high, g.nt * T::BY);
  }
}

template <class Op, int DIR, class T, int NSTAGE, class Out>
int run_grouped_tile(const char *what, const char *tag, const GroupedParams &p, hipStream_t s) {
  constexpr int lds = NSTAGE * (T::STAGE + (Op::kMx ? ((T::BX + T::BY) * 8 + 1023) / 1024 * 1024 : 0));
  static_assert(lds <= kMaxLds, "ring does not fit the LDS");
  auto kern = grouped_tile<Op, DIR, T, NSTAGE, Out>;
  static thread_local bool allowed = false;
  if (!allowed && lds > 65536) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, kMaxLds);
    if (e != hipSuccess) return fail(UNIT_E_LAUNCH, "%s: hipFuncSetAttribute: %s", what, hipGetErrorString(e));
    allowed = true;
  }
  const int ys = DIR == FORWARD ? p.n : p.k, nts = ceil_div(ys, T::BY), xts = ceil_div(p.n, T::BX);
  long wgs;
  if (DIR == GRAD_WEIGHT) {
    wgs = (long)p.groups * nts * xts;
  } else {
    // at most: every group, and the rows of none, ends inside a tile
    const long parts = p.sizes ? (p.groups + 1 < p.rows ? p.groups + 1 : p.rows) : 1;
    wgs = (p.rows + parts * (T::BX - 1)) / T::BX * nts + 7;  // + 7: an XCD's share is rounded up
  }
  if (wgs * T::NT >= 1l << 32) return fail(UNIT_E_ARG, "%s: %ld tiles exceed one launch", what, wgs);
  hipLaunchKernelGGL(kern, dim3((unsigned)wgs), dim3(T::NT), lds, s, p, nts, xts);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(UNIT_E_LAUNCH, "%s: launch: %s", what, hipGetErrorString(e));
  set_variant("%s_x%d_y%d_k%d_r%d", tag, T::BX, T::BY, T::BKB, NSTAGE);
  return UNIT_OK;
}

// Which tile.  xs, ys: rows of the two operands of a group, the first one's on average over the groups that can have any; only the
// device knows how many each has.  us, measured on both sides of each line (rows x K -> N over groups; * the one taken):
//   FEW     32 rows, two to six workgroups a CU: up to 32 rows a group, and 64 tiles of 32 x 128
//             fp16 16 x 1024 -> 2048 over 16:   FEW *8.2, SMALL 8.9     46 x 3592 -> 264 over 11:  FEW 21.4, SMALL *16.2
//   SMALL   64 x 64, three workgroups a CU: fewer than 192 tiles of 128 x 128
//             MXFP4 1911 x 3280 -> 600:         SMALL *15.2, MIDDLE 18.1  1277 x 1376 -> 2704 over 2: SMALL 14.5, MIDDLE *11.6
//   MIDDLE  128 x 128, two a CU
//   LARGE   256 x 256, one a CU: at least half of the CUs get one, 512 bytes of reduction and 2^32 products in all
//             bf16 16384 x 1024 -> 2048 over 32: MIDDLE 103, LARGE *90    MXFP4 14826 x 384 -> 2176: MIDDLE *32.6, LARGE 39.5
//             fp16 gradients 1000 x 520 -> 776 over 12: SMALL *17.6, MIDDLE 20.6, LARGE 36.4
//   ROUND   192 x 256, one a CU, 16-bit forward products and data gradients: one round of them rather than most of one of 256.  Only
//           where it is one round however the rows fall on the groups (each may end one row into a tile): a second one costs more
//           than the first gains.
//             bf16 8192 x 2048 -> 1024 over 16 of 512 (192 tiles, 128 of LARGE): forward LARGE 54.3, ROUND *48.1; data gradient 53.2, *46.9
//             bf16 5184 x 1024 -> 2304 (243, 189): forward LARGE 26.5, ROUND *24.7; data gradient 26.7, *24.7
//             bf16 4835 x 3848 -> 2400 (260, 190): forward LARGE *93, ROUND 174     6240 x 1032 -> 1536 over 16 of 390 (288, 192): *27.7, 43.7
// Environment: UNIT_AMD_GROUPED_TILE=1..5 pins one (5 where there is no ROUND: LARGE).
enum { TILE_FEW, TILE_SMALL, TILE_MIDDLE, TILE_LARGE, TILE_ROUND };
inline int grouped_tile_size(const GroupedParams &p, int dir, bool mx) {
  if (const int pinned = tuning_override("UNIT_AMD_GROUPED_TILE")) return pinned - 1;
  const long rows = p.rows ? p.rows : 1, busy = p.groups < rows ? p.groups : rows, mean = (rows + busy - 1) / busy;
  const long xs = dir == GRAD_WEIGHT ? p.n : mean, ys = dir == FORWARD ? p.n : p.k, groups = dir == GRAD_WEIGHT ? p.groups : busy;
  const long k = dir == FORWARD ? p.k : dir == GRAD_DATA ? p.n : mean, kbytes = mx ? k / 2 : k * 2;
  const auto tiles = [&](int x, int y) { return (xs + x - 1) / x * ((ys + y - 1) / y) * groups; };
  if (dir == FORWARD && xs <= 32 && tiles(32, 128) >= 64) return TILE_FEW;
  if (xs >= 192 && ys >= 192 && kbytes >= 512 && tiles(256, 256) >= 128 && xs * ys * groups >= (1l << 32) / k) {
    const bool round = !mx && dir != GRAD_WEIGHT && (p.rows + busy * 191) / 192 * ((ys + 255) / 256) <= 256;
    return round ? TILE_ROUND : TILE_LARGE;
  }
  return tiles(128, 128) >= 192 ? TILE_MIDDLE : TILE_SMALL;
}

template <class Op, int DIR, class Out>
int run_grouped_sizes(const char *what, const char *tag, const GroupedParams &p, hipStream_t s) {
  switch (grouped_tile_size(p, DIR, Op::kMx)) {
    case TILE_FEW:
      if constexpr (DIR == FORWARD) return run_grouped_tile<Op, DIR, Tile<32, 128, 128, 1, 4>, 3, Out>(what, tag, p, s);
      [[fallthrough]];
    case TILE_SMALL: return run_grouped_tile<Op, DIR, Tile<64, 64, 128, 2, 2>, 3, Out>(what, tag, p, s);
    case TILE_MIDDLE: return run_grouped_tile<Op, DIR, Tile<128, 128, 64, 2, 2>, 4, Out>(what, tag, p, s);
    case TILE_ROUND:
      if constexpr (DIR != GRAD_WEIGHT) return run_grouped_tile<Op, DIR, Tile<192, 256, 128, 2, 4>, 2, Out>(what, tag, p, s);
      [[fallthrough]];
    default: return run_grouped_tile<Op, DIR, Tile<256, 256, 128, 2, 4>, 2, Out>(what, tag, p, s);
  }
}

}  // namespace unit
