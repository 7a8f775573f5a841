// MXFP4 products of a handful of rows given as floats, in one launch: the waves of a workgroup share the reduction of 16 columns, each
// with operands straight from memory in its registers, and add their parts through LDS in wave order.
//
// What bounds such a product is the time from its start to its first bytes and, of those, how many are on their way: no launch that
// quantises the rows goes before, nothing is staged, all of a wave's units (128 bytes of its weight rows each) are asked for at once
// where there are no more than four, and there is as little code as will do, for cold code takes longer to fetch than the operands.
//
// v_mfma_scale_f32_16x16x128: lane l holds a block, 32 elements, of row l % 16 at 32 * (l / 16), of the weight (first operand) and of
// the rows (second), and receives columns 4 * (l / 16) .. + 3 of row l % 16.  So each lane quantises its own fragment (largest
// magnitude, scale, conversion) without a word to its neighbours; that every workgroup does so again for the same few rows is cheaper
// than a launch.  1 x 4096 x 4096: 5.3 us, 9.0 as two launches.
//
// Loads are bounded by descriptors: rows past the last, elements past a row's end and units past the last read as zeros.
#pragma once
#include "grouped_tile.hpp"

namespace unit {

constexpr u32 kOutsideSplit = 0x80000000u;  // past every descriptor here

template <class X, int KW, class Out>
__global__ __launch_bounds__(KW * 64, 2) void grouped_split(GroupedParams p, int nts) {
  constexpr int BM = 16, BN = 16, PITCH = BN + 4, DEPTH = 4;
  __shared__ __attribute__((aligned(16))) float part[KW * BM * PITCH];
  const int lane = threadIdx.x & 63, r16 = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));

  GroupTileOf t;
  if (p.sizes) {
    t = find_tile<BM, 4>(p, nts, (int)blockIdx.x, lane);
    if (!t.any) return;
  } else {
    t.group = 0, t.first = 0, t.count = p.rows, t.x0 = 0, t.nt = (int)blockIdx.x;
    if (t.nt >= nts) return;
  }
  const int x0 = t.x0, y0 = t.nt * BN, rows = min(t.count - x0, BM), cols = min(p.n - y0, BN);  // both positive
  const int stages = mx_stages(p.k), ld = stages * 128, units = t.group < p.groups ? stages : 0;
  const long wrows = (long)p.groups * p.n, wrow = (long)t.group * p.n + y0;

  auto buffer = [](const void *base, u32 bytes) {
    const unsigned long long b = (unsigned long long)base;
    const unsigned long long u = (unsigned long long)scalar((u32)b) | (unsigned long long)scalar((u32)(b >> 32)) << 32;
    return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void *>(u), 0, (int)scalar(bytes), 0x00020000);
  };
  const auto wsrc = buffer(p.y + wrow * ld, units ? (u32)cols * (u32)ld : 0);
  const auto xsrc = buffer(reinterpret_cast<const X *>(p.x) + (long)(t.first + x0) * p.k, (u32)rows * (u32)p.k * 2);
  const u32 woff = (u32)r16 * (u32)ld + (u32)q * 16, xoff = (u32)r16 * (u32)p.k * 2 + (u32)q * 64;

  v4f acc = {0, 0, 0, 0};
  v4i w[DEPTH][2], x[DEPTH][2][4];
  u32 ws[DEPTH];
  // this wave's i-th unit; the waves of a workgroup read neighbouring lines at a time
  auto fetch = [&](int i, auto slot) __attribute__((always_inline)) {
    constexpr int S = decltype(slot)::value;
    const int u = wave + i * KW;
    const u32 out = u < units ? 0 : kOutsideSplit;
    const auto ssrc = buffer(p.ys + wrow + (long)u * 2 * wrows, u < units ? 0x7fffffffu : 0);
    ws[S] = (u32)__builtin_amdgcn_raw_buffer_load_b32(ssrc, (int)((u32)(q & 1) * (u32)wrows * 4 + (u32)r16 * 4), 0, 0);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int v = 0; v < 4; ++v) {  // K is a multiple of 8: eight elements are inside or outside together
        const int k = u * kMxStage + h * 128 + q * 32 + v * 8;
        const u32 off = k < p.k ? (xoff + (u32)(u * 512 + h * 256 + v * 16)) | out : kOutsideSplit;
        x[S][h][v] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(xsrc, (int)off, 0, 0));
      }
      w[S][h] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(wsrc, (int)((woff + (u32)(u * 128 + h * 64)) | out), 0, 0));
    }
    __builtin_amdgcn_sched_barrier(0);  // slots are filled in the same order on every path, or the waits become waits for everything
  };
  auto consume = [&](auto slot) __attribute__((always_inline)) {
    constexpr int S = decltype(slot)::value;
    typedef typename Eight<X>::b8 b8;
    const int sw = (int)(ws[S] >> (q & 2) * 4);  // of a dword's four scales this lane's are bytes 0 and 2 now
    auto half_unit = [&](auto hc) __attribute__((always_inline)) {
      constexpr int H = decltype(hc)::value;
      u32 top = 0;
#pragma unroll
      for (int v = 0; v < 4; ++v) top = max(top, eight_top<X>(__builtin_bit_cast(b8, x[S][H][v])));
      const u32 e = mx_scale(top);
      const float scale = mx_power(e == 255 ? 127 : e);
      v8i xf = {};
#pragma unroll
      for (int v = 0; v < 4; ++v) xf[v] = (int)eight_codes<X>(__builtin_bit_cast(b8, x[S][H][v]), scale);
      const v8i wf = {w[S][H][0], w[S][H][1], w[S][H][2], w[S][H][3]};
      acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf, xf, acc, 4, 4, 2 * H, sw, 0, (int)e);
    };
    half_unit(std::integral_constant<int, 0>{});
    half_unit(std::integral_constant<int, 1>{});
    __builtin_amdgcn_sched_barrier(0);
  };
  auto each_slot = [&](auto f) __attribute__((always_inline)) {
    f(std::integral_constant<int, 0>{});
    f(std::integral_constant<int, 1>{});
    f(std::integral_constant<int, 2>{});
    f(std::integral_constant<int, 3>{});
  };
  each_slot([&](auto s) __attribute__((always_inline)) { fetch(decltype(s)::value, s); });
  for (int i = 0; i * KW < units; i += DEPTH)
    each_slot([&](auto s) __attribute__((always_inline)) {
      consume(s);
      fetch(i + DEPTH + decltype(s)::value, s);
    });

  *reinterpret_cast<v4f *>(part + (wave * BM + r16) * PITCH + 4 * q) = acc;
  __syncthreads();
  Out *out = reinterpret_cast<Out *>(p.out) + (long)(t.first + x0) * p.n + y0;
  for (int i = threadIdx.x; i < rows * BN; i += KW * 64) {
    const int row = i / BN, c = i % BN;
    if (c >= cols) continue;
    float s = part[row * PITCH + c];
#pragma unroll
    for (int k = 1; k < KW; ++k) s += part[(k * BM + row) * PITCH + c];
    out[(long)row * p.n + c] = (Out)s;  // the one rounding
  }
}

// Which products take it: as many workgroups as the chip holds at once.  More rows or columns are better off quantised once.
inline bool grouped_split_pays(const GroupedParams &p) {
  const long parts = p.sizes ? (p.groups + 1 < p.rows ? p.groups + 1 : p.rows) : 1;
  return p.rows <= 16 && parts * ceil_div(p.n, 16) <= 512;
}

template <class X, class Out>
int run_grouped_split(const char *what, const GroupedParams &p, hipStream_t s) {
  constexpr int KW = 4;
  const int nts = ceil_div(p.n, 16);
  const long parts = p.sizes ? (p.groups + 1 < p.rows ? p.groups + 1 : p.rows) : 1;
  const long wgs = parts * nts + 7;  // rows are at most 16: a tile per part; + 7 as in run_grouped_tile
  auto kern = grouped_split<X, KW, Out>;
  hipLaunchKernelGGL(kern, dim3((unsigned)wgs), dim3(KW * 64), 0, s, p, nts);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(UNIT_E_LAUNCH, "%s: launch: %s", what, hipGetErrorString(e));
  set_variant("mxdense_split_x16_y16_g%d", KW);
  return UNIT_OK;
}

}  // namespace unit
