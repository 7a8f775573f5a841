// Gated 16-bit products of a handful of rows: the waves of a workgroup share the reduction of 16 columns of the gate and the same 16 of the
// up projection, with operands straight from memory in their registers, add their parts through LDS in wave order and finish h there.
//
// Such a product reads its weight once and does next to nothing with it: what bounds it is the time from its start to its first bytes and how
// many are on their way.  Nothing is staged, a wave asks for four units (128 bytes of each of its 32 weight rows) at once and there
// is as little code as will do.  1 x 2048 -> 4096, bf16: 9.0 us, 12.5 by tiles.
//
// v_mfma_f32_16x16x32: lane l holds eight elements of row l % 16 at 8 * (l / 16), of the weight (first operand) and of the rows (second), and
// receives columns 4 * (l / 16) .. + 3 of row l % 16.  Loads are bounded by descriptors: rows past the last and elements past a row's end
// read as zeros.
#pragma once
#include "grouped_tile.hpp"

namespace unit {

constexpr int kSplitRows = 16;

// CB: blocks of 16 columns per workgroup; two where pre-activations are kept in MXFP8, whose blocks are 32 wide.  The order of every sum is
// that of KW alone.
template <class Half, int KW, class Out, int GATE>
__global__ __launch_bounds__(KW * 64, 2) void gated_split(GatedParams p, int nts) {
  constexpr int BM = kSplitRows, CB = GATE == GATE_KEEP8 ? 2 : 1, BN = 16 * CB, PITCH = BN + 4, DEPTH = 4;
  constexpr u32 kOut = 0x80000000u;  // past every descriptor here
  __shared__ __attribute__((aligned(16))) float part[2 * KW * BM * PITCH];
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
  const u32 ld = (u32)p.k * 2;
  const int units = t.group < p.groups ? (int)((ld + 127) / 128) : 0;

  auto buffer = [](const void *base, u32 bytes) {
    const unsigned long long b = (unsigned long long)base;
    const unsigned long long u = (unsigned long long)scalar((u32)b) | (unsigned long long)scalar((u32)(b >> 32)) << 32;
    return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void *>(u), 0, (int)scalar(bytes), 0x00020000);
  };
  const char *w = p.y + ((long)t.group * 2 * p.n + y0) * (long)ld;
  const u32 wbytes = units ? (u32)cols * ld : 0;
  const auto gsrc = buffer(w, wbytes), usrc = buffer(w + (long)p.n * ld, wbytes);
  const auto xsrc = buffer(p.x + (long)(t.first + x0) * (long)ld, (u32)rows * ld);
  const u32 off0 = (u32)r16 * ld + (u32)q * 16;

  v4f acc[2][CB];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int c = 0; c < CB; ++c) acc[m][c] = v4f{0, 0, 0, 0};
  v4i wf[DEPTH][2][CB][2], xf[DEPTH][2];
  auto load = [](auto src, u32 off) __attribute__((always_inline)) { return __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(src, (int)off, 0, 0)); };
  // this wave's i-th unit; the waves of a workgroup read neighbouring lines at a time
  auto fetch = [&](int i, auto slot) __attribute__((always_inline)) {
    constexpr int S = decltype(slot)::value;
    const int u = wave + i * KW;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const u32 at = (u32)(u * 128 + h * 64);
      const bool in = at + (u32)q * 16 < ld;  // K is a multiple of 8: eight elements are inside or outside together
      xf[S][h] = load(xsrc, in ? off0 + at : kOut);
#pragma unroll
      for (int c = 0; c < CB; ++c) {
        const u32 off = in ? off0 + (u32)c * 16 * ld + at : kOut;
        wf[S][0][c][h] = load(gsrc, off);
        wf[S][1][c][h] = load(usrc, off);
      }
    }
    __builtin_amdgcn_sched_barrier(0);  // slots are filled in the same order on every path, or the waits become waits for everything
  };
  auto consume = [&](auto slot) __attribute__((always_inline)) {
    constexpr int S = decltype(slot)::value;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int c = 0; c < CB; ++c) {
          if constexpr (std::is_same_v<Half, _Float16>)
            acc[m][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, wf[S][m][c][h]), __builtin_bit_cast(v8h, xf[S][h]), acc[m][c], 0, 0, 0);
          else
            acc[m][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8b, wf[S][m][c][h]), __builtin_bit_cast(v8b, xf[S][h]), acc[m][c], 0, 0, 0);
        }
    __builtin_amdgcn_sched_barrier(0);
  };
  // f on slots FROM .. TO - 1
  auto slots = [&](auto from, auto to, auto f) __attribute__((always_inline)) {
    constexpr int FROM = decltype(from)::value, TO = decltype(to)::value;
    if constexpr (FROM <= 0 && 0 < TO) f(std::integral_constant<int, 0>{});
    if constexpr (FROM <= 1 && 1 < TO) f(std::integral_constant<int, 1>{});
    if constexpr (FROM <= 2 && 2 < TO) f(std::integral_constant<int, 2>{});
    if constexpr (FROM <= 3 && 3 < TO) f(std::integral_constant<int, 3>{});
  };
  using none = std::integral_constant<int, 0>;
  using all = std::integral_constant<int, DEPTH>;
  // call(n) with n < DEPTH as a constant: no load is issued that brings nothing, and every path fills the slots in one order
  auto counted = [&](int n, auto call) __attribute__((always_inline)) {
    if (n == 0) call(none{});
    else if (n == 1) call(std::integral_constant<int, 1>{});
    else if (n == 2) call(std::integral_constant<int, 2>{});
    else call(std::integral_constant<int, 3>{});
  };
  const int mine = units > wave ? (units - wave + KW - 1) / KW : 0;
  if (mine < DEPTH) {
    counted(mine, [&](auto n) __attribute__((always_inline)) {
      slots(none{}, n, [&](auto s) __attribute__((always_inline)) { fetch(decltype(s)::value, s); });
      slots(none{}, n, consume);
    });
  } else {
    slots(none{}, all{}, [&](auto s) __attribute__((always_inline)) { fetch(decltype(s)::value, s); });
    int i = DEPTH;
    for (; i + DEPTH <= mine; i += DEPTH)
      slots(none{}, all{}, [&](auto s) __attribute__((always_inline)) {
        consume(s);
        fetch(i + decltype(s)::value, s);
      });
    counted(mine - i, [&](auto n) __attribute__((always_inline)) {
      slots(none{}, n, [&](auto s) __attribute__((always_inline)) {
        consume(s);
        fetch(i + decltype(s)::value, s);
      });
      slots(n, all{}, consume);
      slots(none{}, n, consume);
    });
  }

#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int c = 0; c < CB; ++c) *reinterpret_cast<v4f *>(part + ((m * KW + wave) * BM + r16) * PITCH + 16 * c + 4 * q) = acc[m][c];
  __syncthreads();
  const auto sum = [&](int m, int row, int c) __attribute__((always_inline)) {
    float s = part[(m * KW * BM + row) * PITCH + c];
#pragma unroll
    for (int k = 1; k < KW; ++k) s += part[((m * KW + k) * BM + row) * PITCH + c];
    return s;
  };
  const long row0 = t.first + x0;
  for (int i = threadIdx.x; i < rows * BN; i += KW * 64) {
    const int row = i / BN, c = i % BN;
    if (c >= cols) continue;
    const float g = sum(0, row, c), u = sum(1, row, c);
    reinterpret_cast<Out *>(p.out)[(row0 + row) * p.n + y0 + c] = (Out)(act_value(p.act, g) * u);
    if constexpr (GATE == GATE_KEEP) {
      Half *pre = reinterpret_cast<Half *>(p.pre) + (row0 + row) * 2 * p.n + y0 + c;
      pre[0] = (Half)g, pre[p.n] = (Half)u;
    }
  }
  if constexpr (GATE == GATE_KEEP8) {
    // a block of a row in eight lanes, four columns each
    const int nb = mx8_blocks(p.n);
    for (int i = threadIdx.x; i < 2 * BM * 8; i += KW * 64) {
      const int m = i / (BM * 8), row = i / 8 % BM, c = i % 8 * 4;
      v4f f;
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = c + e < cols ? sum(m, row, c + e) : 0.0f;
      const v4u bits = __builtin_bit_cast(v4u, f);
      u32 top = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) top = max(top, bits[e] & 0x7fffffffu);
#pragma unroll
      for (int d = 1; d < 8; d *= 2) top = max(top, (u32)__shfl_xor((int)top, d));
      if (row >= rows) continue;
      const u32 s = mx8_scale(top);
      const long half = (row0 + row) * 2 + m;
      *reinterpret_cast<u32 *>(p.pre + half * nb * 32 + y0 + c) = four_codes8(f, mx_power(s == 255 ? 127 : s));
      if (c == 0) p.pre_scales[half * nb + (y0 >> 5)] = (char)s;
    }
  }
}

template <class Half, int KW, class Out, int GATE>
int launch_gated_split(const char *what, const char *tag, const GatedParams &p, long parts, hipStream_t s) {
  const int nts = ceil_div(p.n, GATE == GATE_KEEP8 ? 32 : 16);
  const long wgs = parts * nts + 7;  // rows are at most 16: a tile per part; + 7 as in run_grouped_tile
  hipLaunchKernelGGL((gated_split<Half, KW, Out, GATE>), dim3((unsigned)wgs), dim3(KW * 64), 0, s, p, nts);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(UNIT_E_LAUNCH, "%s: launch: %s", what, hipGetErrorString(e));
  set_variant("%s_split_x16_g%d", tag, KW);
  return UNIT_OK;
}

// Eight waves a workgroup while there is at most one of them a CU, else four.  us, four and eight, bf16: 1 x 2048 -> 4096 (256 of them) 10.4, 9.0;
// 16 x 1024 -> 2048 over 16 (2048, nine in sixteen at work) 16.1, 21.2
template <class Half, class Out, int GATE>
int run_gated_split(const char *what, const char *tag, const GatedParams &p, hipStream_t s) {
  const long parts = p.sizes ? (p.groups + 1 < p.rows ? p.groups + 1 : p.rows) : 1;
  if (parts * ceil_div(p.n, 16) <= 256) return launch_gated_split<Half, 8, Out, GATE>(what, tag, p, parts, s);
  return launch_gated_split<Half, 4, Out, GATE>(what, tag, p, parts, s);
}

}  // namespace unit
