// Gated feed-forward products: entry points, and the gradients of the gate itself.
#include "grouped_checks.hpp"
#include "gated.hpp"

namespace unit {
namespace {

int check_activation(const char *what, int code, Activation *a) {
  return activation_of(code, a) ? UNIT_OK : fail(UNIT_E_ARG, "%s: activation must be UNIT_SILU or UNIT_GELU_TANH, got %d", what, code);
}

// both halves of a weight are products of N columns each
int check_gated(const char *what, const void *sizes, int size_bytes, int rows, int groups, int N, int K, size_t w_bytes) {
  if (N > 1 << 21) return fail(UNIT_E_ARG, "%s: more than 2^21 columns", what);
  return check_groups(what, sizes, size_bytes, rows, groups, N, K, w_bytes);
}

// dw from the float32 sums of the splits, added in their order, four elements a lane
template <class Out>
__global__ __launch_bounds__(256) void add_splits_kernel(const v4f *parts, Out *out, long quads, int splits) {
  typedef Out v4o __attribute__((ext_vector_type(4)));
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= quads) return;
  v4f sum = parts[i];
#pragma unroll 4
  for (int s = 1; s < splits; ++s) sum += parts[s * quads + i];
  v4o v;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = (Out)sum[e];  // the one rounding
  reinterpret_cast<v4o *>(out)[i] = v;
}

int add_splits(const char *what, const void *parts, void *out, int out_dtype, long elements, int splits, hipStream_t s) {
  const long quads = elements / 4;  // N and K are multiples of 8
  const dim3 grid((unsigned)((quads + 255) / 256));
  const v4f *p = static_cast<const v4f *>(parts);
  if (out_dtype == UNIT_F32)
    hipLaunchKernelGGL(add_splits_kernel<float>, grid, dim3(256), 0, s, p, static_cast<float *>(out), quads, splits);
  else if (out_dtype == UNIT_F16)
    hipLaunchKernelGGL(add_splits_kernel<_Float16>, grid, dim3(256), 0, s, p, static_cast<_Float16 *>(out), quads, splits);
  else
    hipLaunchKernelGGL(add_splits_kernel<__bf16>, grid, dim3(256), 0, s, p, static_cast<__bf16 *>(out), quads, splits);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? UNIT_OK : fail(UNIT_E_LAUNCH, "%s: launch: %s", what, hipGetErrorString(e));
}

// dpre from dh and the pre-activations, eight columns a lane: 16 bytes of each of three operands in, of each of two results out (six,
// eight and two in MXFP8), which is what it is bound by: 8192 x 2048, bf16, 168 MB in 26.8 us (6.3 TB/s).  Workgroups past the first `gates`
// restore rows from MXFP8 for the product that follows: a launch less (777 x 776 beside 777 x 1032: 8.0 us in two, 5.3 in one).
template <class Half, bool MX8, int ROUNDS>
__global__ __launch_bounds__(256) void gate_grad_kernel(const char *pre, const unsigned char *scales, const Half *dh, Half *dpre, int pieces, int N, Activation act,
                                                        FastDiv by_row, int gates, Mx8Rows<Half> rows) {
  if ((int)blockIdx.x >= gates) return restore_pieces<Half, ROUNDS>(rows, (int)blockIdx.x - gates);
  typedef Half v8h __attribute__((ext_vector_type(8)));
  const int first = (int)blockIdx.x * (256 * ROUNDS) + (int)threadIdx.x, blocks = mx8_blocks(N);
  v4u z[ROUNDS][2], d[ROUNDS];
  u32 s[ROUNDS][2];
  int row[ROUNDS], c[ROUNDS];
#pragma unroll
  for (int i = 0; i < ROUNDS; ++i) {
    by_row.divmod(min(first + i * 256, pieces - 1), row[i], c[i]);
    d[i] = *reinterpret_cast<const v4u *>(dh + (size_t)row[i] * N + c[i] * 8);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const size_t half = (size_t)row[i] * 2 + h;
      if constexpr (MX8) {
        const v2u codes = *reinterpret_cast<const v2u *>(pre + half * (blocks * 32) + c[i] * 8);
        z[i][h] = v4u{codes[0], codes[1], 0, 0};
        s[i][h] = scales[half * blocks + (c[i] >> 2)];
      } else {
        z[i][h] = *reinterpret_cast<const v4u *>(pre + (half * N + c[i] * 8) * 2);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < ROUNDS; ++i) {
    if (first + i * 256 >= pieces) break;
    float f[2][8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if constexpr (MX8) {
        const float p = mx8_power(s[i][h]);
        const v4f lo = four_values8(z[i][h][0], p), hi = four_values8(z[i][h][1], p);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[h][j] = j < 4 ? lo[j] : hi[j - 4];
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[h][j] = (float)__builtin_bit_cast(v8h, z[i][h])[j];
      }
    }
    v8h dg, du;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float slope;
      const float a = act_both(act, f[0][j], &slope), g = (float)__builtin_bit_cast(v8h, d[i])[j];
      // the operands of the products that follow: rounded to their type here, once
      dg[j] = (Half)(g * f[1][j] * slope);
      du[j] = (Half)(g * a);
    }
    Half *dst = dpre + (size_t)row[i] * 2 * N + c[i] * 8;
    *reinterpret_cast<v8h *>(dst) = dg;
    *reinterpret_cast<v8h *>(dst + N) = du;
  }
}

// the rows that are restored beside the gate's gradients: at most 2^30 pieces of both
struct Restored {
  const void *codes = nullptr, *scales = nullptr;
  void *out = nullptr;
  int K = 0;
};
inline bool fits_one_launch(int rows, int N, int K) { return (long)rows * (N / 8) <= 1 << 30 && (long)rows * 4 * mx8_blocks(K) <= 1 << 30; }

template <class Half, bool MX8>
int run_gate_grad(const char *what, const void *pre, const void *scales, const void *dh, void *dpre, int rows, int N, const Activation &act, const Restored &x,
                  hipStream_t s) {
  const FastDiv by_row = FastDiv::make(N / 8);
  const int slice = (1 << 30) / (N / 8);  // rows whose pieces are counted in 31 bits
  for (int row = 0; row < rows; row += slice) {
    const int pieces = (rows - row < slice ? rows - row : slice) * (N / 8);
    const size_t pre_row = MX8 ? (size_t)mx8_blocks(N) * 64 : (size_t)N * 4;
    const char *z = static_cast<const char *>(pre) + row * pre_row;
    const unsigned char *zs = MX8 ? static_cast<const unsigned char *>(scales) + (size_t)row * 2 * mx8_blocks(N) : nullptr;
    const Half *d = static_cast<const Half *>(dh) + (size_t)row * N;
    Half *out = static_cast<Half *>(dpre) + (size_t)row * 2 * N;
    const int per_row = x.codes ? 4 * mx8_blocks(x.K) : 1;
    const Mx8Rows<Half> restored{static_cast<const v2u *>(x.codes), static_cast<const unsigned char *>(x.scales), x.codes ? rows * per_row : 0, x.K,
                                 static_cast<Half *>(x.out), FastDiv::make(per_row)};
    const auto launch = [&](auto kern, int per) {  // pieces a workgroup
      const unsigned gates = (unsigned)((pieces + per - 1) / per), more = (unsigned)((restored.pieces + per - 1) / per);
      hipLaunchKernelGGL(kern, dim3(gates + more), dim3(256), 0, s, z, zs, d, out, pieces, N, act, by_row, (int)gates, restored);
    };
    if (pieces >= 512 * 1024)  // two pieces a lane while that makes four workgroups a CU
      launch(gate_grad_kernel<Half, MX8, 2>, 512);
    else
      launch(gate_grad_kernel<Half, MX8, 1>, 256);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fail(UNIT_E_LAUNCH, "%s: launch: %s", what, hipGetErrorString(e));
    if (row > rows - slice) break;  // row + slice may pass 2^31
  }
  set_variant(MX8 ? "gategrad_mx8" : "gategrad");
  return UNIT_OK;
}

}  // namespace

PairPlan gated_pair_plan(int rows, int groups, bool one_group, int both, int k) {
  struct Cost {
    int x, y;
    double a, b;
  };
  struct Form {
    Cost dx, dw;
    int slots;
  };
  static const Form forms[] = {{{64, 64, 3.5, 0.3}, {128, 128, 7, 0.5}, 512},
                               {{128, 128, 6, 0.34}, {128, 128, 6, 0.34}, 256},
                               {{192, 256, 6, 0.95}, {256, 256, 10, 0.95}, 256},
                               {{256, 256, 10, 0.95}, {256, 256, 10, 0.95}, 256},
                               {{128, 256, 8, 1.05}, {128, 256, 8, 1.05}, 512}};
  const double r = rows > 0 ? rows : 1, busy = groups < r ? groups : r;
  const auto up = [](double v, int d) { return (double)(long)((v + d - 1) / d); };
  const int pinned = tuning_override("UNIT_AMD_GATED_PAIR"), pinned_splits = tuning_override("UNIT_AMD_GATED_SPLITS");
  PairPlan best{PAIR_SMALL, 1, 0};
  double least = 1e300;
  for (int f = 0; f < 5; ++f)
    for (int splits = 1; splits <= 16; splits *= 2) {
      if (pinned > 0 ? f != pinned - 1 : f == PAIR_TALL && one_group) continue;
      // a split has 512 rows at least
      if (pinned_splits > 0 && one_group ? splits != pinned_splits : splits > 1 && (!one_group || r < 512.0 * splits)) continue;
      const Form &m = forms[f];
      const double dx_tiles = (one_group ? up(r, m.dx.x) : r / m.dx.x + busy / 2) * up(k, m.dx.y), dw_tiles = (double)groups * splits * up(both, m.dw.x) * up(k, m.dw.y);
      const double rows_w = r / groups / splits, tx = m.dx.a + m.dx.b * both / 64, tw = m.dw.a + m.dw.b * rows_w / 64;
      const double longest_w = m.dw.a + m.dw.b * (one_group ? 1 : 2) * rows_w / 64, longest = tx > longest_w ? tx : longest_w;
      const double total = (dx_tiles * tx + dw_tiles * tw) / m.slots;
      double us = (total > longest ? total : longest) + 0.25 * (total > longest ? longest : total);
      if (splits > 1) us += 4 + (splits + 0.5) * 2.0 * both * k * 4 / 5e6;  // the sums written and read, and a launch
      if (us < least) {
        least = us;
        best = {static_cast<PairTiles>(f), splits, (int)(up(up(r, splits), 64) * 64)};
      }
    }
  while (best.splits > 1 && (long)(best.splits - 1) * best.split_rows >= rows) --best.splits;  // none without rows
  return best;
}

}  // namespace unit

using namespace unit;

extern "C" int unit_gated_dense(const void *x, const void *w, const void *sizes, int32_t size_bytes, void *out, int32_t dtype, int32_t out_dtype, int32_t activation,
                                void *pre, void *pre_scales, int32_t pre_dtype, int32_t rows, int32_t groups, int32_t N, int32_t K, unit_stream_t stream) {
  const char *what = "unit_gated_dense";
  Activation act;
  if (int rc = check_types(what, dtype, out_dtype)) return rc;
  if (int rc = check_activation(what, activation, &act)) return rc;
  if (int rc = check_gated(what, sizes, size_bytes, rows, groups, N, K, (size_t)N * K * 4)) return rc;
  if (int rc = check_f16(what, N, K)) return rc;
  if (pre && pre_dtype != dtype && pre_dtype != UNIT_MXFP8) return fail(UNIT_E_ARG, "%s: pre_dtype must be the operands' type or UNIT_MXFP8, got %d", what, pre_dtype);
  const int gate = !pre ? GATE_ONLY : pre_dtype == UNIT_MXFP8 ? GATE_KEEP8 : GATE_KEEP;
  if (int rc = check_ptrs(what, rows, {x, w, out})) return rc;
  if (int rc = check_aligned(what, {pre})) return rc;
  if (gate == GATE_KEEP8 && rows && !pre_scales) return fail(UNIT_E_ARG, "%s: null pointer", what);
  if (int rc = check_device()) return rc;
  if (!rows) return UNIT_OK;
  GatedParams p{{static_cast<const char *>(x), static_cast<const char *>(w), nullptr, nullptr, static_cast<char *>(out), sizes, size_bytes, groups, rows, N, K},
                act, static_cast<char *>(pre), static_cast<char *>(pre_scales), nullptr};
  return (dtype == UNIT_F16 ? run_gated_f16 : run_gated_bf16)(what, gate, p, out_dtype, static_cast<hipStream_t>(stream));
}

extern "C" int unit_gated_dense_mxfp4(const void *x, const void *xscales, int32_t x_dtype, const void *wcodes, const void *wscales, const void *sizes,
                                      int32_t size_bytes, void *out, int32_t out_dtype, int32_t activation, int32_t rows, int32_t groups, int32_t N, int32_t K, void *ws,
                                      size_t ws_bytes, unit_stream_t stream) {
  const char *what = "unit_gated_dense_mxfp4";
  Activation act;
  if (int rc = check_activation(what, activation, &act)) return rc;
  if (int rc = check_gated(what, sizes, size_bytes, rows, groups, N, K, N > 0 && K > 0 ? mx_code_bytes(2l * N, K) : 0)) return rc;
  GatedParams p{{static_cast<const char *>(x), static_cast<const char *>(wcodes), static_cast<const u32 *>(xscales), static_cast<const u32 *>(wscales),
                 static_cast<char *>(out), sizes, size_bytes, groups, rows, N, K, x_dtype}, act, nullptr, nullptr, nullptr};
  bool run;
  if (int rc = mxfp4_rows(what, &p, out_dtype, ws, ws_bytes, static_cast<hipStream_t>(stream), gated_mx_takes_floats, &run)) return rc;
  return run ? run_gated_mx(what, p, out_dtype, static_cast<hipStream_t>(stream)) : UNIT_OK;
}

namespace {

// The parts of the workspace of a gradient: dpre, the rows restored from MXFP8, float32 sums of dw's splits (of one group's dw beside dx)
struct GradParts {
  size_t dpre, x, sums;
  GradParts(bool restored, bool shared_out, int rows, int N, int K) {
    const auto lines = [](size_t bytes) { return (bytes + 255) / 256 * 256; };
    const int splits = shared_out && rows ? gated_pair_plan(rows, 1, true, 2 * N, K).splits : 1;
    dpre = lines((size_t)rows * N * 4);
    x = restored ? lines((size_t)rows * K * 2) : 0;
    sums = splits > 1 ? (size_t)splits * N * K * 8 : 0;
  }
  size_t bytes() const { return dpre + x + sums; }
};

int check_grad_shape(const char *what, int x_dtype, int dtype, int rows, int groups, int N, int K) {
  if (dtype != UNIT_F16 && dtype != UNIT_BF16) return fail(UNIT_E_ARG, "%s: dtype must be UNIT_F16 or UNIT_BF16, got %d", what, dtype);
  if (x_dtype != dtype && x_dtype != UNIT_MXFP8) return fail(UNIT_E_ARG, "%s: x_dtype must be dtype or UNIT_MXFP8, got %d", what, x_dtype);
  const int unused = 0;
  if (int rc = check_gated(what, &unused, 4, rows, groups, N, K, N > 0 && K > 0 ? (size_t)N * K * 4 : 0)) return rc;
  return check_f16(what, N, K);
}

}  // namespace

namespace {

int workspace(const char *what, bool both, int x_dtype, int dtype, int rows, int groups, int N, int K, size_t *bytes) {
  if (int rc = check_grad_shape(what, x_dtype, dtype, rows, groups, N, K)) return rc;
  if (!bytes) return fail(UNIT_E_ARG, "%s: null pointer", what);
  *bytes = GradParts(x_dtype == UNIT_MXFP8, both && groups == 1, rows, N, K).bytes();
  return UNIT_OK;
}

}  // namespace

extern "C" int unit_gated_dense_grad_ws_bytes(int32_t x_dtype, int32_t dtype, int32_t rows, int32_t groups, int32_t N, int32_t K, size_t *bytes) {
  return workspace("unit_gated_dense_grad_ws_bytes", true, x_dtype, dtype, rows, groups, N, K, bytes);
}

extern "C" int unit_gated_dense_grad_one_ws_bytes(int32_t x_dtype, int32_t dtype, int32_t rows, int32_t groups, int32_t N, int32_t K, size_t *bytes) {
  return workspace("unit_gated_dense_grad_one_ws_bytes", false, x_dtype, dtype, rows, groups, N, K, bytes);
}

extern "C" int unit_gated_dense_grad(const void *x, const void *x_scales, int32_t x_dtype, const void *w, const void *dh, const void *pre, const void *pre_scales,
                                     int32_t pre_dtype, const void *sizes, int32_t size_bytes, void *dx, int32_t dx_dtype, void *dw, int32_t dw_dtype, int32_t dtype,
                                     int32_t activation, int32_t rows, int32_t groups, int32_t N, int32_t K, void *ws, size_t ws_bytes, unit_stream_t stream) {
  const char *what = "unit_gated_dense_grad";
  Activation act;
  if (int rc = check_grad_shape(what, x_dtype, dtype, rows, groups, N, K)) return rc;
  if (int rc = check_groups(what, sizes, size_bytes, rows, groups, N, K, 0)) return rc;
  if (int rc = check_activation(what, activation, &act)) return rc;
  if (dx && dx_dtype != UNIT_F32 && dx_dtype != dtype) return fail(UNIT_E_ARG, "%s: out_dtype of dx must be UNIT_F32 or dtype, got %d", what, dx_dtype);
  if (dw && dw_dtype != UNIT_F32 && dw_dtype != dtype) return fail(UNIT_E_ARG, "%s: out_dtype of dw must be UNIT_F32 or dtype, got %d", what, dw_dtype);
  if (pre && pre_dtype != dtype && pre_dtype != UNIT_MXFP8) return fail(UNIT_E_ARG, "%s: pre_dtype must be dtype or UNIT_MXFP8, got %d", what, pre_dtype);
  const bool needs_x = dw || !pre, x8 = x_dtype == UNIT_MXFP8;
  const GradParts parts(x8 && needs_x, dx && dw && !sizes, rows, N, K);
  if (int rc = check_ptrs(what, rows, {w, dh, ws})) return rc;
  if (int rc = check_ptrs(what, rows && needs_x, {x})) return rc;
  if (int rc = check_aligned(what, {pre, dx, dw})) return rc;
  if (rows && ((x8 && needs_x && !x_scales) || (pre && pre_dtype == UNIT_MXFP8 && !pre_scales))) return fail(UNIT_E_ARG, "%s: null pointer", what);
  if (ws_bytes < parts.bytes()) return fail(UNIT_E_ARG, "%s: workspace of %zu bytes, %zu needed", what, ws_bytes, parts.bytes());
  if (int rc = check_device()) return rc;
  if (!dx && !dw) return UNIT_OK;
  hipStream_t s = static_cast<hipStream_t>(stream);
  char *const dpre = static_cast<char *>(ws);
  Restored restored;
  if (x8 && needs_x && rows) {
    char *const x16 = dpre + parts.dpre;
    if (pre && fits_one_launch(rows, N, K))
      restored = {x, x_scales, x16, K};
    else if (int rc = unit_dequantize_mxfp8(x, x_scales, rows, K, x16, dtype, stream))
      return rc;
    x = x16;
  }
  if (rows && pre) {
    const bool pre8 = pre_dtype == UNIT_MXFP8;
    const auto run = dtype == UNIT_F16 ? (pre8 ? run_gate_grad<_Float16, true> : run_gate_grad<_Float16, false>)
                                       : (pre8 ? run_gate_grad<__bf16, true> : run_gate_grad<__bf16, false>);
    if (int rc = run(what, pre, pre_scales, dh, dpre, rows, N, act, restored, s)) return rc;
  } else if (rows) {
    GatedParams p{{static_cast<const char *>(x), static_cast<const char *>(w), nullptr, nullptr, dpre, sizes, size_bytes, groups, rows, N, K},
                  act, nullptr, nullptr, static_cast<const char *>(dh)};
    if (int rc = (dtype == UNIT_F16 ? run_gated_f16 : run_gated_bf16)(what, GATE_GRAD, p, dtype, s)) return rc;
  }
  if (dx && dw && rows) {
    PairPlan plan = gated_pair_plan(rows, groups, !sizes, 2 * N, K);
    const bool split = plan.splits > 1;
    char *const sums = dpre + parts.dpre + parts.x;
    const auto product = [&](const void *y, void *out) {
      return GroupedParams{dpre, static_cast<const char *>(y), nullptr, nullptr, static_cast<char *>(out), sizes, size_bytes, groups, rows, 2 * N, K};
    };
    // dh, dpre, the rows and dx, w and dw; what was kept
    const size_t weights = (size_t)groups * N * K * 4, half = (size_t)rows * N * 2;
    const size_t kept = !pre ? 0 : pre_dtype == UNIT_MXFP8 ? mx8_code_bytes(2l * rows, N) : 2 * half;
    const size_t moved = kept + 3 * half + (size_t)rows * K * (dx_dtype == UNIT_F32 ? 6 : 4) + 2 * weights;
    GroupedParams pw = product(x, split ? sums : dw);
    pw.past_caches = dw_past_caches(weights, moved, pre != nullptr);
    const auto run = dtype == UNIT_F16 ? run_gated_pair_f16 : run_gated_pair_bf16;
    if (int rc = run(what, product(w, dx), dx_dtype, pw, split ? (int)UNIT_F32 : dw_dtype, plan, s)) return rc;
    return split ? add_splits(what, sums, dw, dw_dtype, 2l * N * K, plan.splits, s) : UNIT_OK;
  }
  if (dx)
    if (int rc = unit_grouped_dense_grad_data(dpre, w, sizes, size_bytes, dx, dtype, dx_dtype, rows, groups, 2 * N, K, stream)) return rc;
  if (dw)
    if (int rc = unit_grouped_dense_grad_weight(x, dpre, sizes, size_bytes, dw, dtype, dw_dtype, rows, groups, 2 * N, K, stream)) return rc;
  return UNIT_OK;
}
