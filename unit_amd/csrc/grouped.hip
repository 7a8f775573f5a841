// Grouped products, their gradients and the MXFP4 products: entry points and kernels.
#include "grouped.hpp"

namespace unit {
namespace {

enum { FORWARD, GRAD_DATA, GRAD_WEIGHT };

struct OpHalf : OpF16 {
  using elem = _Float16;
};
struct OpMx {
  using elem = void;
};

// The plain kernel: one wave per 32 x 32 block of the result, operands straight from memory into the fragments (lane l:
// row or column l % 32, eight consecutive reduction elements at 8 * (l / 32)).
template <class Op, int DIR, class Out>
__global__ __launch_bounds__(64) void grouped_plain(GroupedParams p) {
  constexpr bool MX = std::is_same_v<Op, OpMx>;
  const int lane = threadIdx.x, l32 = lane & 31, half = lane >> 5;
  int g = 0, first = 0, count = 0, x0 = 0;
  if constexpr (DIR == GRAD_WEIGHT) {
    g = blockIdx.z;
    for (int i = 0; i <= g; ++i) {
      first += count;
      const int s = group_size(p, i);
      count = s < p.rows - first ? s : p.rows - first;
    }
    x0 = blockIdx.x * 32;
  } else {
    int tile = blockIdx.x;
    for (;; ++g) {
      first += count;
      const int s = g < p.groups ? group_size(p, g) : p.rows;
      count = s < p.rows - first ? s : p.rows - first;
      const int tiles = (count + 31) / 32;
      if (tile < tiles) break;
      tile -= tiles;
      if (g == p.groups) return;
    }
    x0 = tile * 32;
  }
  const int y0 = blockIdx.y * 32;
  v16f acc;
#pragma unroll
  for (int r = 0; r < 16; ++r) acc[r] = 0;
  // extents of the result block: rows (columns) of this tile's group
  const int xs = DIR == GRAD_WEIGHT ? p.n : count, ys = DIR == FORWARD ? p.n : p.k;
  const int xr = x0 + l32 < xs ? x0 + l32 : xs - 1, yr = y0 + l32 < ys ? y0 + l32 : ys - 1;  // in bounds; surplus ones are not stored
  if (DIR == GRAD_WEIGHT || g < p.groups) {
    if constexpr (MX) {
      const int stages = mx_stages(p.k);
      const size_t ld = (size_t)stages * 128;
      const size_t row = (size_t)first + xr, col = (size_t)g * p.n + yr;
      for (int s = 0; s < stages; ++s) {
        const u32 sx = p.xs[(size_t)(2 * s + half) * p.rows + row], sy = p.ys[(size_t)(2 * s + half) * p.groups * p.n + col];
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          const v4i x = *reinterpret_cast<const v4i *>(p.x + row * ld + s * 128 + (2 * kk + half) * 16);
          const v4i y = *reinterpret_cast<const v4i *>(p.y + col * ld + s * 128 + (2 * kk + half) * 16);
          const v8i x8 = {x[0], x[1], x[2], x[3]}, y8 = {y[0], y[1], y[2], y[3]};
          acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(x8, y8, acc, 4, 4, 0, (int)(sx >> 8 * kk), 0, (int)(sy >> 8 * kk));
        }
      }
    } else {
      using E = typename Op::elem;
      typedef E v8e __attribute__((ext_vector_type(8)));
      const E *X = reinterpret_cast<const E *>(p.x), *Y = reinterpret_cast<const E *>(p.y);
      const size_t wrow = (size_t)g * p.n;
      const int K = DIR == FORWARD ? p.k : DIR == GRAD_DATA ? p.n : count;
      for (int k0 = 8 * half; k0 - 8 * half < K; k0 += 16) {
        v8e x, y;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int k = k0 + i;
          x[i] = y[i] = (E)0.0f;
          if (k < K) {
            if constexpr (DIR == FORWARD) {
              x[i] = X[((size_t)first + xr) * p.k + k];
              y[i] = Y[(wrow + yr) * p.k + k];
            } else if constexpr (DIR == GRAD_DATA) {
              x[i] = X[((size_t)first + xr) * p.n + k];
              y[i] = Y[(wrow + k) * p.k + yr];
            } else {
              x[i] = X[((size_t)first + k) * p.n + xr];
              y[i] = Y[((size_t)first + k) * p.k + yr];
            }
          }
        }
        acc = Op::mma(__builtin_bit_cast(v4i, x), __builtin_bit_cast(v4i, y), acc);
      }
    }
  }
  Out *out = reinterpret_cast<Out *>(p.out);
  if (y0 + l32 < ys) {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int x = x0 + 8 * (r >> 2) + 4 * half + (r & 3);
      if (x < xs) out[((DIR == GRAD_WEIGHT ? (size_t)g * p.n : (size_t)first) + x) * ys + y0 + l32] = (Out)acc[r];  // the one rounding
    }
  }
}

template <class Op, int DIR, class Out>
int run_grouped(const char *what, const GroupedParams &p, hipStream_t s) {
  const int ys = DIR == FORWARD ? p.n : p.k;
  dim3 grid;
  if constexpr (DIR == GRAD_WEIGHT) {
    grid = dim3(ceil_div(p.n, 32), ceil_div(ys, 32), p.groups);
  } else {
    // at most: every group (and the rows of none) ends inside a tile
    const long parts = p.sizes ? (p.groups + 1 < p.rows ? p.groups + 1 : p.rows) : 1;
    grid = dim3((unsigned)((p.rows + parts * 31) / 32), ceil_div(ys, 32));
  }
  hipLaunchKernelGGL((grouped_plain<Op, DIR, Out>), grid, dim3(64), 0, s, p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(UNIT_E_LAUNCH, "%s: launch: %s", what, hipGetErrorString(e));
  return UNIT_OK;
}

template <class Op, int DIR>
int run_out(const char *what, const GroupedParams &p, int out_dtype, hipStream_t s) {
  if (out_dtype == UNIT_F32) return run_grouped<Op, DIR, float>(what, p, s);
  if (out_dtype == UNIT_F16) return run_grouped<Op, DIR, _Float16>(what, p, s);
  return run_grouped<Op, DIR, __bf16>(what, p, s);
}

template <int DIR>
int run_typed(const char *what, const GroupedParams &p, int dtype, int out_dtype, hipStream_t s) {
  return dtype == UNIT_F16 ? run_out<OpHalf, DIR>(what, p, out_dtype, s) : run_out<OpBF16, DIR>(what, p, out_dtype, s);
}

int check_types(const char *what, int dtype, int out_dtype) {
  if (dtype != UNIT_F16 && dtype != UNIT_BF16) return fail(UNIT_E_ARG, "%s: dtype must be UNIT_F16 or UNIT_BF16, got %d", what, dtype);
  if (out_dtype != UNIT_F32 && out_dtype != UNIT_F16 && out_dtype != UNIT_BF16)
    return fail(UNIT_E_ARG, "%s: out_dtype must be UNIT_F32, UNIT_F16 or UNIT_BF16, got %d", what, out_dtype);
  return UNIT_OK;
}

// sizes and the limits that all of the products share; rows may be 0
int check_groups(const char *what, const void *sizes, int size_bytes, int rows, int groups, int n, int k, size_t w_bytes) {
  if (rows < 0 || groups <= 0 || n <= 0 || k <= 0) return fail(UNIT_E_ARG, "%s: groups, N and K must be positive and rows not negative", what);
  if (size_bytes != 4 && size_bytes != 8) return fail(UNIT_E_ARG, "%s: group sizes are 4- or 8-byte integers, got %d bytes", what, size_bytes);
  if (!sizes) return fail(UNIT_E_ARG, "%s: null pointer", what);
  if ((uintptr_t)sizes % size_bytes) return fail(UNIT_E_ARG, "%s: group sizes are not aligned to their type", what);
  // 32-bit offsets inside one group's weight and inside one tile; the tensors themselves may be larger
  if (!fits(w_bytes)) return fail(UNIT_E_ARG, "%s: a group's weight exceeds 2^31-1 bytes", what);
  if (rows > 1 << 30 || groups > 1 << 20 || n > 1 << 22 || k > 1 << 22) return fail(UNIT_E_ARG, "%s: sizes beyond 2^30 rows, 2^20 groups or 2^22 columns", what);
  return UNIT_OK;
}

int check_f16(const char *what, int n, int k) {
  if (n % 8 || k % 8) return fail(UNIT_E_ARG, "%s: N and K must be multiples of 8 (16-byte rows), got %d and %d", what, n, k);
  return UNIT_OK;
}

int check_ptrs(const char *what, bool any, std::initializer_list<const void *> ptrs) {
  for (const void *p : ptrs)
    if (!p && any) return fail(UNIT_E_ARG, "%s: null pointer", what);
  return check_aligned(what, ptrs);
}

}  // namespace
}  // namespace unit

using namespace unit;

extern "C" int unit_grouped_dense(const void *x, const void *w, const void *sizes, int32_t size_bytes, void *out, int32_t dtype, int32_t out_dtype, int32_t rows,
                                  int32_t groups, int32_t N, int32_t K, unit_stream_t stream) {
  const char *what = "unit_grouped_dense";
  if (int rc = check_types(what, dtype, out_dtype)) return rc;
  if (int rc = check_groups(what, sizes, size_bytes, rows, groups, N, K, (size_t)N * K * 2)) return rc;
  if (int rc = check_f16(what, N, K)) return rc;
  if (int rc = check_ptrs(what, rows, {x, w, out})) return rc;
  if (int rc = check_device()) return rc;
  if (!rows) return UNIT_OK;
  GroupedParams p{static_cast<const char *>(x), static_cast<const char *>(w), nullptr, nullptr, static_cast<char *>(out), sizes, size_bytes, groups, rows, N, K};
  return run_typed<FORWARD>(what, p, dtype, out_dtype, static_cast<hipStream_t>(stream));
}

extern "C" int unit_grouped_dense_grad_data(const void *dy, const void *w, const void *sizes, int32_t size_bytes, void *dx, int32_t dtype, int32_t out_dtype,
                                            int32_t rows, int32_t groups, int32_t N, int32_t K, unit_stream_t stream) {
  const char *what = "unit_grouped_dense_grad_data";
  if (int rc = check_types(what, dtype, out_dtype)) return rc;
  if (int rc = check_groups(what, sizes, size_bytes, rows, groups, N, K, (size_t)N * K * 2)) return rc;
  if (int rc = check_f16(what, N, K)) return rc;
  if (int rc = check_ptrs(what, rows, {dy, w, dx})) return rc;
  if (int rc = check_device()) return rc;
  if (!rows) return UNIT_OK;
  GroupedParams p{static_cast<const char *>(dy), static_cast<const char *>(w), nullptr, nullptr, static_cast<char *>(dx), sizes, size_bytes, groups, rows, N, K};
  return run_typed<GRAD_DATA>(what, p, dtype, out_dtype, static_cast<hipStream_t>(stream));
}

extern "C" int unit_grouped_dense_grad_weight(const void *x, const void *dy, const void *sizes, int32_t size_bytes, void *dw, int32_t dtype, int32_t out_dtype,
                                              int32_t rows, int32_t groups, int32_t N, int32_t K, unit_stream_t stream) {
  const char *what = "unit_grouped_dense_grad_weight";
  if (int rc = check_types(what, dtype, out_dtype)) return rc;
  if (int rc = check_groups(what, sizes, size_bytes, rows, groups, N, K, (size_t)N * K * 4)) return rc;
  if (int rc = check_f16(what, N, K)) return rc;
  if (int rc = check_ptrs(what, rows, {x, dy})) return rc;
  if (int rc = check_ptrs(what, true, {dw})) return rc;
  if (int rc = check_device()) return rc;
  GroupedParams p{static_cast<const char *>(dy), static_cast<const char *>(x), nullptr, nullptr, static_cast<char *>(dw), sizes, size_bytes, groups, rows, N, K};
  return run_typed<GRAD_WEIGHT>(what, p, dtype, out_dtype, static_cast<hipStream_t>(stream));
}

namespace {

// x: floats, quantised into the workspace first, or codes (with their scales)
int run_mxfp4(const char *what, const void *x, const void *xscales, int x_dtype, const void *wcodes, const void *wscales, const void *sizes, int size_bytes, void *out,
              int out_dtype, int rows, int groups, int N, int K, void *ws, size_t ws_bytes, hipStream_t s) {
  const bool floats = x_dtype != UNIT_MXFP4;
  if (floats && x_dtype != UNIT_F32 && x_dtype != UNIT_F16 && x_dtype != UNIT_BF16)
    return fail(UNIT_E_ARG, "%s: x_dtype must be UNIT_F32, UNIT_F16, UNIT_BF16 or UNIT_MXFP4, got %d", what, x_dtype);
  if (out_dtype != UNIT_F32 && out_dtype != UNIT_F16 && out_dtype != UNIT_BF16)
    return fail(UNIT_E_ARG, "%s: out_dtype must be UNIT_F32, UNIT_F16 or UNIT_BF16, got %d", what, out_dtype);
  const size_t codes = mx_code_bytes(rows, K), need = codes + mx_scale_bytes(rows, K);
  if (int rc = check_ptrs(what, rows, {wcodes, wscales, out})) return rc;
  if (floats && rows && ws_bytes < need) return fail(UNIT_E_ARG, "%s: workspace of %zu bytes, %zu needed", what, ws_bytes, need);
  if (floats) {
    if (int rc = check_ptrs(what, rows, {ws})) return rc;
    if (!x && rows) return fail(UNIT_E_ARG, "%s: null pointer", what);
  } else if (int rc = check_ptrs(what, rows, {x, xscales})) {
    return rc;
  }
  if (int rc = check_device()) return rc;
  if (!rows) return UNIT_OK;
  if (floats) {
    char *buf = static_cast<char *>(ws);
    if (int rc = unit_quantize_mxfp4(x, x_dtype, rows, K, buf, buf + codes, s)) return rc;
    x = buf;
    xscales = buf + codes;
  }
  GroupedParams p{static_cast<const char *>(x), static_cast<const char *>(wcodes), static_cast<const u32 *>(xscales), static_cast<const u32 *>(wscales),
                  static_cast<char *>(out), sizes, size_bytes, groups, rows, N, K};
  return run_out<OpMx, FORWARD>(what, p, out_dtype, s);
}

}  // namespace

extern "C" int unit_mxfp4_workspace_bytes(int32_t rows, int32_t K, size_t *bytes) {
  if (rows < 0 || K <= 0 || !bytes) return fail(UNIT_E_ARG, "unit_mxfp4_workspace_bytes: rows must not be negative, K positive, bytes not null");
  *bytes = mx_code_bytes(rows, K) + mx_scale_bytes(rows, K);
  return UNIT_OK;
}

extern "C" int unit_dense_mxfp4(const void *x, const void *xscales, int32_t x_dtype, const void *wcodes, const void *wscales, void *out, int32_t out_dtype, int32_t M,
                                int32_t N, int32_t K, void *ws, size_t ws_bytes, unit_stream_t stream) {
  const char *what = "unit_dense_mxfp4";
  static const int unused = 0;  // one group, no sizes
  if (int rc = check_groups(what, &unused, 4, M, 1, N, K, N > 0 && K > 0 ? mx_code_bytes(N, K) : 0)) return rc;
  return run_mxfp4(what, x, xscales, x_dtype, wcodes, wscales, nullptr, 4, out, out_dtype, M, 1, N, K, ws, ws_bytes, static_cast<hipStream_t>(stream));
}

extern "C" int unit_grouped_dense_mxfp4(const void *x, const void *xscales, int32_t x_dtype, const void *wcodes, const void *wscales, const void *sizes,
                                        int32_t size_bytes, void *out, int32_t out_dtype, int32_t rows, int32_t groups, int32_t N, int32_t K, void *ws, size_t ws_bytes,
                                        unit_stream_t stream) {
  const char *what = "unit_grouped_dense_mxfp4";
  if (int rc = check_groups(what, sizes, size_bytes, rows, groups, N, K, N > 0 && K > 0 ? mx_code_bytes(N, K) : 0)) return rc;
  return run_mxfp4(what, x, xscales, x_dtype, wcodes, wscales, sizes, size_bytes, out, out_dtype, rows, groups, N, K, ws, ws_bytes, static_cast<hipStream_t>(stream));
}
