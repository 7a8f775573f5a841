// Grouped products, their gradients and the MXFP4 products: entry points and kernels.
#include "grouped.hpp"

namespace unit {
namespace {

int run_typed(const char *what, int dir, const GroupedParams &p, int dtype, int out_dtype, hipStream_t s) {
  return (dtype == UNIT_F16 ? run_grouped_f16 : run_grouped_bf16)(what, dir, p, out_dtype, s);
}

int check_types(const char *what, int dtype, int out_dtype) {
  if (dtype != UNIT_F16 && dtype != UNIT_BF16) return fail(UNIT_E_ARG, "%s: dtype must be UNIT_F16 or UNIT_BF16, got %d", what, dtype);
  if (out_dtype != UNIT_F32 && out_dtype != dtype) return fail(UNIT_E_ARG, "%s: out_dtype must be UNIT_F32 or the operands' type, got %d", what, out_dtype);
  return UNIT_OK;
}

// sizes and the limits that all of the products share; rows may be 0
int check_groups(const char *what, const void *sizes, int size_bytes, int rows, int groups, int n, int k, size_t w_bytes) {
  if (rows < 0 || groups <= 0 || n <= 0 || k <= 0) return fail(UNIT_E_ARG, "%s: groups, N and K must be positive and rows not negative", what);
  if (size_bytes != 4 && size_bytes != 8) return fail(UNIT_E_ARG, "%s: group sizes are 4- or 8-byte integers, got %d bytes", what, size_bytes);
  if (!sizes) return fail(UNIT_E_ARG, "%s: null pointer", what);
  if ((uintptr_t)sizes % size_bytes) return fail(UNIT_E_ARG, "%s: group sizes are not aligned to their type", what);
  // 32-bit offsets inside one group's weight and inside one tile (a tile of a weight's gradient in fp32 stays below 2^32 bytes with
  // the 16-bit weight below 2^31); the tensors themselves may be larger
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
  return run_typed(what, FORWARD, p, dtype, out_dtype, static_cast<hipStream_t>(stream));
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
  return run_typed(what, GRAD_DATA, p, dtype, out_dtype, static_cast<hipStream_t>(stream));
}

extern "C" int unit_grouped_dense_grad_weight(const void *x, const void *dy, const void *sizes, int32_t size_bytes, void *dw, int32_t dtype, int32_t out_dtype,
                                              int32_t rows, int32_t groups, int32_t N, int32_t K, unit_stream_t stream) {
  const char *what = "unit_grouped_dense_grad_weight";
  if (int rc = check_types(what, dtype, out_dtype)) return rc;
  if (int rc = check_groups(what, sizes, size_bytes, rows, groups, N, K, (size_t)N * K * 2)) return rc;
  if (int rc = check_f16(what, N, K)) return rc;
  if (int rc = check_ptrs(what, rows, {x, dy})) return rc;
  if (int rc = check_ptrs(what, true, {dw})) return rc;
  if (int rc = check_device()) return rc;
  GroupedParams p{static_cast<const char *>(dy), static_cast<const char *>(x), nullptr, nullptr, static_cast<char *>(dw), sizes, size_bytes, groups, rows, N, K};
  return run_typed(what, GRAD_WEIGHT, p, dtype, out_dtype, static_cast<hipStream_t>(stream));
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
  GroupedParams p{static_cast<const char *>(x), static_cast<const char *>(wcodes), static_cast<const u32 *>(xscales), static_cast<const u32 *>(wscales),
                  static_cast<char *>(out), sizes, size_bytes, groups, rows, N, K, x_dtype};
  if (floats && grouped_mx_takes_floats(p)) return run_grouped_mx(what, p, out_dtype, s);
  if (floats) {
    char *buf = static_cast<char *>(ws);
    if (int rc = unit_quantize_mxfp4(x, x_dtype, rows, K, buf, buf + codes, s)) return rc;
    p.x = buf;
    p.xs = reinterpret_cast<const u32 *>(buf + codes);
    p.x_dtype = UNIT_MXFP4;
  }
  return run_grouped_mx(what, p, out_dtype, s);
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
