// Grouped products, their gradients and the MXFP4 products: entry points and kernels.
#include "grouped_checks.hpp"

namespace unit {
namespace {

int run_typed(const char *what, int dir, const GroupedParams &p, int dtype, int out_dtype, hipStream_t s) {
  return (dtype == UNIT_F16 ? run_grouped_f16 : run_grouped_bf16)(what, dir, p, out_dtype, s);
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

int run_mxfp4(const char *what, const void *x, const void *xscales, int x_dtype, const void *wcodes, const void *wscales, const void *sizes, int size_bytes, void *out,
              int out_dtype, int rows, int groups, int N, int K, void *ws, size_t ws_bytes, hipStream_t s) {
  GroupedParams p{static_cast<const char *>(x), static_cast<const char *>(wcodes), static_cast<const u32 *>(xscales), static_cast<const u32 *>(wscales),
                  static_cast<char *>(out), sizes, size_bytes, groups, rows, N, K, x_dtype};
  bool run;
  if (int rc = mxfp4_rows(what, &p, out_dtype, ws, ws_bytes, s, grouped_mx_takes_floats, &run)) return rc;
  return run ? run_grouped_mx(what, p, out_dtype, s) : UNIT_OK;
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
  if (int rc = check_groups(what, nullptr, 4, M, 1, N, K, N > 0 && K > 0 ? mx_code_bytes(N, K) : 0)) return rc;
  return run_mxfp4(what, x, xscales, x_dtype, wcodes, wscales, nullptr, 4, out, out_dtype, M, 1, N, K, ws, ws_bytes, static_cast<hipStream_t>(stream));
}

extern "C" int unit_grouped_dense_mxfp4(const void *x, const void *xscales, int32_t x_dtype, const void *wcodes, const void *wscales, const void *sizes,
                                        int32_t size_bytes, void *out, int32_t out_dtype, int32_t rows, int32_t groups, int32_t N, int32_t K, void *ws, size_t ws_bytes,
                                        unit_stream_t stream) {
  const char *what = "unit_grouped_dense_mxfp4";
  if (int rc = check_groups(what, sizes, size_bytes, rows, groups, N, K, N > 0 && K > 0 ? mx_code_bytes(N, K) : 0)) return rc;
  return run_mxfp4(what, x, xscales, x_dtype, wcodes, wscales, sizes, size_bytes, out, out_dtype, rows, groups, N, K, ws, ws_bytes, static_cast<hipStream_t>(stream));
}
