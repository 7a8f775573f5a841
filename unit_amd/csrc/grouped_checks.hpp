// What the entry points of the grouped products check, and how those in MXFP4 come by their rows.
#pragma once
#include "grouped.hpp"

namespace unit {

inline int check_types(const char *what, int dtype, int out_dtype) {
  if (dtype != UNIT_F16 && dtype != UNIT_BF16) return fail(UNIT_E_ARG, "%s: dtype must be UNIT_F16 or UNIT_BF16, got %d", what, dtype);
  if (out_dtype != UNIT_F32 && out_dtype != dtype) return fail(UNIT_E_ARG, "%s: out_dtype must be UNIT_F32 or the operands' type, got %d", what, out_dtype);
  return UNIT_OK;
}

// sizes and the limits that all of the products share; rows may be 0
inline int check_groups(const char *what, const void *sizes, int size_bytes, int rows, int groups, int n, int k, size_t w_bytes) {
  if (rows < 0 || groups <= 0 || n <= 0 || k <= 0) return fail(UNIT_E_ARG, "%s: groups, N and K must be positive and rows not negative", what);
  if (size_bytes != 4 && size_bytes != 8) return fail(UNIT_E_ARG, "%s: group sizes are 4- or 8-byte integers, got %d bytes", what, size_bytes);
  if (!sizes && groups != 1) return fail(UNIT_E_ARG, "%s: null pointer", what);  // one group: all rows
  if ((uintptr_t)sizes % size_bytes) return fail(UNIT_E_ARG, "%s: group sizes are not aligned to their type", what);
  // 32-bit offsets inside one group's weight and inside one tile (a tile of a weight's gradient in fp32 stays below 2^32 bytes with
  // the 16-bit weight below 2^31); the tensors themselves may be larger
  if (!fits(w_bytes)) return fail(UNIT_E_ARG, "%s: a group's weight exceeds 2^31-1 bytes", what);
  if (rows > 1 << 30 || groups > 1 << 20 || n > 1 << 22 || k > 1 << 22) return fail(UNIT_E_ARG, "%s: sizes beyond 2^30 rows, 2^20 groups or 2^22 columns", what);
  return UNIT_OK;
}

inline int check_f16(const char *what, int n, int k) {
  if (n % 8 || k % 8) return fail(UNIT_E_ARG, "%s: N and K must be multiples of 8 (16-byte rows), got %d and %d", what, n, k);
  return UNIT_OK;
}

inline int check_ptrs(const char *what, bool any, std::initializer_list<const void *> ptrs) {
  for (const void *p : ptrs)
    if (!p && any) return fail(UNIT_E_ARG, "%s: null pointer", what);
  return check_aligned(what, ptrs);
}

// The rows of an MXFP4 product: codes and scales as they are, or floats, which are quantised into the workspace first where the kernel
// does not do so by itself (takes_floats).  *run: there are rows, and p->x is what the kernel takes.
template <class F>
int mxfp4_rows(const char *what, GroupedParams *p, int out_dtype, void *ws, size_t ws_bytes, hipStream_t s, F takes_floats, bool *run) {
  const bool floats = p->x_dtype != UNIT_MXFP4;
  *run = false;
  if (floats && p->x_dtype != UNIT_F32 && p->x_dtype != UNIT_F16 && p->x_dtype != UNIT_BF16)
    return fail(UNIT_E_ARG, "%s: x_dtype must be UNIT_F32, UNIT_F16, UNIT_BF16 or UNIT_MXFP4, got %d", what, p->x_dtype);
  if (out_dtype != UNIT_F32 && out_dtype != UNIT_F16 && out_dtype != UNIT_BF16)
    return fail(UNIT_E_ARG, "%s: out_dtype must be UNIT_F32, UNIT_F16 or UNIT_BF16, got %d", what, out_dtype);
  const size_t codes = mx_code_bytes(p->rows, p->k), need = codes + mx_scale_bytes(p->rows, p->k);
  if (int rc = check_ptrs(what, p->rows, {p->y, p->ys, p->out})) return rc;
  if (floats && p->rows && ws_bytes < need) return fail(UNIT_E_ARG, "%s: workspace of %zu bytes, %zu needed", what, ws_bytes, need);
  if (floats) {
    if (int rc = check_ptrs(what, p->rows, {ws})) return rc;
    if (!p->x && p->rows) return fail(UNIT_E_ARG, "%s: null pointer", what);
  } else if (int rc = check_ptrs(what, p->rows, {p->x, p->xs})) {
    return rc;
  }
  if (int rc = check_device()) return rc;
  *run = p->rows;
  if (!p->rows || !floats || takes_floats(*p)) return UNIT_OK;
  char *buf = static_cast<char *>(ws);
  if (int rc = unit_quantize_mxfp4(p->x, p->x_dtype, p->rows, p->k, buf, buf + codes, s)) return rc;
  p->x = buf;
  p->xs = reinterpret_cast<const u32 *>(buf + codes);
  p->x_dtype = UNIT_MXFP4;
  return UNIT_OK;
}

}  // namespace unit
