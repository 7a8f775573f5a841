// Products whose rows belong to groups (the experts of a mixture): rows 0 .. sizes[0] - 1 to group 0, the next sizes[1] to group
// 1, and so on; sizes live in device memory, so that no call waits for the host to know them.
//   forward       out[r][n] = sum_k x[r][k] w[g(r)][n][k]
//   data gradient dx[r][k]  = sum_n dy[r][n] w[g(r)][n][k]
//   weight gradient dw[g][n][k] = sum over the rows r of g of dy[r][n] x[r][k]
// Sizes are taken as min(max(size, 0), rows left), so whatever they hold, no access leaves the tensors; rows behind the last
// group's are written as zeros.
#pragma once
#include "host.hpp"
#include "mxfp4.hpp"

namespace unit {

typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef int v8i __attribute__((ext_vector_type(8)));

struct GroupedParams {
  const char *x, *y;       // first operand (rows), second operand (weights; x for the weight gradient)
  const u32 *xs, *ys;      // MXFP4: scales of the two
  char *out;
  const void *sizes;       // null: one group of all rows
  int size_bytes;          // 4 or 8
  int groups, rows;        // groups, rows of the row operands
  int n, k;                // weight (groups, n, k)
  int x_dtype;             // MXFP4 products: UNIT_MXFP4, or UNIT_F16 / UNIT_BF16 for x still in floats
  int past_caches = 0;     // weight gradients of 16 bits in whole lines: nt
};

// More than 64 KiB of dynamic LDS for a kernel: granted to it on the current device, so asked for once a device (and thread).  allowed: of the
// kernel, a bit per device that has granted it; devices past the 64th are asked every time.
inline int allow_lds(const char *what, const void *kern, unsigned long long *allowed) {
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return fail(UNIT_E_DEVICE, "%s: hipGetDevice: %s", what, hipGetErrorString(e));
  const unsigned long long bit = dev < 64 ? 1ull << dev : 0;
  if (*allowed & bit) return UNIT_OK;
  e = hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize, kMaxLds);
  if (e != hipSuccess) return fail(UNIT_E_LAUNCH, "%s: hipFuncSetAttribute: %s", what, hipGetErrorString(e));
  *allowed |= bit;
  return UNIT_OK;
}

__device__ __forceinline__ int group_size(const GroupedParams &p, int g) {
  if (!p.sizes) return p.rows;
  long s = p.size_bytes == 8 ? static_cast<const long *>(p.sizes)[g] : (long)static_cast<const int *>(p.sizes)[g];
  s = s < 0 ? 0 : s;
  return (int)(s < p.rows ? s : p.rows);
}

// the products by operand type (dir: FORWARD, GRAD_DATA, GRAD_WEIGHT); out_dtype UNIT_F32 or the operands' type, MXFP4: any
enum { FORWARD, GRAD_DATA, GRAD_WEIGHT };
int run_grouped_f16(const char *what, int dir, const GroupedParams &p, int out_dtype, hipStream_t s);
int run_grouped_bf16(const char *what, int dir, const GroupedParams &p, int out_dtype, hipStream_t s);
bool grouped_mx_takes_floats(const GroupedParams &p);
int run_grouped_mx(const char *what, const GroupedParams &p, int out_dtype, hipStream_t s);

}  // namespace unit
