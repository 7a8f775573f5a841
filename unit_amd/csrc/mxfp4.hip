// MXFP4: floats -> codes and scales, back, and a checkpoint's codes and scales into the layout of mxfp4.hpp.
#include "host.hpp"
#include "mxfp4.hpp"

namespace unit {
namespace {

template <class T>
__device__ __forceinline__ float as_float(T v) {
  return (float)v;
}

// One lane takes eight elements, four lanes a block.  Scaling by a power of two and rounding to the nearest element (ties to
// the even mantissa, magnitudes above 6 to 6) are v_cvt_scalef32_pk_fp4_f32.
template <class T>
__global__ __launch_bounds__(256) void quantize_kernel(const T *x, long rows, int K, u32 *codes, unsigned char *scales) {
  const int per_row = mx_stages(K) * 32;  // lanes per row
  const long id = (long)blockIdx.x * 256 + threadIdx.x;
  const long row = id / per_row;
  const int lane = (int)(id % per_row), k0 = lane * 8;
  const bool live = row < rows;
  float v[8];
  u32 top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[i] = live && k0 + i < K ? as_float(x[row * K + k0 + i]) : 0.0f;
    const u32 a = __builtin_bit_cast(u32, v[i]) & 0x7fffffffu;
    top = a > top ? a : top;
  }
  u32 other = __shfl_xor(top, 1);
  top = other > top ? other : top;
  other = __shfl_xor(top, 2);
  top = other > top ? other : top;
  if (!live) return;
  const u32 s = mx_scale(top);
  const float p = mx_power(s == 255 ? 127 : s);
  u32 c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], p, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], p, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], p, 2);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], p, 3);
  codes[row * per_row + lane] = c;
  const int b = lane / 4;
  if (lane % 4 == 0) scales[((long)(b / 8 * 2 + b % 2) * rows + row) * 4 + b % 8 / 2] = (unsigned char)s;
}

template <class T>
__global__ __launch_bounds__(256) void dequantize_kernel(const u32 *codes, const unsigned char *scales, long rows, int K, T *out) {
  const int per_row = mx_stages(K) * 32;
  const long id = (long)blockIdx.x * 256 + threadIdx.x;
  const long row = id / per_row;
  const int lane = (int)(id % per_row), k0 = lane * 8;
  if (row >= rows || k0 >= K) return;
  const int b = lane / 4;
  const u32 s = scales[((long)(b / 8 * 2 + b % 2) * rows + row) * 4 + b % 8 / 2];
  const u32 c = codes[row * per_row + lane];
  // 255 is NaN; 2^127 and the other powers are multiplied in single precision, once
  const float p = s == 255 ? __builtin_nanf("") : mx_power(s);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const u32 h = c >> (4 * i) & 15, m = h & 7;
    // 0, 0.5, then 2^(m / 2 - 1) * (1 + m % 2 / 2)
    const float a = m < 2 ? 0.5f * (float)m : __builtin_bit_cast(float, (126u + (m >> 1)) << 23 | (m & 1) << 22);
    if (k0 + i < K) out[row * K + k0 + i] = (T)((h & 8 ? -a : a) * p);
  }
}

// codes (rows, 16 * blocks), scales (rows, blocks), blocks = K / 32 rounded up; whatever the last block holds behind K is dropped
__global__ __launch_bounds__(256) void prepare_kernel(const unsigned char *codes_in, const unsigned char *scales_in, long rows, int K,
                                                      u32 *codes, unsigned char *scales) {
  const int per_row = mx_stages(K) * 32, blocks = (K + 31) / 32;
  const long id = (long)blockIdx.x * 256 + threadIdx.x;
  const long row = id / per_row;
  const int lane = (int)(id % per_row), k0 = lane * 8, b = lane / 4;
  if (row >= rows) return;
  u32 c = 0;
  if (k0 < K) {
    const unsigned char *src = codes_in + row * (16l * blocks) + lane * 4;
    c = src[0] | (u32)src[1] << 8 | (u32)src[2] << 16 | (u32)src[3] << 24;
    if (K - k0 < 8) c &= (1u << 4 * (K - k0)) - 1;
  }
  codes[row * per_row + lane] = c;
  if (lane % 4 == 0) scales[((long)(b / 8 * 2 + b % 2) * rows + row) * 4 + b % 8 / 2] = b < blocks ? scales_in[row * blocks + b] : 0;
}

int check_mx(const char *what, int64_t rows, int32_t K, std::initializer_list<const void *> ptrs) {
  if (rows < 0 || K <= 0) return fail(UNIT_E_ARG, "%s: rows must not be negative and K must be positive", what);
  if (rows > (int64_t)1 << 40 || rows * mx_stages(K) >= (int64_t)1 << 27) return fail(UNIT_E_ARG, "%s: 2^35 elements or more", what);
  for (const void *p : ptrs)
    if (!p && rows) return fail(UNIT_E_ARG, "%s: null pointer", what);
  return UNIT_OK;
}

unsigned mx_grid(int64_t rows, int32_t K) { return (unsigned)((rows * mx_stages(K) * 32 + 255) / 256); }

int launched(const char *what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? UNIT_OK : fail(UNIT_E_LAUNCH, "%s: launch: %s", what, hipGetErrorString(e));
}

}  // namespace
}  // namespace unit

using namespace unit;

extern "C" int unit_mxfp4_bytes(int64_t rows, int32_t K, size_t *codes, size_t *scales) {
  if (int rc = check_mx("unit_mxfp4_bytes", rows, K, {})) return rc;
  if (!codes || !scales) return fail(UNIT_E_ARG, "unit_mxfp4_bytes: null pointer");
  *codes = mx_code_bytes(rows, K);
  *scales = mx_scale_bytes(rows, K);
  return UNIT_OK;
}

extern "C" int unit_quantize_mxfp4(const void *x, int32_t dtype, int64_t rows, int32_t K, void *codes, void *scales, unit_stream_t stream) {
  const char *what = "unit_quantize_mxfp4";
  if (int rc = check_mx(what, rows, K, {x, codes, scales})) return rc;
  if (dtype != UNIT_F32 && dtype != UNIT_F16 && dtype != UNIT_BF16) return fail(UNIT_E_ARG, "%s: dtype must be UNIT_F32, UNIT_F16 or UNIT_BF16, got %d", what, dtype);
  if (int rc = check_aligned(what, {codes, scales})) return rc;
  if ((uintptr_t)x % (dtype == UNIT_F32 ? 4 : 2)) return fail(UNIT_E_ARG, "%s: x is not aligned to its elements", what);
  if (int rc = check_device()) return rc;
  if (!rows) return UNIT_OK;
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto run = [&](auto *p) {
    hipLaunchKernelGGL(quantize_kernel, dim3(mx_grid(rows, K)), dim3(256), 0, s, p, (long)rows, K, static_cast<u32 *>(codes), static_cast<unsigned char *>(scales));
  };
  if (dtype == UNIT_F32) run(static_cast<const float *>(x));
  if (dtype == UNIT_F16) run(static_cast<const _Float16 *>(x));
  if (dtype == UNIT_BF16) run(static_cast<const __bf16 *>(x));
  set_variant("mxquantize");
  return launched(what);
}

extern "C" int unit_dequantize_mxfp4(const void *codes, const void *scales, int64_t rows, int32_t K, void *out, int32_t dtype, unit_stream_t stream) {
  const char *what = "unit_dequantize_mxfp4";
  if (int rc = check_mx(what, rows, K, {codes, scales, out})) return rc;
  if (dtype != UNIT_F32 && dtype != UNIT_F16 && dtype != UNIT_BF16) return fail(UNIT_E_ARG, "%s: dtype must be UNIT_F32, UNIT_F16 or UNIT_BF16, got %d", what, dtype);
  if (int rc = check_aligned(what, {codes, scales, out})) return rc;
  if (int rc = check_device()) return rc;
  if (!rows) return UNIT_OK;
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto run = [&](auto *p) {
    hipLaunchKernelGGL(dequantize_kernel, dim3(mx_grid(rows, K)), dim3(256), 0, s, static_cast<const u32 *>(codes), static_cast<const unsigned char *>(scales), (long)rows, K, p);
  };
  if (dtype == UNIT_F32) run(static_cast<float *>(out));
  if (dtype == UNIT_F16) run(static_cast<_Float16 *>(out));
  if (dtype == UNIT_BF16) run(static_cast<__bf16 *>(out));
  set_variant("mxdequantize");
  return launched(what);
}

extern "C" int unit_prepare_mxfp4(const void *codes_in, const void *scales_in, int64_t rows, int32_t K, void *codes, void *scales, unit_stream_t stream) {
  const char *what = "unit_prepare_mxfp4";
  if (int rc = check_mx(what, rows, K, {codes_in, scales_in, codes, scales})) return rc;
  if (int rc = check_aligned(what, {codes, scales})) return rc;
  if (int rc = check_device()) return rc;
  if (!rows) return UNIT_OK;
  hipLaunchKernelGGL(prepare_kernel, dim3(mx_grid(rows, K)), dim3(256), 0, static_cast<hipStream_t>(stream), static_cast<const unsigned char *>(codes_in),
                     static_cast<const unsigned char *>(scales_in), (long)rows, K, static_cast<u32 *>(codes), static_cast<unsigned char *>(scales));
  set_variant("mxprepare");
  return launched(what);
}
