// MXFP4: floats -> codes and scales, back, and a checkpoint's codes and scales into the layout of mxfp4.hpp.
#include "host.hpp"
#include "mxfp4.hpp"

namespace unit {
namespace {

// A workgroup takes 8 * ROUNDS rows of one 256-element stage, half a wave a row: a lane eight elements, four lanes a block.
// All of a lane's loads are issued before the first is used; the scales of a stage, one dword per row and half, are gathered in
// LDS so that they leave in runs of consecutive rows.
template <class T, int ROUNDS>
struct StageRows {
  static constexpr int kRows = 8 * ROUNDS;
  typedef typename Eight<T>::bits bits;
  typedef typename Eight<T>::b8 b8 __attribute__((aligned(sizeof(T))));  // rows begin on any element
  typedef T v8 __attribute__((ext_vector_type(8), aligned(sizeof(T))));
};

template <class T, int ROUNDS>
__global__ __launch_bounds__(256) void quantize_kernel(const T *x, int rows, int K, u32 *codes, u32 *scales, FastDiv by_stages) {
  using R = StageRows<T, ROUNDS>;
  __shared__ unsigned char gather[2 * R::kRows * 4];
  const int t = threadIdx.x, l32 = t & 31, stages = by_stages.d;
  int s, row0;
  by_stages.divmod((int)blockIdx.x, row0, s);
  row0 *= R::kRows;
  const int k0 = s * kMxStage + l32 * 8;
  typename R::b8 v[ROUNDS];
#pragma unroll
  for (int i = 0; i < ROUNDS; ++i) {
    const int row = min(row0 + i * 8 + (t >> 5), rows - 1);
    const typename R::bits *src = reinterpret_cast<const typename R::bits *>(x) + (size_t)row * K + k0;
    if (k0 + 8 <= K) {
      v[i] = *reinterpret_cast<const typename R::b8 *>(src);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = k0 + j < K ? src[j] : 0;
    }
  }
#pragma unroll
  for (int i = 0; i < ROUNDS; ++i) {
    const int r = i * 8 + (t >> 5), row = row0 + r;
    u32 top = eight_top<T>(v[i]);
    top = max(top, (u32)__builtin_amdgcn_mov_dpp((int)top, 0xb1, 0xf, 0xf, true));  // lanes 1, 0, 3, 2
    top = max(top, (u32)__builtin_amdgcn_mov_dpp((int)top, 0x4e, 0xf, 0xf, true));  // lanes 2, 3, 0, 1
    const u32 e = mx_scale(top);
    const u32 c = eight_codes<T>(v[i], mx_power(e == 255 ? 127 : e));
    if (row < rows) codes[(size_t)row * (stages * 32) + s * 32 + l32] = c;
    const int b = l32 >> 2;
    if ((l32 & 3) == 0) gather[((b & 1) * R::kRows + r) * 4 + (b >> 1)] = (unsigned char)e;
  }
  __syncthreads();
  const int h = t / R::kRows, r = t % R::kRows;
  if (h < 2 && row0 + r < rows) scales[(size_t)(2 * s + h) * rows + row0 + r] = reinterpret_cast<const u32 *>(gather)[t];
}

template <class T, int ROUNDS>
__global__ __launch_bounds__(256) void dequantize_kernel(const u32 *codes, const u32 *scales, int rows, int K, T *out, FastDiv by_stages) {
  using R = StageRows<T, ROUNDS>;
  const int t = threadIdx.x, l32 = t & 31, stages = by_stages.d;
  int s, row0;
  by_stages.divmod((int)blockIdx.x, row0, s);
  row0 = row0 * R::kRows + (t >> 5);
  const int k0 = s * kMxStage + l32 * 8, b = l32 >> 2;
  u32 c[ROUNDS], e[ROUNDS];
#pragma unroll
  for (int i = 0; i < ROUNDS; ++i) {
    const int row = min(row0 + i * 8, rows - 1);
    c[i] = codes[(size_t)row * (stages * 32) + s * 32 + l32];
    e[i] = scales[(size_t)(2 * s + (b & 1)) * rows + row] >> (8 * (b >> 1)) & 255;
  }
#pragma unroll
  for (int i = 0; i < ROUNDS; ++i) {
    const int row = row0 + i * 8;
    if (row >= rows || k0 >= K) continue;
    const float p = e[i] == 255 ? __builtin_nanf("") : mx_power(e[i]);
    typename R::v8 v;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const u32 h = c[i] >> (4 * j) & 15, m = h & 7;
      // 0, 0.5, then 2^(m / 2 - 1) * (1 + m % 2 / 2); one rounding, to T
      const u32 a = m < 2 ? m * 0x3f000000u : (126u + (m >> 1)) << 23 | (m & 1) << 22;
      v[j] = (T)(__builtin_bit_cast(float, a | (h & 8) << 28) * p);
    }
    T *dst = out + (size_t)row * K + k0;
    if (k0 + 8 <= K) {
      *reinterpret_cast<typename R::v8 *>(dst) = v;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (k0 + j < K) dst[j] = v[j];
    }
  }
}

// codes (rows, 16 * blocks), scales (rows, blocks), blocks = K / 32 rounded up; whatever the last block holds behind K is dropped
template <int ROUNDS>
__global__ __launch_bounds__(256) void prepare_kernel(const unsigned char *codes_in, const unsigned char *scales_in, int rows, int K, u32 *codes, u32 *scales,
                                                      FastDiv by_stages) {
  constexpr int ROWS = 8 * ROUNDS;
  typedef u32 u32_any __attribute__((aligned(1)));
  const int t = threadIdx.x, l32 = t & 31, stages = by_stages.d, blocks = (K + 31) / 32;
  int s, row0;
  by_stages.divmod((int)blockIdx.x, row0, s);
  row0 *= ROWS;
  const int k0 = s * kMxStage + l32 * 8;
  u32 c[ROUNDS];
#pragma unroll
  for (int i = 0; i < ROUNDS; ++i) {
    const int row = min(row0 + i * 8 + (t >> 5), rows - 1);
    c[i] = 0;
    if (k0 < K) c[i] = *reinterpret_cast<const u32_any *>(codes_in + (size_t)row * (16 * blocks) + s * 128 + l32 * 4);
    if (k0 < K && K - k0 < 8) c[i] &= (1u << 4 * (K - k0)) - 1;
  }
#pragma unroll
  for (int i = 0; i < ROUNDS; ++i) {
    const int row = row0 + i * 8 + (t >> 5);
    if (row < rows) codes[(size_t)row * (stages * 32) + s * 32 + l32] = c[i];
  }
  const int h = t / ROWS, row = row0 + t % ROWS;
  if (h < 2 && row < rows) {
    u32 e = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int b = s * 8 + 2 * j + h;
      if (b < blocks) e |= (u32)scales_in[(size_t)row * blocks + b] << (8 * j);
    }
    scales[(size_t)(2 * s + h) * rows + row] = e;
  }
}

int check_mx(const char *what, int64_t rows, int32_t K, std::initializer_list<const void *> ptrs) {
  if (rows < 0 || K <= 0) return fail(UNIT_E_ARG, "%s: rows must not be negative and K must be positive", what);
  if (rows > (int64_t)1 << 40 || rows * mx_stages(K) >= (int64_t)1 << 27) return fail(UNIT_E_ARG, "%s: 2^35 elements or more", what);
  for (const void *p : ptrs)
    if (!p && rows) return fail(UNIT_E_ARG, "%s: null pointer", what);
  return UNIT_OK;
}

// run(rounds, workgroups, divider): 64 rows a workgroup while that makes two workgroups per CU, else 8
template <class F>
void by_stage(int64_t rows, int32_t K, F run) {
  const int stages = mx_stages(K);
  const int64_t tall = (rows + 63) / 64 * stages;
  if (tall >= 512)
    run(std::integral_constant<int, 8>{}, dim3((unsigned)tall), FastDiv::make(stages));
  else
    run(std::integral_constant<int, 1>{}, dim3((unsigned)((rows + 7) / 8 * stages)), FastDiv::make(stages));
}

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
    by_stage(rows, K, [&](auto rounds, dim3 grid, FastDiv by_stages) {
      using T = std::remove_const_t<std::remove_pointer_t<decltype(p)>>;
      hipLaunchKernelGGL((quantize_kernel<T, decltype(rounds)::value>), grid, dim3(256), 0, s, p, (int)rows, K, static_cast<u32 *>(codes), static_cast<u32 *>(scales),
                         by_stages);
    });
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
    by_stage(rows, K, [&](auto rounds, dim3 grid, FastDiv by_stages) {
      using T = std::remove_pointer_t<decltype(p)>;
      hipLaunchKernelGGL((dequantize_kernel<T, decltype(rounds)::value>), grid, dim3(256), 0, s, static_cast<const u32 *>(codes), static_cast<const u32 *>(scales),
                         (int)rows, K, p, by_stages);
    });
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
  by_stage(rows, K, [&](auto rounds, dim3 grid, FastDiv by_stages) {
    hipLaunchKernelGGL((prepare_kernel<decltype(rounds)::value>), grid, dim3(256), 0, static_cast<hipStream_t>(stream), static_cast<const unsigned char *>(codes_in),
                       static_cast<const unsigned char *>(scales_in), (int)rows, K, static_cast<u32 *>(codes), static_cast<u32 *>(scales), by_stages);
  });
  set_variant("mxprepare");
  return launched(what);
}
