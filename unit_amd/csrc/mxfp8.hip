// MXFP8: floats -> codes and scales, and back.  Both are bound by memory: a lane moves eight elements at a time, four lanes a block.
#include "host.hpp"
#include "mxfp8.hpp"

namespace unit {
namespace {

// A lane's eight elements of piece i (rows of 4 * blocks pieces): loads of all ROUNDS pieces are issued before the first is used.
template <class T, int ROUNDS>
__global__ __launch_bounds__(256) void quantize8_kernel(const T *x, int pieces, int K, v2u *codes, unsigned char *scales, FastDiv by_row) {
  typedef typename Eight<T>::bits bits;
  typedef typename Eight<T>::b8 b8;
  typedef b8 b8_any __attribute__((aligned(sizeof(T))));  // rows begin on any element
  b8 v[ROUNDS];
  const int first = (int)blockIdx.x * (256 * ROUNDS) + (int)threadIdx.x;
#pragma unroll
  for (int i = 0; i < ROUNDS; ++i) {
    int row, c;
    by_row.divmod(min(first + i * 256, pieces - 1), row, c);
    const int k0 = c * 8;
    const bits *src = reinterpret_cast<const bits *>(x) + (size_t)row * K + k0;
    if (k0 + 8 <= K) {
      v[i] = *reinterpret_cast<const b8_any *>(src);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = k0 + j < K ? src[j] : 0;
    }
  }
#pragma unroll
  for (int i = 0; i < ROUNDS; ++i) {
    const int at = first + i * 256;
    u32 top = eight_top<T>(v[i]);
    top = max(top, (u32)__builtin_amdgcn_mov_dpp((int)top, 0xb1, 0xf, 0xf, true));  // lanes 1, 0, 3, 2
    top = max(top, (u32)__builtin_amdgcn_mov_dpp((int)top, 0x4e, 0xf, 0xf, true));  // lanes 2, 3, 0, 1
    const u32 s = mx8_scale(top);
    const float p = mx_power(s == 255 ? 127 : s);
    v2u c;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      typedef T t8 __attribute__((ext_vector_type(8)));
      const t8 t = __builtin_bit_cast(t8, v[i]);
      v4f f;
#pragma unroll
      for (int j = 0; j < 4; ++j) f[j] = (float)t[4 * h + j];
      c[h] = four_codes8(f, p);
    }
    if (at < pieces) {
      codes[at] = c;
      if ((at & 3) == 0) scales[at >> 2] = (unsigned char)s;
    }
  }
}

template <class T, int ROUNDS>
__global__ __launch_bounds__(256) void dequantize8_kernel(Mx8Rows<T> r) {
  restore_pieces<T, ROUNDS>(r, (int)blockIdx.x);
}

int check_mx8(const char *what, int64_t rows, int32_t K, std::initializer_list<const void *> ptrs) {
  if (rows < 0 || K <= 0) return fail(UNIT_E_ARG, "%s: rows must not be negative and K must be positive", what);
  if (K > 1 << 28 || rows > (int64_t)1 << 40 || rows * mx8_blocks(K) >= (int64_t)1 << 33) return fail(UNIT_E_ARG, "%s: 2^38 elements or more, or rows of more than 2^28", what);
  for (const void *p : ptrs)
    if (!p && rows) return fail(UNIT_E_ARG, "%s: null pointer", what);
  return UNIT_OK;
}

int check_mx8_type(const char *what, int32_t dtype) {
  return dtype == UNIT_F32 || dtype == UNIT_F16 || dtype == UNIT_BF16 ? UNIT_OK : fail(UNIT_E_ARG, "%s: dtype must be UNIT_F32, UNIT_F16 or UNIT_BF16, got %d", what, dtype);
}

// run(rounds, workgroups, first row, pieces) over slices of rows whose pieces are counted in 31 bits: four pieces a lane while that makes
// four workgroups a CU, else one
template <class F>
int by_pieces(const char *what, int64_t rows, int32_t K, F run) {
  const int64_t per_row = 4 * mx8_blocks(K), slice = ((int64_t)1 << 30) / per_row;
  for (int64_t row = 0; row < rows; row += slice) {
    const int64_t pieces = (rows - row < slice ? rows - row : slice) * per_row;
    if (pieces >= 1024 * 1024)
      run(std::integral_constant<int, 4>{}, dim3((unsigned)((pieces + 1023) / 1024)), row, (int)pieces);
    else
      run(std::integral_constant<int, 1>{}, dim3((unsigned)((pieces + 255) / 256)), row, (int)pieces);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fail(UNIT_E_LAUNCH, "%s: launch: %s", what, hipGetErrorString(e));
  }
  return UNIT_OK;
}

}  // namespace
}  // namespace unit

using namespace unit;

extern "C" int unit_mxfp8_bytes(int64_t rows, int32_t K, size_t *codes, size_t *scales) {
  if (int rc = check_mx8("unit_mxfp8_bytes", rows, K, {})) return rc;
  if (!codes || !scales) return fail(UNIT_E_ARG, "unit_mxfp8_bytes: null pointer");
  *codes = mx8_code_bytes(rows, K);
  *scales = mx8_scale_bytes(rows, K);
  return UNIT_OK;
}

extern "C" int unit_quantize_mxfp8(const void *x, int32_t dtype, int64_t rows, int32_t K, void *codes, void *scales, unit_stream_t stream) {
  const char *what = "unit_quantize_mxfp8";
  if (int rc = check_mx8(what, rows, K, {x, codes, scales})) return rc;
  if (int rc = check_mx8_type(what, dtype)) return rc;
  if (int rc = check_aligned(what, {codes})) return rc;
  if ((uintptr_t)x % (dtype == UNIT_F32 ? 4 : 2)) return fail(UNIT_E_ARG, "%s: x is not aligned to its elements", what);
  if (int rc = check_device()) return rc;
  if (!rows) return UNIT_OK;
  const FastDiv by_row = FastDiv::make(4 * mx8_blocks(K));
  auto run = [&](auto *p) {
    return by_pieces(what, rows, K, [&](auto rounds, dim3 grid, int64_t row, int pieces) {
      using T = std::remove_const_t<std::remove_pointer_t<decltype(p)>>;
      hipLaunchKernelGGL((quantize8_kernel<T, decltype(rounds)::value>), grid, dim3(256), 0, static_cast<hipStream_t>(stream), p + row * K, pieces, K,
                         reinterpret_cast<v2u *>(static_cast<char *>(codes) + mx8_code_bytes(row, K)), static_cast<unsigned char *>(scales) + mx8_scale_bytes(row, K), by_row);
    });
  };
  set_variant("mx8quantize");
  if (dtype == UNIT_F32) return run(static_cast<const float *>(x));
  return dtype == UNIT_F16 ? run(static_cast<const _Float16 *>(x)) : run(static_cast<const __bf16 *>(x));
}

extern "C" int unit_dequantize_mxfp8(const void *codes, const void *scales, int64_t rows, int32_t K, void *out, int32_t dtype, unit_stream_t stream) {
  const char *what = "unit_dequantize_mxfp8";
  if (int rc = check_mx8(what, rows, K, {codes, scales, out})) return rc;
  if (int rc = check_mx8_type(what, dtype)) return rc;
  if (int rc = check_aligned(what, {codes, out})) return rc;
  if (int rc = check_device()) return rc;
  if (!rows) return UNIT_OK;
  const FastDiv by_row = FastDiv::make(4 * mx8_blocks(K));
  auto run = [&](auto *p) {
    return by_pieces(what, rows, K, [&](auto rounds, dim3 grid, int64_t row, int pieces) {
      using T = std::remove_pointer_t<decltype(p)>;
      const Mx8Rows<T> r{reinterpret_cast<const v2u *>(static_cast<const char *>(codes) + mx8_code_bytes(row, K)),
                         static_cast<const unsigned char *>(scales) + mx8_scale_bytes(row, K), pieces, K, p + row * K, by_row};
      hipLaunchKernelGGL((dequantize8_kernel<T, decltype(rounds)::value>), grid, dim3(256), 0, static_cast<hipStream_t>(stream), r);
    });
  };
  set_variant("mx8dequantize");
  if (dtype == UNIT_F32) return run(static_cast<float *>(out));
  return dtype == UNIT_F16 ? run(static_cast<_Float16 *>(out)) : run(static_cast<__bf16 *>(out));
}
