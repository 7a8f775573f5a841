// MXFP4 storage: rows of 4-bit floats (1 sign, 2 exponent, 1 mantissa bits: 0, 0.5, 1, 1.5, 2, 3, 4, 6), 32 consecutive elements
// of a row sharing the power of two 2^(s - 127) of one byte s (255: the whole block is NaN), as the OCP microscaling formats
// define them.
//
// Layout in memory, the one the matrix products read:
//   codes   rows of kb * 128 bytes, kb = K / 256 rounded up: the even element of a pair in the low half of its byte, zeros behind
//           K.  A row is a whole number of cache lines and of the products' 128-byte stages.
//   scales  [kb][2][rows][4] bytes: block b of a row lies at [b / 8][b % 2][row][(b % 8) / 2].  One v_mfma_scale_f32_32x32x64
//           takes 64 elements of 32 rows, lane l the block l / 32 of row l % 32; the four instructions of a 128-byte stage
//           therefore take the four bytes of one dword per lane, and the 32 lanes of a half read 128 consecutive bytes.
#pragma once
#include "mma_core.hpp"

namespace unit {

constexpr int kMxBlock = 32;   // elements per scale
constexpr int kMxStage = 256;  // elements per 128 bytes of codes, the padding of a row

inline __host__ __device__ int mx_stages(int K) { return (K + kMxStage - 1) / kMxStage; }
inline size_t mx_code_bytes(long rows, int K) { return (size_t)rows * mx_stages(K) * 128; }
// 1 KiB behind the last plane: the products fetch the scales of whole tiles of up to 256 rows
inline size_t mx_scale_bytes(long rows, int K) { return (size_t)rows * mx_stages(K) * 8 + 1024; }

// The block's scale: the exponent of its largest magnitude less 2 (the largest element, 6, is 1.5 * 2^2), biased by 127.
// amax_bits: the bits of that magnitude as a float.  Subnormal magnitudes lie below the smallest scale times the smallest
// element but for their upper bits and take scale 0 like every exponent below it.
__device__ __forceinline__ u32 mx_scale(u32 amax_bits) {
  const u32 e = amax_bits >> 23;
  return e == 255 ? 255u : e < 2 ? 0u : e - 2;
}
// 2^(s - 127); s = 0 is a subnormal float
__device__ __forceinline__ float mx_power(u32 s) { return __builtin_bit_cast(float, s ? s << 23 : 1u << 22); }

// eight elements of a row as their bits
template <class T>
struct Eight {
  using bits = std::conditional_t<sizeof(T) == 4, u32, unsigned short>;
  typedef bits b8 __attribute__((ext_vector_type(8)));
};

// Scaling by a power of two and rounding to the nearest element (ties to the even mantissa, magnitudes above 6 to 6) are what
// v_cvt_scalef32_pk_fp4 does.
template <class T>
__device__ __forceinline__ u32 eight_codes(typename Eight<T>::b8 v, float p) {
  u32 c = 0;
  auto two = [&](auto n) __attribute__((always_inline)) {
    constexpr int N = decltype(n)::value;
    if constexpr (std::is_same_v<T, float>) {
      typedef float v8f __attribute__((ext_vector_type(8)));
      const v8f f = __builtin_bit_cast(v8f, v);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[2 * N], f[2 * N + 1], p, N);
    } else {
      typedef T v2 __attribute__((ext_vector_type(2)));
      const u32 pair = __builtin_bit_cast(v4u, v)[N];
      if constexpr (std::is_same_v<T, _Float16>)
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(v2, pair), p, N);
      else
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(v2, pair), p, N);
    }
  };
  two(std::integral_constant<int, 0>{});
  two(std::integral_constant<int, 1>{});
  two(std::integral_constant<int, 2>{});
  two(std::integral_constant<int, 3>{});
  return c;
}

// the bits of the largest magnitude of eight elements, as a float; infinities and NaN are the largest
template <class T>
__device__ __forceinline__ u32 eight_top(typename Eight<T>::b8 v) {
  u32 top = 0;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, v[i] & 0x7fffffffu);
    return top;
  } else {
    // sign-less 16-bit patterns are ordered like the values: two at a time
    const v4u w = __builtin_bit_cast(v4u, v);
    typedef unsigned short v2s __attribute__((ext_vector_type(2)));
    v2s m = __builtin_bit_cast(v2s, w[0] & 0x7fff7fffu);
#pragma unroll
    for (int i = 1; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(v2s, w[i] & 0x7fff7fffu));
    top = max((u32)m[0], (u32)m[1]);
    if constexpr (std::is_same_v<T, __bf16>) return top << 16;
    return __builtin_bit_cast(u32, (float)__builtin_bit_cast(_Float16, (unsigned short)top)) & 0x7fffffffu;  // NaN stays NaN
  }
}

}  // namespace unit
