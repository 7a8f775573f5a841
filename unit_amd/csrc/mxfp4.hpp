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

}  // namespace unit
