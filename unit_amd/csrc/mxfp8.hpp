// MXFP8 storage of activation checkpoints: rows of 8-bit floats (e4m3: 1 sign, 4 exponent, 3 mantissa bits, up to 448), 32 consecutive
// elements of a row sharing the power of two 2^(s - 127) of one byte s (255: the whole block is NaN).
//
// Layout in memory: codes rows of 32 * blocks bytes, blocks = K / 32 rounded up, zeros behind K; scales (rows, blocks) bytes.
// Rows of codes are whole pieces of 16 bytes, which is all that a kernel that reads them row by row needs.
#pragma once
#include "mxfp4.hpp"

namespace unit {

inline __host__ __device__ int mx8_blocks(int K) { return (K + kMxBlock - 1) / kMxBlock; }
inline size_t mx8_code_bytes(long rows, int K) { return (size_t)rows * mx8_blocks(K) * 32; }
inline size_t mx8_scale_bytes(long rows, int K) { return (size_t)rows * mx8_blocks(K); }

// The block's scale, biased by 127: the smallest power of two (2^-127 at least) for which the block's largest magnitude is at most
// 448 = 1.75 * 2^8.  Nothing saturates: the formats' own rule, the exponent less 8 throughout, would cut magnitudes of 449 to 511
// down to 448, up to an eighth off, where a rounding is off by a sixteenth at most (of an element of 2^-6 scales or more; below, in the
// subnormal range, by 2^-10 scales, all of a smaller element).  amax_bits: that magnitude as a float's bits.
__device__ __forceinline__ u32 mx8_scale(u32 amax_bits) {
  const u32 e = amax_bits >> 23, above = (amax_bits & 0x7fffffu) > 0x600000u;
  return e == 255 ? 255u : e + above < 8 ? 0u : e + above - 8;
}

// v / 2^(s - 127), rounded to the nearest 8-bit float (ties to the even mantissa): what v_cvt_scalef32_pk_fp8 does.  p: mx_power(s)
__device__ __forceinline__ u32 four_codes8(v4f v, float p) {
  typedef short v2h __attribute__((ext_vector_type(2)));
  v2h c = {0, 0};
  c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(c, v[0], v[1], p, false);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(c, v[2], v[3], p, true);
  return __builtin_bit_cast(u32, c);
}

// what four codes stand for; p: the scale's power of two, NaN for 255
__device__ __forceinline__ v4f four_values8(u32 c, float p) {
  typedef float v2f __attribute__((ext_vector_type(2)));
  const v2f lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
  return v4f{lo[0] * p, lo[1] * p, hi[0] * p, hi[1] * p};
}
__device__ __forceinline__ float mx8_power(u32 s) { return s == 255 ? __builtin_nanf("") : mx_power(s); }

// Rows to be restored, in pieces of eight elements (4 * blocks a row).
template <class T>
struct Mx8Rows {
  const v2u *codes;
  const unsigned char *scales;
  int pieces, K;
  T *out;  // (rows, K)
  FastDiv by_row;
};
// the pieces of workgroup `group` of 256 lanes, ROUNDS a lane
template <class T, int ROUNDS>
__device__ __forceinline__ void restore_pieces(const Mx8Rows<T> &r, int group) {
  typedef T v8 __attribute__((ext_vector_type(8), aligned(sizeof(T))));
  v2u c[ROUNDS];
  u32 s[ROUNDS];
  const int first = group * (256 * ROUNDS) + (int)threadIdx.x;
#pragma unroll
  for (int i = 0; i < ROUNDS; ++i) {
    const int at = min(first + i * 256, r.pieces - 1);
    c[i] = r.codes[at];
    s[i] = r.scales[at >> 2];
  }
#pragma unroll
  for (int i = 0; i < ROUNDS; ++i) {
    const int at = first + i * 256;
    int row, q;
    r.by_row.divmod(min(at, r.pieces - 1), row, q);
    const int k0 = q * 8;
    if (at >= r.pieces || k0 >= r.K) continue;
    const float p = mx8_power(s[i]);
    const v4f lo = four_values8(c[i][0], p), hi = four_values8(c[i][1], p);
    v8 v;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = (T)(j < 4 ? lo[j] : hi[j - 4]);  // one rounding, where T does not hold the value
    T *dst = r.out + (size_t)row * r.K + k0;
    if (k0 + 8 <= r.K) {
      *reinterpret_cast<v8 *>(dst) = v;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (k0 + j < r.K) dst[j] = v[j];
    }
  }
}

}  // namespace unit
