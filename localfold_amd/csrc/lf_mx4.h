// Device code of the 4-bit format: scales, codes, fragments.
#pragma once
#include "lf_step.h"

namespace lf {

typedef int i32x8 __attribute__((ext_vector_type(8)));

// The stored byte of the smallest power of two that puts a magnitude, as its bits, within 6 = 1.5 * 2^2: f * 2^p
// with f in [1, 2) needs 2^(p - 2), or 2^(p - 1) when f > 1.5.  255 for an infinity or a NaN.
__device__ __forceinline__ int mx_scale_byte(uint32_t bits) {
  const int b = (int)(bits >> 23) - 2 + ((bits & 0x7fffffu) > 0x400000u ? 1 : 0);
  return bits >= 0x7f800000u ? 255 : b < 1 ? 1 : b;
}
// Largest magnitude of eight values as bits (a NaN's are above an infinity's).
__device__ __forceinline__ uint32_t amax_bits8(const float (&v)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) m = max(m, __float_as_uint(v[k]) & 0x7fffffffu);
  return m;
}
// Eight values over a power of two as codes: the instruction divides exactly and rounds to nearest even.
__device__ __forceinline__ uint32_t mx_encode8(const float* v, float scale) {
  uint32_t w = 0;
#if __HIP_DEVICE_COMPILE__
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], scale, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], scale, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], scale, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], scale, 3);
#endif
  return w;
}
// The scale as a number; 2^127 or anything else finite for 255, whose codes do not matter.
__device__ __forceinline__ float mx_scale_value(int b) { return __uint_as_float((uint32_t)min(b, 254) << 23); }

// Largest over the four lanes of an aligned quad.
__device__ __forceinline__ uint32_t quad_max(uint32_t m) {
  m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0xB1, 0xF, 0xF, true));
  return max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x4E, 0xF, 0xF, true));
}

// acc += 16 rows of a times 16 rows of b over 128 columns: a lane holds 32 codes of row lane % 16, columns 32
// (lane / 16) on, and that group's scale byte in byte SA or SB of its word.  Measured: products and their sum
// within a group are exact, what the instruction adds up beyond it is off by at most 2^-24 of the magnitudes, and
// byte 255 makes NaN.
template <int SA, int SB>
__device__ __forceinline__ f4 mx_mma(u32x4 a, u32x4 b, f4 acc, uint32_t sa, uint32_t sb) {
#if __HIP_DEVICE_COMPILE__
  const i32x8 x = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
  const i32x8 y = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, acc, 4, 4, SA, (int)sa, SB, (int)sb);
#else
  (void)a, (void)b, (void)sa, (void)sb;
  return acc;
#endif
}

}  // namespace lf
