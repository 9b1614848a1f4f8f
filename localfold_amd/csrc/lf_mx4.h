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

// 32 activations of a row, one group: loaded as they are stored, then quantised to codes and the scale byte.
typedef unsigned short us2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
template <int ACT>
struct MxRaw {
  static constexpr int WORDS = ACT == DT_F32 ? 32 : 16;
  uint32_t w[WORDS];
  // p[0..32), of which the first n exist
  __device__ __forceinline__ void load(const typename Act<ACT>::T* p, int n) {
    if (n >= 32) {
      __builtin_memcpy(w, p, sizeof(w));
      return;
    }
#pragma unroll
    for (int k = 0; k < WORDS; ++k) {
      if constexpr (ACT == DT_F32) {
        w[k] = k < n ? __float_as_uint(p[k]) : 0u;
      } else {
        uint16_t lo = 0, hi = 0;
        if (2 * k < n) __builtin_memcpy(&lo, p + 2 * k, 2);
        if (2 * k + 1 < n) __builtin_memcpy(&hi, p + 2 * k + 1, 2);
        w[k] = lo | (uint32_t)hi << 16;
      }
    }
  }
  // The codes, and the scale byte returned.
  __device__ __forceinline__ int quantise(u32x4& codes) const {
    uint32_t m;
    if constexpr (ACT == DT_F32) {
      m = 0;
#pragma unroll
      for (int k = 0; k < WORDS; ++k) m = max(m, w[k] & 0x7fffffffu);
    } else {
      us2 q = {0, 0};
#pragma unroll
      for (int k = 0; k < WORDS; ++k) q = __builtin_elementwise_max(q, __builtin_bit_cast(us2, w[k] & 0x7fff7fffu));
      const uint16_t h = q[0] > q[1] ? q[0] : q[1];
      m = ACT == DT_BF16 ? (uint32_t)h << 16 : __float_as_uint(h2f(h));
    }
    const int b = mx_scale_byte(m);
    const float f = mx_scale_value(b);
#if __HIP_DEVICE_COMPILE__
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      uint32_t c = 0;
      if constexpr (ACT == DT_F32) {
        const uint32_t* v = w + 8 * k;
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, __uint_as_float(v[0]), __uint_as_float(v[1]), f, 0);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, __uint_as_float(v[2]), __uint_as_float(v[3]), f, 1);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, __uint_as_float(v[4]), __uint_as_float(v[5]), f, 2);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, __uint_as_float(v[6]), __uint_as_float(v[7]), f, 3);
      } else if constexpr (ACT == DT_BF16) {
        const uint32_t* v = w + 4 * k;
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf2, v[0]), f, 0);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf2, v[1]), f, 1);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf2, v[2]), f, 2);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf2, v[3]), f, 3);
      } else {
        const uint32_t* v = w + 4 * k;
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(h2, v[0]), f, 0);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(h2, v[1]), f, 1);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(h2, v[2]), f, 2);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, __builtin_bit_cast(h2, v[3]), f, 3);
      }
      codes[k] = c;
    }
#else
    (void)f;
    codes = u32x4{0, 0, 0, 0};
#endif
    return b;
  }
};

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

// acc[t][q] += tile q of x times tile t of w; the scale bytes of an operand's tiles are those of one word.
template <int MT>
__device__ __forceinline__ void mx_mma_set(f4 (&acc)[4][MT], const u32x4 (&x)[MT], const u32x4 (&w)[4], uint32_t sx, uint32_t sw) {
  static_assert(MT == 2 || MT == 4, "rows of a lane");
  acc[0][0] = mx_mma<0, 0>(x[0], w[0], acc[0][0], sx, sw);
  acc[1][0] = mx_mma<0, 1>(x[0], w[1], acc[1][0], sx, sw);
  acc[2][0] = mx_mma<0, 2>(x[0], w[2], acc[2][0], sx, sw);
  acc[3][0] = mx_mma<0, 3>(x[0], w[3], acc[3][0], sx, sw);
  acc[0][1] = mx_mma<1, 0>(x[1], w[0], acc[0][1], sx, sw);
  acc[1][1] = mx_mma<1, 1>(x[1], w[1], acc[1][1], sx, sw);
  acc[2][1] = mx_mma<1, 2>(x[1], w[2], acc[2][1], sx, sw);
  acc[3][1] = mx_mma<1, 3>(x[1], w[3], acc[3][1], sx, sw);
  if constexpr (MT == 4) {
    acc[0][2] = mx_mma<2, 0>(x[2], w[0], acc[0][2], sx, sw);
    acc[1][2] = mx_mma<2, 1>(x[2], w[1], acc[1][2], sx, sw);
    acc[2][2] = mx_mma<2, 2>(x[2], w[2], acc[2][2], sx, sw);
    acc[3][2] = mx_mma<2, 3>(x[2], w[3], acc[3][2], sx, sw);
    acc[0][3] = mx_mma<3, 0>(x[3], w[0], acc[0][3], sx, sw);
    acc[1][3] = mx_mma<3, 1>(x[3], w[1], acc[1][3], sx, sw);
    acc[2][3] = mx_mma<3, 2>(x[3], w[2], acc[2][3], sx, sw);
    acc[3][3] = mx_mma<3, 3>(x[3], w[3], acc[3][3], sx, sw);
  }
}

}  // namespace lf
