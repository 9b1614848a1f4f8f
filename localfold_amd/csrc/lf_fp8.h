// Device code shared by the kernels that multiply 8-bit operands: fragments, the order of weight tiles in
// LDS, and one step of a wave's product.
//
// w is the matrix instruction's first operand, so a lane's accumulators hold 4 consecutive outputs of one
// row per tile of 16; which tile holds which outputs is chosen so that a lane's runs fill 16-byte stores
// (n_of).  w lies in LDS as tiles of 128 x 128 codes, copied there by direct loads in an order that
// spreads a fragment's rows over the banks (key_of).
//
// Operands are converted in registers for the bf16 instruction: codes times a power of two fit bfloat16, products
// are exact and sums are f32's.  The 8-bit instructions, with and without scales, drop what lies 2^-13 below
// the largest of 8 products that they add at a time (measured: 1.6e-5 of the result for normal inputs; where large
// ones cancel, up to 1e-3 of those), always downwards.
#pragma once
#include "lf_train.h"

namespace lf {

typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));

constexpr int OUT_KEPT = 3;               // beside DT_F32, DT_F16, DT_BF16
constexpr int WTILE = GROUP * GROUP;      // bytes of a weight tile

static __device__ const uint4 fp8_zero16 = {0, 0, 0, 0};

// Which output tile t (of 8), row i (of 16) of the first operand is: runs of 4 * PER consecutive outputs
// a lane group, PER tiles each: 16 bytes of f32, of 16-bit values or of codes.
template <int OUT> struct Run { static constexpr int PER = OUT == DT_F32 ? 1 : OUT == OUT_KEPT ? 4 : 2; };
template <int OUT>
__device__ __forceinline__ int n_of(int t, int i) {
  constexpr int P = Run<OUT>::PER;
  return t / P * (16 * P) + (i >> 2) * (4 * P) + t % P * 4 + (i & 3);
}
// 16-byte chunk c of LDS row n lies at c ^ key_of(n): the rows that 8 neighbouring lanes read differ in it.
template <int OUT>
__device__ __forceinline__ int key_of(int n) {
  return (n & 3) | ((n / (4 * Run<OUT>::PER)) & 1) << 2;
}

// Eight codes times a power of two as bf16, exact.
__device__ __forceinline__ b8 codes_bf16(uint32_t lo, uint32_t hi, float s) {
  const b2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)lo, s, false);
  const b2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)lo, s, true);
  const b2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)hi, s, false);
  const b2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)hi, s, true);
  return b8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// One step's rows of x for a lane: rows MT r + t (r = lane % 16), columns 16 g .. and 64 + 16 g .. of the
// group (both operands take their columns in this order), and those rows' scale bytes.
template <int MT>
struct XFrag {
  u32x4 v[MT][2];
  uint32_t scale;
};

// Copies weight tile (nb, kb) of [outputs][pitch] codes to LDS: instruction `part` of 16 fills 8 rows.  Rows
// past the end repeat the last one (their outputs are not stored); a half group's other half is zeros.
template <int OUT>
__device__ __forceinline__ void w_stage(uint8_t* dst, const uint8_t* w, int pitch, int outputs, int nb, int kb, int part,
                                        int lane) {
  const int row = part * 8 + (lane >> 3);
  const int c = (lane & 7) ^ key_of<OUT>(row);
  const uint8_t* src = w + (size_t)min(nb * GROUP + row, outputs - 1) * pitch + kb * GROUP + c * 16;
  if (kb * GROUP + c * 16 >= pitch) src = reinterpret_cast<const uint8_t*>(&fp8_zero16);
#if __HIP_DEVICE_COMPILE__   // a target builtin: the host pass, which only emits the launch stub, lacks it
  __builtin_amdgcn_global_load_lds(src, dst + part * 1024, 16, 0, 0);
#else
  (void)src;
#endif
}

// acc[q] += 16 outputs x 16 MT rows x 128 columns, w a lane's two pieces of its output's codes.
template <int MT>
__device__ __forceinline__ void mma_frag(f4 (&acc)[MT], const u32x4 (&w)[2], const XFrag<MT>& x, int wscale) {
#if __HIP_DEVICE_COMPILE__
  const float sw = scale_value(wscale);
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const b8 a0 = codes_bf16(w[half].x, w[half].y, sw), a1 = codes_bf16(w[half].z, w[half].w, sw);
#pragma unroll
    for (int q = 0; q < MT; ++q) {
      const float sx = scale_value((x.scale >> (8 * q)) & 255);
      const u32x4 v = x.v[q][half];
      acc[q] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a0, codes_bf16(v.x, v.y, sx), acc[q], 0, 0, 0);
      acc[q] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a1, codes_bf16(v.z, v.w, sx), acc[q], 0, 0, 0);
    }
  }
#else
  (void)acc;
  (void)w;
  (void)x;
  (void)wscale;
#endif
}

// acc += one step: 16 NT outputs x 16 MT rows x 128 columns (HALF: 64, the others are zeros); FIRST: acc =
// bias + the step, bias 16 NT floats in LDS.  w: the lane's place in an LDS tile, wx the same with the other
// half of the columns.  A tile's fragment is read while the one before it is multiplied; the barriers keep the
// compiler from reading all eight at once, which would spill.  next() may load over x: it is called once x is
// no longer read.
template <int OUT, bool FIRST, bool HALF, int NT, int MT, class NEXT>
__device__ __forceinline__ void mma(f4 (&acc)[NT][MT], const uint8_t* w, const uint8_t* wx, const XFrag<MT>& x, int wscale,
                                    const float* bias, int g, NEXT next) {
#if __HIP_DEVICE_COMPILE__
  f4 c;
  const float sw = scale_value(wscale);
#pragma unroll
  for (int half = 0; half < (HALF ? 1 : 2); ++half) {
    const uint8_t* wh = half ? wx : w;
    b8 b[MT][2];
    u32x4 a[2];
    a[0] = *reinterpret_cast<const u32x4*>(wh);
#pragma unroll
    for (int q = 0; q < MT; ++q) {
      const float sx = scale_value((x.scale >> (8 * q)) & 255);
      const u32x4 v = x.v[q][half];
      b[q][0] = codes_bf16(v.x, v.y, sx);
      b[q][1] = codes_bf16(v.z, v.w, sx);
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if (t < NT - 1) a[(t + 1) & 1] = *reinterpret_cast<const u32x4*>(wh + n_of<OUT>(t + 1, 0) * GROUP);
      if constexpr (FIRST)
        if (half == 0) c = *reinterpret_cast<const f4*>(bias + n_of<OUT>(t, 4 * g));
      const u32x4 v = a[t & 1];
      const b8 a0 = codes_bf16(v.x, v.y, sw), a1 = codes_bf16(v.z, v.w, sw);
#pragma unroll
      for (int q = 0; q < MT; ++q)
        acc[t][q] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a0, b[q][0], FIRST && half == 0 ? c : acc[t][q], 0, 0, 0);
#pragma unroll
      for (int q = 0; q < MT; ++q) acc[t][q] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a1, b[q][1], acc[t][q], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
#endif
  next();
}

// Zeros where the gate's code is zero or negative: a byte's top bit of `pos` says that it is positive (NaN too).
__device__ __forceinline__ void gate4(f4& v, uint32_t codes) {
  const uint32_t pos = ((codes & 0x7f7f7f7fu) + 0x7f7f7f7fu) & ~codes;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    v[j] = __uint_as_float(__float_as_uint(v[j]) & (uint32_t)__builtin_amdgcn_sbfe((int)pos, 8 * j + 7, 1));
}

// A row's scale byte from the largest magnitude of a lane's 32 values, `top`; `finite` finds the largest
// finite one, where top is infinite.
template <class F>
__device__ __forceinline__ int row_byte(float top, F finite) {
  top = lanes4_max(top);
  if (__builtin_expect(__any(top == __builtin_inff()), 0)) top = lanes4_max(finite());
  return scale_byte(top);
}

// A wave's tile (OUT_KEPT's order) as codes: a lane's 32 outputs of a row are the columns that XFrag has of
// it, so the codes are the next product's operand as they are.
template <int MT>
__device__ __forceinline__ void keep_tile(const f4 (&acc)[8][MT], XFrag<MT>& h) {
  h.scale = 0;
#pragma unroll
  for (int q = 0; q < MT; ++q) {
    __builtin_amdgcn_sched_barrier(0);   // one row of a lane at a time
    float top = 0.f;
#pragma unroll
    for (int t = 0; t < 8; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j) top = fmaxf(top, fabsf(acc[t][q][j]));
    const int byte = row_byte(top, [&] {
      float f = 0.f;
#pragma unroll
      for (int t = 0; t < 8; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) f = fmaxf(f, fabsf(acc[t][q][j]) < __builtin_inff() ? fabsf(acc[t][q][j]) : 0.f);
      return f;
    });
    const float f = scale_value(byte);
    h.scale |= (uint32_t)byte << (8 * q);
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const f4 v = acc[a * 4 + b][q];
        h.v[q][a][b] = encode4(v[0], v[1], v[2], v[3], f);
      }
  }
}

// Stores a wave's codes and scale bytes: `codes` and `scales` at its first row and group, `left` rows exist,
// `width` bytes of a row from the group on.
template <int MT>
__device__ __forceinline__ void store_kept(const XFrag<MT>& h, uint8_t* codes, uint8_t* scales, int pitch, int left,
                                           int width, int r, int g) {
#pragma unroll
  for (int q = 0; q < MT; ++q)
#pragma unroll
    for (int a = 0; a < 2; ++a)
      if (MT * r + q < left && a * 64 < width)
        *reinterpret_cast<u32x4*>(codes + __umul24(MT * r + q, pitch) + a * 64 + g * 16) = h.v[q][a];
  if (g == 0) {
    if (MT * r + MT - 1 < left) {
      if constexpr (MT == 4) *reinterpret_cast<uint32_t*>(scales + MT * r) = h.scale;
      else *reinterpret_cast<uint16_t*>(scales + MT * r) = (uint16_t)h.scale;
    } else {
#pragma unroll
      for (int q = 0; q < MT - 1; ++q)
        if (MT * r + q < left) scales[MT * r + q] = (uint8_t)(h.scale >> (8 * q));
    }
  }
}

// Storage words of a run of outputs: 16 bytes.
template <int OUT>
__device__ __forceinline__ float run_get(const u32x4& o, int j) {
  if constexpr (OUT == DT_F32) return __uint_as_float(o[j]);
  else if constexpr (OUT == DT_BF16) return __uint_as_float(j & 1 ? o[j / 2] & 0xffff0000u : o[j / 2] << 16);
  else return h2f((uint16_t)(j & 1 ? o[j / 2] >> 16 : o[j / 2]));
}
template <int OUT>
__device__ __forceinline__ uint32_t run_word(float v0, float v1) {
  if constexpr (OUT == DT_F32) return __float_as_uint(v0);
  else if constexpr (OUT == DT_BF16) return (uint32_t)f2bf(v0) | (uint32_t)f2bf(v1) << 16;
  else return __builtin_bit_cast(uint32_t, h2{(_Float16)v0, (_Float16)v1});
}

// A wave's tile stored: ReLU or its gradient, then the residual.
template <int OUT, int NT, int MT>
__device__ __forceinline__ void finish(f4 (&acc)[NT][MT], const LinearParams& p, long long m0, int n0, int r, int g) {
  typedef typename Act<OUT>::T T;
  constexpr int P = Run<OUT>::PER, L = 4 * P, RUNS = NT / P;    // a lane: RUNS runs of L outputs for each of MT rows
  constexpr int E = 4 / (int)sizeof(T);                        // outputs of a word
  const int left = (int)min((long long)16 * MT, p.rows - m0), N = p.outputs - n0;
#pragma unroll
  for (int q = 0; q < MT; ++q) {
    __builtin_amdgcn_sched_barrier(0);   // one row of a lane at a time
    if (p.relu) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[t][q][j] = __builtin_elementwise_maximum(acc[t][q][j], 0.f);   // keeps NaN
    }
    if (p.relu_of) {
      const uint8_t* gate = p.relu_of + (size_t)(m0 + min(MT * r + q, left - 1)) * p.q.pitch + n0;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int n = n_of<OUT>(t, 4 * g);
        gate4(acc[t][q], *reinterpret_cast<const uint32_t*>(gate + min(n, p.q.pitch - n0 - 4)));
      }
    }
  }
  T* const out = static_cast<T*>(p.out) + (size_t)m0 * p.outputs + n0;
  const T* const res = static_cast<const T*>(p.residual) + (size_t)m0 * p.outputs + n0;
  if (left == 16 * MT && (N >= 16 * NT || N % (16 * P) == 0)) {     // uniform: rows and runs exist as a whole
    const char* const rb = reinterpret_cast<const char*>(res);
    char* const ob = reinterpret_cast<char*>(out);
#pragma unroll
    for (int q = 0; q < MT; ++q) {
      __builtin_amdgcn_sched_barrier(0);
      const uint32_t at = __umul24(MT * r + q, p.outputs * (int)sizeof(T)) + 16 * g;   // a run is 16 bytes, 4 lanes' 64
      if (p.residual) {
        u32x4 o[RUNS];
#pragma unroll
        for (int a = 0; a < RUNS; ++a)
          if (a * 16 * P < N) __builtin_memcpy(&o[a], rb + (at + a * 64), 16);
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[t][q][j] += run_get<OUT>(o[t / P], t % P * 4 + j);
      }
#pragma unroll
      for (int a = 0; a < RUNS; ++a) {
        u32x4 w;
#pragma unroll
        for (int j = 0; j < L; j += E) w[j / E] = run_word<OUT>(acc[a * P + j / 4][q][j % 4], acc[a * P + j / 4][q][(j + E - 1) % 4]);
        if (a * 16 * P < N) __builtin_memcpy(ob + (at + a * 64), &w, 16);
      }
    }
    return;
  }
  asm volatile("" : "+v"(r), "+v"(g));     // or the offsets of this rare path would be kept in registers throughout
#pragma unroll
  for (int q = 0; q < MT; ++q) {
    __builtin_amdgcn_sched_barrier(0);
    if (MT * r + q >= left) continue;
    const size_t at = (size_t)(MT * r + q) * p.outputs;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int n = n_of<OUT>(t, 4 * g) + j;
        if (n < N) {
          float v = acc[t][q][j];
          if (p.residual) v += Act<OUT>::ld(res + at + n);
          Act<OUT>::st(out + at + n, v);
        }
      }
  }
}

}  // namespace lf
