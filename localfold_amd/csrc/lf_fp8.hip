// Products of 8-bit operands: out[m][n] = sum_k x[m][k] w[n][k], x a checkpoint (a scale per row and 128
// columns), w packed (a scale per tile of 128 x 128), with bias, ReLU or a ReLU's gradient, residual,
// and an output that is kept in 8 bits itself.
//
// A wave computes 16 MT rows by 128 outputs.  w is the matrix instruction's first operand, so a lane's
// accumulators hold 4 consecutive outputs of one row per tile of 16; which tile holds which outputs is
// chosen so that a lane's runs fill 16-byte stores (n_of).  w lies in LDS as tiles of 128 x 128 codes,
// copied there by direct loads in an order that spreads a fragment's rows over the banks (key_of).
//
// 16-bit outputs take the scaled 8-bit instruction (16x16x128), which multiplies the powers of two itself
// and has twice bfloat16's rate.  Of 8 products that it adds at a time it drops what lies 2^-13 below the
// largest (measured: 1.6e-5 of the result for normal inputs, where bfloat16 and half round by 2e-3 and
// 2e-4).  f32 outputs, and kept ones, whose codes would fall the other way near a border, take the bf16
// instruction on operands converted in registers, exactly: codes times a power of two fit bfloat16.
#include <algorithm>

#include "lf_train.h"

namespace lf {

typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));
typedef int i8v __attribute__((ext_vector_type(8)));

constexpr int OUT_KEPT = 3;               // beside DT_F32, DT_F16, DT_BF16
constexpr int WTILE = GROUP * GROUP;      // bytes of a weight tile
constexpr int RESIDENT_TILES = 9;         // 144 KB of LDS, which leaves room for the biases

__device__ const uint4 fp8_zero16 = {0, 0, 0, 0};

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

// No load has a condition, or the compiler could not count those in flight and would wait for all: rows past
// the end repeat the last one, and a half group's other half repeats its first until x_zero clears it.
// 24-bit products: a 64-bit multiply-add reads a register pair whose other half may be a load in flight.
template <int MT>
__device__ __forceinline__ void x_load(XFrag<MT>& x, const LinearParams& p, long long m0, int kb, int r, int g) {
  const uint8_t* base = p.x.codes + (size_t)m0 * p.x.pitch + kb * GROUP;
  const int left = (int)min((long long)16 * MT, p.rows - m0);
  const int second = kb * GROUP + 64 < p.x.pitch ? 64 : 0;    // uniform
#pragma unroll
  for (int t = 0; t < MT; ++t) {   // a uniform base and a 32-bit lane offset
    const uint32_t a = __umul24(min(MT * r + t, left - 1), p.x.pitch) + 16 * g;
    x.v[t][0] = *reinterpret_cast<const u32x4*>(base + a);
    x.v[t][1] = *reinterpret_cast<const u32x4*>(base + second + a);
  }
  // rows of scales are whole sixteens, so these are in bounds
  const uint8_t* sc = p.x.scales + (size_t)kb * p.x.sp + m0 + (uint32_t)min(MT * r, (left - 1) & ~(MT - 1));
  static_assert(MT == 2 || MT == 4, "scales of a lane's rows are one word");
  x.scale = MT == 2 ? *reinterpret_cast<const uint16_t*>(sc) : *reinterpret_cast<const uint32_t*>(sc);
}
template <int MT>
__device__ __forceinline__ void x_zero(XFrag<MT>& x, const LinearParams& p, int kb) {
  if (kb * GROUP + 64 >= p.x.pitch)
#pragma unroll
    for (int t = 0; t < MT; ++t) x.v[t][1] = u32x4{0, 0, 0, 0};
}

// Copies weight tile (nb, kb) to LDS: instruction `part` of 16 fills 8 rows.  Rows past the end repeat the
// last one (their outputs are not stored); a half group's other half is zeros.
template <int OUT>
__device__ __forceinline__ void w_stage(uint8_t* dst, const LinearParams& p, int nb, int kb, int part, int lane) {
  const int row = part * 8 + (lane >> 3);
  const int c = (lane & 7) ^ key_of<OUT>(row);
  const uint8_t* src = p.w + (size_t)min(nb * GROUP + row, p.outputs - 1) * p.x.pitch + kb * GROUP + c * 16;
  if (kb * GROUP + c * 16 >= p.x.pitch) src = reinterpret_cast<const uint8_t*>(&fp8_zero16);
#if __HIP_DEVICE_COMPILE__   // a target builtin: the host pass, which only emits the launch stub, lacks it
  __builtin_amdgcn_global_load_lds(src, dst + part * 1024, 16, 0, 0);
#else
  (void)src;
#endif
}

// acc += one step: 128 outputs x 16 MT rows x 128 columns; FIRST: acc = bias + the step, bias 128 floats in
// LDS.  w: the lane's place in an LDS tile, wx the same with the other half of the columns.  A tile's
// fragment is read while the one before it is multiplied; the barriers keep the compiler from reading
// all eight at once, which would spill.  next() may load over x: it is called once x is no longer read.
template <int OUT, bool FIRST, int MT, class NEXT>
__device__ __forceinline__ void mma(f4 (&acc)[8][MT], const uint8_t* w, const uint8_t* wx, const XFrag<MT>& x, int wscale,
                                    const float* bias, int g, NEXT next) {
  f4 c;
#if __HIP_DEVICE_COMPILE__
  if constexpr (OUT == DT_F16 || OUT == DT_BF16) {
    u32x4 a0[2], a1[2];
    a0[0] = *reinterpret_cast<const u32x4*>(w);
    a1[0] = *reinterpret_cast<const u32x4*>(wx);
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      if (t < 7) {
        const int at = n_of<OUT>(t + 1, 0) * GROUP;
        a0[(t + 1) & 1] = *reinterpret_cast<const u32x4*>(w + at);
        a1[(t + 1) & 1] = *reinterpret_cast<const u32x4*>(wx + at);
      }
      if constexpr (FIRST) c = *reinterpret_cast<const f4*>(bias + n_of<OUT>(t, 4 * g));
      const u32x4 c0 = a0[t & 1], c1 = a1[t & 1];
      const i8v a = {(int)c0.x, (int)c0.y, (int)c0.z, (int)c0.w, (int)c1.x, (int)c1.y, (int)c1.z, (int)c1.w};
#define LF_MM(q)                                                                                                  \
  if constexpr (q < MT) {                                                                                         \
    const i8v b = {(int)x.v[q][0].x, (int)x.v[q][0].y, (int)x.v[q][0].z, (int)x.v[q][0].w,                        \
                   (int)x.v[q][1].x, (int)x.v[q][1].y, (int)x.v[q][1].z, (int)x.v[q][1].w};                       \
    acc[t][q] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, FIRST ? c : acc[t][q], 0, 0, 0, wscale, q, \
                                                                 (int)x.scale);                                   \
  }
      LF_MM(0) LF_MM(1)
      if constexpr (MT == 4) {
        LF_MM(MT - 2) LF_MM(MT - 1)
      }
#undef LF_MM
      __builtin_amdgcn_sched_barrier(0);
    }
  } else {
    const float sw = scale_value(wscale);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
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
      for (int t = 0; t < 8; ++t) {
        if (t < 7) a[(t + 1) & 1] = *reinterpret_cast<const u32x4*>(wh + n_of<OUT>(t + 1, 0) * GROUP);
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
  }
#endif
  next();
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

// Zeros where the gate's code is zero or negative: a byte's top bit of `pos` says that it is positive (NaN too).
__device__ __forceinline__ void gate4(f4& v, uint32_t codes) {
  const uint32_t pos = ((codes & 0x7f7f7f7fu) + 0x7f7f7f7fu) & ~codes;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    v[j] = __uint_as_float(__float_as_uint(v[j]) & (uint32_t)__builtin_amdgcn_sbfe((int)pos, 8 * j + 7, 1));
}

// A wave's tile kept in 8 bits: ReLU or its gradient, the rows' scales, codes.
template <int MT>
__device__ __forceinline__ void finish_kept(f4 (&acc)[8][MT], const LinearParams& p, long long m0, int nb, int r, int g) {
  const int left = (int)min((long long)16 * MT, p.rows - m0), N = p.outputs - nb * GROUP, P = p.q.pitch - nb * GROUP;
  uint8_t* const codes = p.q.codes + (size_t)m0 * p.q.pitch + nb * GROUP;
  if (p.relu_of) {
    const uint8_t* const of = p.relu_of + (size_t)m0 * p.q.pitch + nb * GROUP;
    u32x4 gate[MT][2];
#pragma unroll
    for (int q = 0; q < MT; ++q)
#pragma unroll
      for (int a = 0; a < 2; ++a)
        gate[q][a] = *reinterpret_cast<const u32x4*>(of + __umul24(min(MT * r + q, left - 1), p.q.pitch) + min(a * 64 + g * 16, P - 16));
#pragma unroll
    for (int q = 0; q < MT; ++q)
#pragma unroll
      for (int t = 0; t < 8; ++t) gate4(acc[t][q], gate[q][t >> 2][t & 3]);
  }
  uint32_t bytes = 0;
#pragma unroll
  for (int q = 0; q < MT; ++q) {
    __builtin_amdgcn_sched_barrier(0);   // one row of a lane at a time
    if (p.relu) {
#pragma unroll
      for (int t = 0; t < 8; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[t][q][j] = __builtin_elementwise_maximum(acc[t][q][j], 0.f);   // keeps NaN
    }
    if (N < GROUP) {    // codes behind the last output are zeros
#pragma unroll
      for (int t = 0; t < 8; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n_of<OUT_KEPT>(t, 4 * g) + j >= N) acc[t][q][j] = 0.f;
    }
    float top = 0.f;
#pragma unroll
    for (int t = 0; t < 8; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j) top = fmaxf(top, fabsf(acc[t][q][j]));
    top = lanes4_max(top);
    if (__builtin_expect(__any(top == __builtin_inff()), 0)) {
      float f = 0.f;
#pragma unroll
      for (int t = 0; t < 8; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) f = fmaxf(f, fabsf(acc[t][q][j]) < __builtin_inff() ? fabsf(acc[t][q][j]) : 0.f);
      top = lanes4_max(f);
    }
    const int byte = scale_byte(top);
    const float f = scale_value(byte);
    bytes |= (uint32_t)byte << (8 * q);
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      u32x4 c;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const f4 v = acc[a * 4 + b][q];
        c[b] = encode4(v[0], v[1], v[2], v[3], f);
      }
      if (MT * r + q < left && a * 64 < P)
        *reinterpret_cast<u32x4*>(codes + __umul24(MT * r + q, p.q.pitch) + a * 64 + g * 16) = c;
    }
  }
  if (g == 0) {
    uint8_t* const sc = p.q.scales + (size_t)nb * p.q.sp + m0;
    if (MT * r + MT - 1 < left) {
      if constexpr (MT == 4) *reinterpret_cast<uint32_t*>(sc + MT * r) = bytes;
      else *reinterpret_cast<uint16_t*>(sc + MT * r) = (uint16_t)bytes;
    } else {
#pragma unroll
      for (int q = 0; q < MT - 1; ++q)
        if (MT * r + q < left) sc[MT * r + q] = (uint8_t)(bytes >> (8 * q));
    }
  }
}

// A wave's tile stored: ReLU or its gradient, then the residual.
template <int OUT, int MT>
__device__ __forceinline__ void finish(f4 (&acc)[8][MT], const LinearParams& p, long long m0, int nb, int r, int g) {
  if constexpr (OUT == OUT_KEPT) {
    finish_kept(acc, p, m0, nb, r, g);
  } else {
  typedef typename Act<OUT>::T T;
  constexpr int P = Run<OUT>::PER, L = 4 * P, RUNS = 8 / P;    // a lane: RUNS runs of L outputs for each of MT rows
  constexpr int E = 4 / (int)sizeof(T);                        // outputs of a word
  const int left = (int)min((long long)16 * MT, p.rows - m0), N = p.outputs - nb * GROUP;
#pragma unroll
  for (int q = 0; q < MT; ++q) {
    __builtin_amdgcn_sched_barrier(0);   // one row of a lane at a time
    if (p.relu) {
#pragma unroll
      for (int t = 0; t < 8; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[t][q][j] = __builtin_elementwise_maximum(acc[t][q][j], 0.f);   // keeps NaN
    }
    if (p.relu_of) {
      const uint8_t* gate = p.relu_of + (size_t)(m0 + min(MT * r + q, left - 1)) * p.q.pitch + nb * GROUP;
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        const int n = n_of<OUT>(t, 4 * g);
        gate4(acc[t][q], *reinterpret_cast<const uint32_t*>(gate + min(n, p.q.pitch - nb * GROUP - 4)));
      }
    }
  }
  T* const out = static_cast<T*>(p.out) + (size_t)m0 * p.outputs + nb * GROUP;
  const T* const res = static_cast<const T*>(p.residual) + (size_t)m0 * p.outputs + nb * GROUP;
  if (left == 16 * MT && (N >= GROUP || N % (16 * P) == 0)) {     // uniform: rows and runs exist as a whole
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
        for (int t = 0; t < 8; ++t)
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
    for (int t = 0; t < 8; ++t)
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
}

struct LinearGrid {
  int per;                      // resident: output groups of a subset
  int subsets;                  // subsets; stream: pairs of output groups
  int blocks;                   // blocks of a subset; stream: row tiles of 256
};

// Weights resident: a block copies its subset of output groups, all their columns, to LDS once; its waves
// then run through (32 rows, output group) units with no barrier, x straight from memory to registers.
// These shapes are bound by memory: 16 waves of 128 registers hide its latency better than 8 of 256 with
// 64 rows, at twice the LDS reads, of which there are enough.  Units of the same rows run in
// neighbouring waves.
constexpr int RW = 16, RM = 2;            // waves of a block, tiles of 16 rows of a wave

template <int OUT>
__global__ __launch_bounds__(RW * 64) void fp8_linear_resident_kernel(LinearParams p, LinearGrid q) {
  extern __shared__ __attribute__((aligned(16))) uint8_t fp8_smem[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int nbs = (p.outputs + GROUP - 1) / GROUP, kbs = (p.inputs + GROUP - 1) / GROUP;
  // blocks of the same rows and other subsets share an XCD (blocks are dealt out to 8 in turn)
  const int slot = blockIdx.x >> 3, subset = slot % q.subsets, blk = slot / q.subsets * 8 + (blockIdx.x & 7);
  if (blk >= q.blocks) return;
  const int nb0 = subset * q.per, per = min(q.per, nbs - nb0);
  float* bias = reinterpret_cast<float*>(fp8_smem + (size_t)q.per * kbs * WTILE);
  for (int i = wave; i < per * kbs * 16; i += RW)
    w_stage<OUT>(fp8_smem + (i >> 4) * WTILE, p, nb0 + (i >> 4) / kbs, (i >> 4) % kbs, i & 15, lane);
  for (int i = threadIdx.x; i < per * GROUP; i += RW * 64)
    bias[i] = p.bias && nb0 * GROUP + i < p.outputs ? p.bias[nb0 * GROUP + i] : 0.f;
  // this block's units, of (rows / 32) x per, and the wave's first; a unit is (row tile, output group)
  const long long units = ((long long)p.rows + 16 * RM - 1) / (16 * RM) * per;
  const int u0 = (int)(units * blk / q.blocks), u1 = (int)(units * (blk + 1) / q.blocks);
  const int i16 = n_of<OUT>(0, r);
  const uint8_t* wl = fp8_smem + i16 * GROUP + ((g ^ key_of<OUT>(i16)) << 4);
  const uint8_t* wlx = fp8_smem + i16 * GROUP + ((g ^ key_of<OUT>(i16) ^ 4) << 4);
  f4 acc[8][RM];
  XFrag<RM> x;
  int u = u0 + wave, mt = u / per, nb = u % per;
  const int mstep = RW / per, nstep = RW % per;
  const bool any = u < u1;
  x_load(x, p, any ? (long long)mt * 16 * RM : 0, 0, r, g);    // under way with the weights
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (!any) return;
  for (;;) {
    const int mt_now = mt, nb_now = nb;
    u += RW;
    if (u < u1) {      // past the last unit the same rows again, which nothing uses
      mt += mstep;
      nb += nstep;
      if (nb >= per) {
        nb -= per;
        ++mt;
      }
    }
    const uint8_t* const ws = p.ws + (nb0 + nb_now) * kbs;
    const float* const bn = bias + nb_now * GROUP;
    int at = nb_now * kbs * WTILE;
    x_zero(x, p, 0);
    mma<OUT, true>(acc, wl + at, wlx + at, x, ws[0], bn, g, [&]() __attribute__((always_inline)) {
      x_load(x, p, (long long)(kbs == 1 ? mt : mt_now) * 16 * RM, kbs == 1 ? 0 : 1, r, g);
    });
    for (int kb = 1; kb < kbs; ++kb) {
      at += WTILE;
      const bool last = kb + 1 == kbs;
      x_zero(x, p, kb);
      mma<OUT, false>(acc, wl + at, wlx + at, x, ws[kb], bn, g, [&]() __attribute__((always_inline)) {
        x_load(x, p, (long long)(last ? mt : mt_now) * 16 * RM, last ? 0 : kb + 1, r, g);
      });
    }
    finish<OUT>(acc, p, (long long)mt_now * 16 * RM, nb0 + nb_now, r, g);
    if (u >= u1) break;
  }
}

constexpr int SW = 8, SM = 4, MROWS = 16 * SM;   // the streaming kernel's waves, tiles and rows of a wave

// Copies rows m0 .. m0 + 63 of column group kb to an LDS tile whose chunk c of row m lies at
// c ^ ((m >> 2) & 7); instruction `part` of 8 fills 8 rows.
__device__ __forceinline__ void x_stage(uint8_t* dst, const LinearParams& p, long long m0, int kb, int part, int lane) {
  const int row = part * 8 + (lane >> 3), c = (lane & 7) ^ (row >> 2 & 7);
  const long long m = min(m0 + row, (long long)p.rows - 1);
  const uint8_t* src = p.x.codes + (size_t)m * p.x.pitch + kb * GROUP + c * 16;
  if (kb * GROUP + c * 16 >= p.x.pitch) src = reinterpret_cast<const uint8_t*>(&fp8_zero16);
#if __HIP_DEVICE_COMPILE__
  __builtin_amdgcn_global_load_lds(src, dst + part * 1024, 16, 0, 0);
#else
  (void)src;
#endif
}

// Long reductions: a block of 256 rows and two output groups walks the columns 128 at a time, tiles of both
// operands in two LDS buffers in turn.  One barrier a step; the next step's tiles are under way during this
// one's products.  Blocks on one XCD run through 4 row tiles and then the outputs, so its L2 serves both.
template <int OUT>
__global__ __launch_bounds__(SW * 64, 2) void fp8_linear_stream_kernel(LinearParams p, LinearGrid q) {
  extern __shared__ __attribute__((aligned(16))) uint8_t fp8_smem[];   // [2][2 weight tiles, 4 x tiles of 64 rows]
  __shared__ __attribute__((aligned(16))) float bias[2 * GROUP];
  constexpr int STAGE = 2 * WTILE + 4 * MROWS * GROUP;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int kbs = (p.inputs + GROUP - 1) / GROUP, nbs = (p.outputs + GROUP - 1) / GROUP;
  const int slot = blockIdx.x >> 3, nt = q.subsets, turn = slot / (4 * nt), in = slot % (4 * nt);
  const int mblk = (turn * 4 + in % 4) * 8 + (blockIdx.x & 7), nblk = in / 4;
  if (mblk >= q.blocks) return;
  const int wn = wave & 1, wm = wave >> 1, nb = nblk * 2 + wn;
  const long long m0 = (long long)mblk * 4 * MROWS + wm * MROWS;
  const int nbl = min(nb, nbs - 1);
  for (int i = threadIdx.x; i < 2 * GROUP; i += SW * 64) {
    const int n = nblk * 2 * GROUP + i;
    bias[i] = p.bias && n < p.outputs ? p.bias[n] : 0.f;
  }
  auto stage = [&](uint8_t* dst, int kb) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int part = wave * 4 + i;
      w_stage<OUT>(dst + (part >> 4) * WTILE, p, min(nblk * 2 + (part >> 4), nbs - 1), kb, part & 15, lane);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int part = wave * 4 + i;
      x_stage(dst + 2 * WTILE + (part >> 3) * MROWS * GROUP, p, (long long)(mblk * 4 + (part >> 3)) * MROWS, kb, part & 7, lane);
    }
  };
  const int i16 = n_of<OUT>(0, r);
  const int wl = wn * WTILE + i16 * GROUP + ((g ^ key_of<OUT>(i16)) << 4), wlx = wl ^ 64;
  // rows 4 r + t: chunk g ^ (r & 7)
  const int xl = 2 * WTILE + wm * MROWS * GROUP + r * 4 * GROUP + ((g ^ (r & 7)) << 4), xlx = xl ^ 64;
  const long long srow = min(m0 + 4 * r, (long long)p.x.sp - 4);
  stage(fp8_smem, 0);
  __syncthreads();     // the biases
  f4 acc[8][SM];
#pragma unroll
  for (int t = 0; t < 8; ++t)
#pragma unroll
    for (int q = 0; q < 4; ++q) acc[t][q] = *reinterpret_cast<const f4*>(bias + wn * GROUP + n_of<OUT>(t, 4 * g));
  uint32_t scale = *reinterpret_cast<const uint32_t*>(p.x.scales + srow);
  for (int kb = 0; kb < kbs; ++kb) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();     // step kb in LDS for every wave; every wave done with the other buffer
    const int kn = min(kb + 1, kbs - 1);
    const uint8_t* buf = fp8_smem + (kb & 1) * STAGE;
    XFrag<SM> x;
    x.scale = scale;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      x.v[t][0] = *reinterpret_cast<const u32x4*>(buf + xl + t * GROUP);
      x.v[t][1] = *reinterpret_cast<const u32x4*>(buf + xlx + t * GROUP);
    }
    stage(fp8_smem + ((kb + 1) & 1) * STAGE, kn);
    scale = *reinterpret_cast<const uint32_t*>(p.x.scales + (size_t)kn * p.x.sp + srow);
    mma<OUT, false>(acc, buf + wl, buf + wlx, x, p.ws[(size_t)nbl * kbs + kb], bias, g, []() {});
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the last copy, which nothing reads
  if (m0 < p.rows && nb < nbs) finish<OUT>(acc, p, m0, nb, r, g);
}

namespace {

template <int OUT>
int go(lf_context* ctx, const LinearParams& p) {
  const int nbs = (p.outputs + GROUP - 1) / GROUP, kbs = (p.inputs + GROUP - 1) / GROUP;
  const int cus = ctx->num_cus;
  LinearGrid q{};
  if (kbs <= RESIDENT_TILES) {
    const long long mt = ((long long)p.rows + 16 * RM - 1) / (16 * RM);
    // as many output groups a block as fit, but no more than keep every wave of the chip in units
    const int fit = RESIDENT_TILES / kbs;
    const long long busy = std::max<long long>(1, mt * nbs / ((long long)cus * RW));
    q.per = (int)std::min<long long>(std::min(fit, nbs), busy);
    q.subsets = (nbs + q.per - 1) / q.per;
    q.blocks = (int)std::min<long long>((mt * q.per + RW - 1) / RW, std::max(1, cus / q.subsets));
    static const bool lds = hipFuncSetAttribute(reinterpret_cast<const void*>(&fp8_linear_resident_kernel<OUT>),
                                                hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024) == hipSuccess;
    if (!lds) return set_error(LF_ERR_DEVICE, "fp8 linear: the device refuses the LDS it needs");
    const size_t smem = (size_t)q.per * (kbs * WTILE + GROUP * 4);
    const unsigned grid = (unsigned)((q.blocks + 7) / 8 * q.subsets * 8);
    hipLaunchKernelGGL((fp8_linear_resident_kernel<OUT>), dim3(grid), dim3(RW * 64), smem, ctx->stream, p, q);
    return check_hip(hipGetLastError(), "fp8 linear launch");
  }
  const long long mt = ((long long)p.rows + MROWS - 1) / MROWS;
  constexpr int smem = 2 * (2 * WTILE + 4 * MROWS * GROUP);
  static const bool lds = hipFuncSetAttribute(reinterpret_cast<const void*>(&fp8_linear_stream_kernel<OUT>),
                                              hipFuncAttributeMaxDynamicSharedMemorySize, smem) == hipSuccess;
  if (!lds) return set_error(LF_ERR_DEVICE, "fp8 linear: the device refuses the LDS it needs");
  q.subsets = (nbs + 1) / 2;
  q.blocks = (int)((mt + 3) / 4);
  const unsigned grid = (unsigned)(((long long)q.blocks + 31) / 32 * 32 * q.subsets);
  hipLaunchKernelGGL((fp8_linear_stream_kernel<OUT>), dim3(grid), dim3(SW * 64), smem, ctx->stream, p, q);
  return check_hip(hipGetLastError(), "fp8 linear launch");
}

}  // namespace

int run_fp8_linear(lf_context* ctx, const LinearParams& p, int out_dtype, const char* label) {
  LaunchScope ls(ctx, label);
  if (!p.out) return go<OUT_KEPT>(ctx, p);
  if (out_dtype == LF_F32) return go<DT_F32>(ctx, p);
  if (out_dtype == LF_F16) return go<DT_F16>(ctx, p);
  return go<DT_BF16>(ctx, p);
}

}  // namespace lf
