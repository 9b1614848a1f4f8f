// Products of 8-bit operands: out[m][n] = sum_k x[m][k] w[n][k], x a checkpoint (a scale per row and 128
// columns), w packed (a scale per tile of 128 x 128), with bias, ReLU or a ReLU's gradient, residual,
// and an output that is kept in 8 bits itself.
//
// A wave computes 64 rows by 128 outputs.  w is the matrix instruction's first operand, so a lane's
// accumulators hold 4 consecutive outputs of one row per tile of 16; which tile holds which outputs is
// chosen so that a lane's runs fill 16-byte stores (n_of).  x goes from memory straight to registers, one
// step of 128 columns ahead; w lies in LDS as tiles of 128 x 128 codes, copied there by direct loads in
// an order that spreads a fragment's rows over the banks (key_of).
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
constexpr int WAVES = 8, NT = WAVES * 64;
constexpr int MROWS = 64;                 // rows of a wave's tile
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

// One step's rows of x for a lane: rows 4 r + t (r = lane % 16), columns 16 g .. and 64 + 16 g .. of the
// group (both operands take their columns in this order), and the four rows' scale bytes.
struct XFrag {
  u32x4 v[4][2];
  uint32_t scale;
};

__device__ __forceinline__ void x_load(XFrag& x, const LinearParams& p, long long m0, int kb, int r, int g) {
  const uint8_t* base = p.x.codes + (size_t)m0 * p.x.pitch + kb * GROUP;
  const int left = (int)min((long long)MROWS, p.rows - m0);
  const bool whole = kb * GROUP + 64 < p.x.pitch;    // uniform
#pragma unroll
  for (int t = 0; t < 4; ++t) {   // a uniform base and a 32-bit lane offset
    const uint32_t a = (uint32_t)min(4 * r + t, left - 1) * (uint32_t)p.x.pitch + 16 * g;
    x.v[t][0] = *reinterpret_cast<const u32x4*>(base + a);
    if (whole) x.v[t][1] = *reinterpret_cast<const u32x4*>(base + a + 64);
    else x.v[t][1] = u32x4{0, 0, 0, 0};
  }
  const long long s = min(m0 + 4 * r, (long long)p.x.sp - 4);
  x.scale = *reinterpret_cast<const uint32_t*>(p.x.scales + (size_t)kb * p.x.sp + s);
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

// acc = bias, 128 floats in LDS: a lane's accumulators of tile t are 4 consecutive outputs.
template <int OUT>
__device__ __forceinline__ void start(f4 (&acc)[8][4], const float* bias, int g) {
#pragma unroll
  for (int t = 0; t < 8; ++t)
#pragma unroll
    for (int q = 0; q < 4; ++q) acc[t][q] = *reinterpret_cast<const f4*>(bias + n_of<OUT>(t, 4 * g));
}

// acc += one step: 128 outputs x 64 rows x 128 columns.  w: the lane's place in an LDS tile, wx
// the same with the other half of the columns.  A tile's fragment is read while the one before it is
// multiplied; the barriers keep the compiler from reading all eight at once, which would spill.  next()
// loads the next step's rows: once the first half of this one's is converted, where it is.
template <int OUT, class NEXT>
__device__ __forceinline__ void mma(f4 (&acc)[8][4], const uint8_t* w, const uint8_t* wx, const XFrag& x, int wscale,
                                    NEXT next) {
#if __HIP_DEVICE_COMPILE__
  if constexpr (OUT == DT_F16 || OUT == DT_BF16) {
    next();
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
      const u32x4 c0 = a0[t & 1], c1 = a1[t & 1];
      const i8v a = {(int)c0.x, (int)c0.y, (int)c0.z, (int)c0.w, (int)c1.x, (int)c1.y, (int)c1.z, (int)c1.w};
#define LF_MM(q)                                                                                                   \
  {                                                                                                                \
    const i8v b = {(int)x.v[q][0].x, (int)x.v[q][0].y, (int)x.v[q][0].z, (int)x.v[q][0].w,                         \
                   (int)x.v[q][1].x, (int)x.v[q][1].y, (int)x.v[q][1].z, (int)x.v[q][1].w};                        \
    acc[t][q] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc[t][q], 0, 0, 0, wscale, q,                  \
                                                                 (int)x.scale);                                    \
  }
      LF_MM(0) LF_MM(1) LF_MM(2) LF_MM(3)
#undef LF_MM
      __builtin_amdgcn_sched_barrier(0);
    }
  } else {
    const float sw = scale_value(wscale);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const uint8_t* wh = half ? wx : w;
      b8 b[4][2];
      u32x4 a[2];
      a[0] = *reinterpret_cast<const u32x4*>(wh);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float sx = scale_value((x.scale >> (8 * q)) & 255);
        const u32x4 v = x.v[q][half];
        b[q][0] = codes_bf16(v.x, v.y, sx);
        b[q][1] = codes_bf16(v.z, v.w, sx);
      }
      if (half) next();
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        if (t < 7) a[(t + 1) & 1] = *reinterpret_cast<const u32x4*>(wh + n_of<OUT>(t + 1, 0) * GROUP);
        const u32x4 v = a[t & 1];
        const b8 a0 = codes_bf16(v.x, v.y, sw), a1 = codes_bf16(v.z, v.w, sw);
#pragma unroll
        for (int q = 0; q < 4; ++q)
          acc[t][q] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a0, b[q][0], acc[t][q], 0, 0, 0);
#pragma unroll
        for (int q = 0; q < 4; ++q) acc[t][q] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a1, b[q][1], acc[t][q], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
#endif
}

// ReLU or a ReLU's gradient, residual and store of a wave's tile.
template <int OUT>
__device__ __forceinline__ void finish(f4 (&acc)[8][4], const LinearParams& p, long long m0, int nb, int r, int g) {
  constexpr int P = Run<OUT>::PER, L = 4 * P, RUNS = 8 / P;    // a lane: RUNS runs of L outputs for each of 4 rows
  const int N = p.outputs;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const long long m = m0 + 4 * r + q;
    const bool row_ok = m < p.rows;
    const size_t row = row_ok ? (size_t)m : (size_t)p.rows - 1;
    __builtin_amdgcn_sched_barrier(0);   // one row of a lane at a time
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      if (p.relu) {
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[t][q][j] = __builtin_elementwise_maximum(acc[t][q][j], 0.f);   // keeps NaN
      }
    }
    if (p.relu_of) {
      const uint8_t* gate = p.relu_of + row * p.q.pitch + nb * GROUP;
#pragma unroll
      for (int a = 0; a < RUNS; ++a) {
        const int nl = a * 16 * P + g * L;
        if (nb * GROUP + nl < p.q.pitch) {
          uint32_t w[P];
          __builtin_memcpy(w, gate + nl, L);
#pragma unroll
          for (int b = 0; b < P; ++b)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if ((int8_t)(w[b] >> (8 * j)) <= 0) acc[a * P + b][q][j] = 0.f;
        }
      }
    }
    if constexpr (OUT == OUT_KEPT) {
      if (nb * GROUP + GROUP > N) {    // codes behind the last output are zeros
#pragma unroll
        for (int t = 0; t < 8; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (nb * GROUP + n_of<OUT>(t, 4 * g) + j >= N) acc[t][q][j] = 0.f;
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
      uint8_t* dst = p.q.codes + row * p.q.pitch + nb * GROUP;
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        u32x4 c;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const f4 v = acc[a * 4 + b][q];
          c[b] = encode4(v[0], v[1], v[2], v[3], f);
        }
        const int nl = a * 64 + g * 16;
        if (row_ok && nb * GROUP + nl < p.q.pitch) *reinterpret_cast<u32x4*>(dst + nl) = c;
      }
      if (row_ok && g == 0) p.q.scales[(size_t)nb * p.q.sp + row] = (uint8_t)byte;
    } else {
      typedef typename Act<OUT>::T T;
      if (row_ok) {
        const size_t at = row * (size_t)N + nb * GROUP;
#pragma unroll
        for (int a = 0; a < RUNS; ++a) {
          const int nl = a * 16 * P + g * L, left = N - nb * GROUP - nl;
          if (left >= L) {
            u32x4 o;
            if (p.residual) {
              float res[L];
              __builtin_memcpy(&o, static_cast<const T*>(p.residual) + at + nl, 16);
#pragma unroll
              for (int j = 0; j < L; ++j) {
                const uint32_t w = o[j * (int)sizeof(T) / 4];
                if constexpr (OUT == DT_F32) res[j] = __uint_as_float(w);
                else if constexpr (OUT == DT_BF16) res[j] = __uint_as_float(j & 1 ? w & 0xffff0000u : w << 16);
                else res[j] = h2f((uint16_t)(j & 1 ? w >> 16 : w));
                acc[a * P + j / 4][q][j % 4] += res[j];
              }
            }
#pragma unroll
            for (int j = 0; j < L; j += 4 / (int)sizeof(T)) {
              const float v0 = acc[a * P + j / 4][q][j % 4];
              uint32_t w;
              if constexpr (OUT == DT_F32) {
                w = __float_as_uint(v0);
              } else {
                const float v1 = acc[a * P + j / 4][q][j % 4 + 1];
                if constexpr (OUT == DT_BF16) w = (uint32_t)f2bf(v0) | (uint32_t)f2bf(v1) << 16;
                else w = __builtin_bit_cast(uint32_t, h2{(_Float16)v0, (_Float16)v1});
              }
              o[j * (int)sizeof(T) / 4] = w;
            }
            __builtin_memcpy(static_cast<T*>(p.out) + at + nl, &o, 16);
          } else {
#pragma unroll
            for (int j = 0; j < L; ++j)
              if (j < left) {
                float v = acc[a * P + j / 4][q][j % 4];
                if (p.residual) v += Act<OUT>::ld(static_cast<const T*>(p.residual) + at + nl + j);
                Act<OUT>::st(static_cast<T*>(p.out) + at + nl + j, v);
              }
          }
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
// then run through (64 rows, output group) units with no barrier, each loading the next step's rows
// before it multiplies this one's.  Units of the same rows run in neighbouring waves.
template <int OUT>
__global__ __launch_bounds__(NT, 2) void fp8_linear_resident_kernel(LinearParams p, LinearGrid q) {
  extern __shared__ __attribute__((aligned(16))) uint8_t fp8_smem[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int nbs = (p.outputs + GROUP - 1) / GROUP, kbs = (p.inputs + GROUP - 1) / GROUP;
  // blocks of the same rows and other subsets share an XCD (blocks are dealt out to 8 in turn)
  const int slot = blockIdx.x >> 3, subset = slot % q.subsets, blk = slot / q.subsets * 8 + (blockIdx.x & 7);
  if (blk >= q.blocks) return;
  const int nb0 = subset * q.per, per = min(q.per, nbs - nb0);
  float* bias = reinterpret_cast<float*>(fp8_smem + (size_t)q.per * kbs * WTILE);
  for (int i = wave; i < per * kbs * 16; i += WAVES)
    w_stage<OUT>(fp8_smem + (i >> 4) * WTILE, p, nb0 + (i >> 4) / kbs, (i >> 4) % kbs, i & 15, lane);
  for (int i = threadIdx.x; i < per * GROUP; i += NT)
    bias[i] = p.bias && nb0 * GROUP + i < p.outputs ? p.bias[nb0 * GROUP + i] : 0.f;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();

  // this block's units, of (rows / 64) x per, and the wave's first; a unit is (row tile, output group)
  const long long units = ((long long)p.rows + MROWS - 1) / MROWS * per;
  const int u0 = (int)(units * blk / q.blocks), u1 = (int)(units * (blk + 1) / q.blocks);
  const int i16 = n_of<OUT>(0, r);
  const uint8_t* wl = fp8_smem + i16 * GROUP + ((g ^ key_of<OUT>(i16)) << 4);
  const uint8_t* wlx = fp8_smem + i16 * GROUP + ((g ^ key_of<OUT>(i16) ^ 4) << 4);
  f4 acc[8][4];
  XFrag x, xn;
  int u = u0 + wave, kb = 0, mt = u / per, nb = u % per;
  const int mstep = WAVES / per, nstep = WAVES % per;
  if (u >= u1) return;
  x_load(x, p, (long long)mt * MROWS, 0, r, g);
  for (;;) {
    const int kb_now = kb, mt_now = mt, nb_now = nb;
    if (++kb == kbs) {
      kb = 0;
      u += WAVES;
      if (u < u1) {      // past the last step the same rows again, which nothing uses
        mt += mstep;
        nb += nstep;
        if (nb >= per) {
          nb -= per;
          ++mt;
        }
      }
    }
    if (kb_now == 0) start<OUT>(acc, bias + nb_now * GROUP, g);
    const int at = (nb_now * kbs + kb_now) * WTILE;
    mma<OUT>(acc, wl + at, wlx + at, x, p.ws[(nb0 + nb_now) * kbs + kb_now],
             [&]() __attribute__((always_inline)) { x_load(xn, p, (long long)mt * MROWS, kb, r, g); });
    if (kb_now == kbs - 1) finish<OUT>(acc, p, (long long)mt_now * MROWS, nb0 + nb_now, r, g);
    if (u >= u1) break;
    x = xn;
  }
}

// Rows m0 .. m0 + 63 of column group kb as x_load's fragments, from an LDS tile of 64 x 128 codes whose
// chunk c of row m lies at c ^ ((m >> 2) & 7), and their scale bytes from memory.
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
__global__ __launch_bounds__(NT, 2) void fp8_linear_stream_kernel(LinearParams p, LinearGrid q) {
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
  for (int i = threadIdx.x; i < 2 * GROUP; i += NT) {
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
  f4 acc[8][4];
  stage(fp8_smem, 0);
  uint32_t scale = *reinterpret_cast<const uint32_t*>(p.x.scales + srow);
  for (int kb = 0; kb < kbs; ++kb) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();     // step kb in LDS for every wave; every wave done with the other buffer
    if (kb == 0) start<OUT>(acc, bias + wn * GROUP, g);
    const int kn = min(kb + 1, kbs - 1);
    const uint8_t* buf = fp8_smem + (kb & 1) * STAGE;
    XFrag x;
    x.scale = scale;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      x.v[t][0] = *reinterpret_cast<const u32x4*>(buf + xl + t * GROUP);
      x.v[t][1] = *reinterpret_cast<const u32x4*>(buf + xlx + t * GROUP);
    }
    stage(fp8_smem + ((kb + 1) & 1) * STAGE, kn);
    scale = *reinterpret_cast<const uint32_t*>(p.x.scales + (size_t)kn * p.x.sp + srow);
    mma<OUT>(acc, buf + wl, buf + wlx, x, p.ws[(size_t)nbl * kbs + kb], []() {});
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the last copy, which nothing reads
  if (m0 < p.rows && nb < nbs) finish<OUT>(acc, p, m0, nb, r, g);
}

namespace {

template <int OUT>
int go(lf_context* ctx, const LinearParams& p) {
  const int nbs = (p.outputs + GROUP - 1) / GROUP, kbs = (p.inputs + GROUP - 1) / GROUP;
  const long long mt = ((long long)p.rows + MROWS - 1) / MROWS;
  const int cus = ctx->num_cus;
  LinearGrid q{};
  if (kbs <= RESIDENT_TILES) {
    // as many output groups a block as fit, but no more than keep every wave of the chip in units
    const int fit = RESIDENT_TILES / kbs;
    const long long busy = std::max<long long>(1, mt * nbs / ((long long)cus * WAVES));
    q.per = (int)std::min<long long>(std::min(fit, nbs), busy);
    q.subsets = (nbs + q.per - 1) / q.per;
    q.blocks = (int)std::min<long long>((mt * q.per + WAVES - 1) / WAVES, std::max(1, cus / q.subsets));
    static const bool lds = hipFuncSetAttribute(reinterpret_cast<const void*>(&fp8_linear_resident_kernel<OUT>),
                                                hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024) == hipSuccess;
    if (!lds) return set_error(LF_ERR_DEVICE, "fp8 linear: the device refuses the LDS it needs");
    const size_t smem = (size_t)q.per * (kbs * WTILE + GROUP * 4);
    const unsigned grid = (unsigned)((q.blocks + 7) / 8 * q.subsets * 8);
    hipLaunchKernelGGL((fp8_linear_resident_kernel<OUT>), dim3(grid), dim3(NT), smem, ctx->stream, p, q);
    return check_hip(hipGetLastError(), "fp8 linear launch");
  }
  constexpr int smem = 2 * (2 * WTILE + 4 * MROWS * GROUP);
  static const bool lds = hipFuncSetAttribute(reinterpret_cast<const void*>(&fp8_linear_stream_kernel<OUT>),
                                              hipFuncAttributeMaxDynamicSharedMemorySize, smem) == hipSuccess;
  if (!lds) return set_error(LF_ERR_DEVICE, "fp8 linear: the device refuses the LDS it needs");
  q.subsets = (nbs + 1) / 2;
  q.blocks = (int)((mt + 3) / 4);
  const unsigned grid = (unsigned)(((long long)q.blocks + 31) / 32 * 32 * q.subsets);
  hipLaunchKernelGGL((fp8_linear_stream_kernel<OUT>), dim3(grid), dim3(NT), smem, ctx->stream, p, q);
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
