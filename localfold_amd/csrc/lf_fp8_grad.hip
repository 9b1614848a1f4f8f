// Weight gradients of 8-bit operands: out[i][j] = sum_m a[m][i] b[m][j], a and b checkpoints of the same
// rows, and the column sums of one of them (the bias gradient).
//
// The reduction runs over the rows, along which each value has a scale of its own, so the codes are turned
// into bf16 (exactly) as they are staged into LDS, and the fragments, whose lanes need 8 rows of a column,
// are read from there by transposing reads.  A block of two teams of four waves computes a tile of
// 32 FI x 128 outputs over its share of the rows, the teams on alternate steps of 32 rows, joined in LDS;
// the blocks' partial sums are added in order by a second kernel.  Column sums are a product with ones.
#include <algorithm>

#include "lf_train.h"

namespace lf {

typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));
typedef short s4v __attribute__((ext_vector_type(4)));

constexpr int GN = 128;                   // outputs of a block along j
constexpr int GSTEP = 32;                 // rows of a step

struct GradParams {
  Kept a, b;
  float* partial;                         // [splits][a.cols][b.cols]; null: one split, straight to out
  float* colsum;                          // [splits][cols of the summed one], or null
  int sum_of;                             // 0: no column sums, 1: of a, 2: of b
  int splits, tiles, tiles_j;
  long long rows_per;                     // rows of a split, a multiple of 2 GSTEP
  void *out, *bias;
  int dt, swapped;                        // out is [b.cols][a.cols]
};

template <int FI>
struct GradShape {
  static constexpr int TI = 32 * FI;                       // outputs along i
  static constexpr int PA = TI * 2 + 32, PB = GN * 2 + 32; // LDS row pitches: 4 rows apart by 32 bytes mod 128
  static constexpr int BUF = GSTEP * (PA + PB);            // one team's buffer
  static constexpr int ITEMS = GSTEP * (TI + GN) / 16 / 256;   // 16-code pieces a lane stages
  static constexpr size_t SMEM = (size_t)(4 * BUF > TI * GN * 4 ? 4 * BUF : TI * GN * 4);
};

// The transposing read: of each 16 lanes, lanes 4k .. 4k+3 address row k's 16 columns, 4 each; lane i
// receives column i of the 4 rows.
__device__ __forceinline__ void tr_read(uint32_t (&o)[2], const uint8_t* p) {
#if __HIP_DEVICE_COMPILE__
  typedef __attribute__((address_space(3))) s4v* lds4;
  const s4v v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)p);
  __builtin_memcpy(o, &v, 8);
#else
  (void)o;
  (void)p;
#endif
}
// 16 columns of 32 rows as a bf16 fragment: lane group g has rows 4g .. and 16 + 4g ..
__device__ __forceinline__ b8 tr_frag(const uint8_t* p, int pitch) {
  uint32_t w[4], h[2];
  tr_read(h, p);
  w[0] = h[0];
  w[1] = h[1];
  tr_read(h, p + 16 * pitch);
  w[2] = h[0];
  w[3] = h[1];
  b8 o;
  __builtin_memcpy(&o, w, 16);
  return o;
}

template <int FI>
__global__ __launch_bounds__(512, 2) void weight_grad_kernel(GradParams p) {
  using S = GradShape<FI>;
  extern __shared__ __attribute__((aligned(16))) uint8_t grad_smem[];
  const int slot = blockIdx.x >> 3, tile = slot % p.tiles, split = slot / p.tiles * 8 + (blockIdx.x & 7);
  if (split >= p.splits) return;
  const int i0 = tile / p.tiles_j * S::TI, j0 = tile % p.tiles_j * GN;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int team = wave >> 2, wi = (wave >> 1) & 1, wj = wave & 1, tid = threadIdx.x & 255;
  const long long m0 = split * p.rows_per, m1 = min((long long)p.a.rows, m0 + p.rows_per);
  const int steps = (int)((m1 - m0 + 2 * GSTEP - 1) / (2 * GSTEP));
  uint8_t* mine = grad_smem + team * 2 * S::BUF;

  u32x4 raw[S::ITEMS];
  int sc[S::ITEMS];
  auto load = [&](int s) __attribute__((always_inline)) {
    const long long base = m0 + (long long)(2 * s + team) * GSTEP;
#pragma unroll
    for (int k = 0; k < S::ITEMS; ++k) {
      const int item = k * 256 + tid;
      const bool of_a = item < GSTEP * S::TI / 16;       // whole waves: the boundary is a multiple of 256
      const int e = of_a ? item : item - GSTEP * S::TI / 16, per = of_a ? S::TI / 16 : GN / 16;
      const int r = e / per, col = (of_a ? i0 : j0) + e % per * 16;
      const Kept& q = of_a ? p.a : p.b;
      raw[k] = u32x4{0, 0, 0, 0};
      sc[k] = 127;
      if (base + r < m1 && col < q.pitch) {
        raw[k] = *reinterpret_cast<const u32x4*>(q.codes + (size_t)(base + r) * q.pitch + col);
        sc[k] = q.scales[(size_t)(col / GROUP) * q.sp + base + r];
      }
    }
  };
  auto store = [&](int s) __attribute__((always_inline)) {
    uint8_t* buf = mine + (s & 1) * S::BUF;
#pragma unroll
    for (int k = 0; k < S::ITEMS; ++k) {
      const int item = k * 256 + tid;
      const bool of_a = item < GSTEP * S::TI / 16;
      const int e = of_a ? item : item - GSTEP * S::TI / 16, per = of_a ? S::TI / 16 : GN / 16;
      uint8_t* dst = buf + (of_a ? 0 : GSTEP * S::PA) + e / per * (of_a ? S::PA : S::PB) + e % per * 32;
      const float f = scale_value(sc[k]);
      uint32_t w[8];
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        w[2 * d] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)raw[k][d], f, false));
        w[2 * d + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)raw[k][d], f, true));
      }
      *reinterpret_cast<u32x4*>(dst) = u32x4{w[0], w[1], w[2], w[3]};
      *reinterpret_cast<u32x4*>(dst + 16) = u32x4{w[4], w[5], w[6], w[7]};
    }
  };

  f4 acc[FI][4], sums[FI / 2];
#pragma unroll
  for (int i = 0; i < FI; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < FI / 2; ++i) sums[i] = f4{0.f, 0.f, 0.f, 0.f};
  // column sums: blocks at the other operand's first tile, each fragment by one of the two waves that read it
  const bool sum_a = p.sum_of == 1 && j0 == 0, sum_b = p.sum_of == 2 && i0 == 0;
  b8 ones;
#pragma unroll
  for (int k = 0; k < 8; ++k) ones[k] = (__bf16)1.0f;
  const int g = lane >> 4, l16 = lane & 15;
  const int row = 4 * g + (l16 >> 2), cb = (l16 & 3) * 8;
  const int ao = row * S::PA + wi * FI * 32 + cb, bo = GSTEP * S::PA + row * S::PB + wj * 128 + cb;

  load(0);
  store(0);
  load(1);
  for (int s = 0; s < steps; ++s) {
    __syncthreads();     // step s in LDS; every wave done with the other buffer
    const uint8_t* buf = mine + (s & 1) * S::BUF;
    b8 fb[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) fb[j] = tr_frag(buf + bo + j * 32, S::PB);
    b8 fa[2];
    fa[0] = tr_frag(buf + ao, S::PA);
    if (s + 1 < steps) store(s + 1);
    load(s + 2);         // past the end: nothing is read
#pragma unroll
    for (int i = 0; i < FI; ++i) {
      if (i + 1 < FI) fa[(i + 1) & 1] = tr_frag(buf + ao + (i + 1) * 32, S::PA);
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa[i & 1], fb[j], acc[i][j], 0, 0, 0);
      if (sum_a && (i & 1) == wj) sums[i >> 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa[i & 1], ones, sums[i >> 1], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (sum_b) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if ((j & 1) == wi) sums[j >> 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, fb[j], sums[j >> 1], 0, 0, 0);
    }
  }

  // the second team's sums are added to the first's
  const int wt = wi * 2 + wj;
  f4* half = reinterpret_cast<f4*>(grad_smem) + wt * 64 + lane;      // [FI * 4][4 waves][64]
  __syncthreads();
  if (team == 1) {
#pragma unroll
    for (int i = 0; i < FI; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) half[(i * 4 + j) * 256] = acc[i][j];
  }
  __syncthreads();
  if (team == 0) {
#pragma unroll
    for (int i = 0; i < FI; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] += half[(i * 4 + j) * 256];
  }
  if (sum_a || sum_b) {     // uniform in the block
    __syncthreads();
    if (team == 1)
#pragma unroll
      for (int i = 0; i < FI / 2; ++i) half[i * 256] = sums[i];
    __syncthreads();
    if (team == 0)
#pragma unroll
      for (int i = 0; i < FI / 2; ++i) sums[i] += half[i * 256];
  }
  if (team == 1) return;
  const int ca = p.a.cols, cb2 = p.b.cols;
  float* dst = p.partial ? p.partial + (size_t)split * ca * cb2 : nullptr;
#pragma unroll
  for (int i = 0; i < FI; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int ci = i0 + (wi * FI + i) * 16 + 4 * g, cj = j0 + wj * 64 + j * 16 + l16;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (ci + k < ca && cj < cb2) {
          if (dst) dst[(size_t)(ci + k) * cb2 + cj] = acc[i][j][k];
          else store_act(p.out, p.dt, p.swapped ? (size_t)cj * ca + ci + k : (size_t)(ci + k) * cb2 + cj, acc[i][j][k]);
        }
    }
  if (sum_a) {
#pragma unroll
    for (int i = 0; i < FI; ++i)
      if ((i & 1) == wj && l16 == 0)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int c = i0 + (wi * FI + i) * 16 + 4 * g + k;
          if (c < ca) {
            if (dst) p.colsum[(size_t)split * ca + c] = sums[i >> 1][k];
            else store_act(p.bias, p.dt, c, sums[i >> 1][k]);
          }
        }
  }
  if (sum_b) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if ((j & 1) == wi && g == 0) {
        const int c = j0 + wj * 64 + j * 16 + l16;
        if (c < cb2) {
          if (dst) p.colsum[(size_t)split * cb2 + c] = sums[j >> 1][0];
          else store_act(p.bias, p.dt, c, sums[j >> 1][0]);
        }
      }
  }
}

// Partial sums added in order: 64 outputs a block, 16 runs of the splits at a time.
__global__ __launch_bounds__(256) void weight_grad_join_kernel(GradParams p, long long n, int cn) {
  __shared__ f4 sm[16][16];
  const int c = threadIdx.x & 15, run = threadIdx.x >> 4;
  const long long blocks_n = (n + 63) / 64;
  const bool main = blockIdx.x < blocks_n;
  const long long len = main ? n : cn, i = ((long long)blockIdx.x - (main ? 0 : blocks_n)) * 64 + c * 4;
  const float* src = main ? p.partial : p.colsum;
  const int per = (p.splits + 15) / 16, s0 = run * per, s1 = min(p.splits, s0 + per);
  f4 t = {0.f, 0.f, 0.f, 0.f};
  if (i + 4 <= len && len % 4 == 0) {
#pragma unroll 4
    for (int s = s0; s < s1; ++s) t += *reinterpret_cast<const f4*>(src + (size_t)s * len + i);
  } else {
    for (int s = s0; s < s1; ++s)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (i + k < len) t[k] += src[(size_t)s * len + i + k];
  }
  sm[run][c] = t;
  __syncthreads();
  if (run != 0) return;
  t = sm[0][c];
  for (int s = 1; s < 16; ++s) t += sm[s][c];
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (i + k < len) {
      const long long at = !main || !p.swapped ? i + k : (i + k) % p.b.cols * p.a.cols + (i + k) / p.b.cols;
      store_act(main ? p.out : p.bias, p.dt, (size_t)at, t[k]);
    }
}

namespace {

struct GradPlan {
  int fi, tiles, tiles_j, splits;
  long long rows_per;
};
// i is the wider matrix (ci >= cj).
GradPlan grad_plan(long long rows, int ci, int cj) {
  GradPlan q{};
  q.fi = ci > 128 ? 8 : 4;
  q.tiles_j = (cj + GN - 1) / GN;
  q.tiles = (ci + 32 * q.fi - 1) / (32 * q.fi) * q.tiles_j;
  const long long want = std::max<long long>(1, 256 / q.tiles);      // a block a CU
  const long long steps = (rows + 2 * GSTEP - 1) / (2 * GSTEP);
  q.rows_per = (steps + want - 1) / want * (2 * GSTEP);
  q.splits = (int)((rows + q.rows_per - 1) / q.rows_per);
  return q;
}

template <int FI>
int go(lf_context* ctx, const GradParams& p) {
  static const bool lds = hipFuncSetAttribute(reinterpret_cast<const void*>(&weight_grad_kernel<FI>),
                                              hipFuncAttributeMaxDynamicSharedMemorySize,
                                              (int)GradShape<FI>::SMEM) == hipSuccess;
  if (!lds) return set_error(LF_ERR_DEVICE, "weight gradient: the device refuses the LDS it needs");
  const unsigned grid = (unsigned)((p.splits + 7) / 8 * p.tiles * 8);
  hipLaunchKernelGGL((weight_grad_kernel<FI>), dim3(grid), dim3(512), GradShape<FI>::SMEM, ctx->stream, p);
  return check_hip(hipGetLastError(), "weight gradient launch");
}

size_t up16(size_t n) { return (n + 15) & ~size_t(15); }

}  // namespace

size_t weight_grad_partials(int rows, int outputs, int inputs) {
  const GradPlan q = grad_plan(rows, std::max(outputs, inputs), std::min(outputs, inputs));
  return up16((size_t)q.splits * outputs * inputs * sizeof(float)) + (size_t)q.splits * std::max(outputs, inputs) * sizeof(float);
}

int run_weight_grad(lf_context* ctx, const Kept& a, const Kept& b, void* out, void* bias, bool bias_of_b, int dt,
                    void* scratch, const char* label) {
  GradParams p{};
  p.swapped = a.cols < b.cols;
  p.a = p.swapped ? b : a;
  p.b = p.swapped ? a : b;
  const GradPlan q = grad_plan(a.rows, p.a.cols, p.b.cols);
  const long long n = (long long)a.cols * b.cols;
  p.sum_of = !bias ? 0 : bias_of_b == (p.swapped != 0) ? 1 : 2;
  p.splits = q.splits;
  p.tiles = q.tiles;
  p.tiles_j = q.tiles_j;
  p.rows_per = q.rows_per;
  p.out = out;
  p.bias = bias;
  p.dt = dt;
  if (q.splits > 1) {
    p.partial = static_cast<float*>(scratch);
    p.colsum = reinterpret_cast<float*>(static_cast<char*>(scratch) + up16((size_t)q.splits * n * sizeof(float)));
  }
  {
    LaunchScope ls(ctx, label);
    LF_TRY(q.fi == 8 ? go<8>(ctx, p) : go<4>(ctx, p));
  }
  if (q.splits == 1) return LF_OK;
  const int cn = p.sum_of == 0 ? 0 : p.sum_of == 1 ? p.a.cols : p.b.cols;
  LaunchScope ls(ctx, "fp8.weight_grad_join");
  hipLaunchKernelGGL(weight_grad_join_kernel, dim3((unsigned)((n + 63) / 64 + (cn + 63) / 64)), dim3(256), 0, ctx->stream, p,
                     n, cn);
  return check_hip(hipGetLastError(), "weight gradient join launch");
}

}  // namespace lf
