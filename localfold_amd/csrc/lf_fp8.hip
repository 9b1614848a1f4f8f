// Products of 8-bit operands: out[m][n] = sum_k x[m][k] w[n][k], x a checkpoint (a scale per row and 128
// columns), w packed (a scale per tile of 128 x 128), with bias, ReLU or a ReLU's gradient, residual,
// and an output that is kept in 8 bits itself.  A wave computes 16 MT rows by 128 outputs (lf_fp8.h).
#include <algorithm>

#include "lf_fp8.h"

namespace lf {

// 144 KB of LDS, which leaves room for the biases.  Longer reductions stream both operands.  bf16, us, resident and
// streamed: 147456 rows of 128 x 512 35 and 46, of 512 x 512 73 and 88, of 640 x 640 129 and 141, of 640 x 128 31
// and 53, of 1024 x 1024 269 and 282, 16384 rows of 1024 x 256 20 and 27; the other way 256 x 1024, 130 and 114.
// f32: 35 and 60 for 640 x 128, 95 and 104 for 1024 x 256, but 190 and 176 for 640 x 640, 337 and 282 for 384 x 1536:
// where outputs are many times the inputs, streaming gains up to 16 %.  The rule stays with what fits: neither
// outputs nor rows tell those shapes from 1152 x 1152, which is faster resident at any number of rows.
constexpr int RESIDENT_TILES = 9;

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

// A wave's tile kept in 8 bits: ReLU or its gradient, the rows' scales, codes.
template <int MT>
__device__ __forceinline__ void finish_kept(f4 (&acc)[8][MT], const LinearParams& p, long long m0, int nb, int r, int g) {
  const int left = (int)min((long long)16 * MT, p.rows - m0), N = p.outputs - nb * GROUP, P = p.q.pitch - nb * GROUP;
  const size_t at = (size_t)m0 * p.q.pitch + nb * GROUP;
  if (p.relu_of) {
    u32x4 gate[MT][2];
#pragma unroll
    for (int q = 0; q < MT; ++q)
#pragma unroll
      for (int a = 0; a < 2; ++a)
        gate[q][a] = *reinterpret_cast<const u32x4*>(p.relu_of + at + (__umul24(min(MT * r + q, left - 1), p.q.pitch) +
                                                                      min(a * 64 + g * 16, P - 16)));
#pragma unroll
    for (int q = 0; q < MT; ++q)
#pragma unroll
      for (int t = 0; t < 8; ++t) gate4(acc[t][q], gate[q][t >> 2][t & 3]);
  }
  if (p.relu) {
#pragma unroll
    for (int q = 0; q < MT; ++q)
#pragma unroll
      for (int t = 0; t < 8; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[t][q][j] = __builtin_elementwise_maximum(acc[t][q][j], 0.f);   // keeps NaN
  }
  if (N < GROUP) {    // codes behind the last output are zeros
#pragma unroll
    for (int q = 0; q < MT; ++q)
#pragma unroll
      for (int t = 0; t < 8; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n_of<OUT_KEPT>(t, 4 * g) + j >= N) acc[t][q][j] = 0.f;
  }
  XFrag<MT> h;
  keep_tile(acc, h);
  store_kept(h, p.q.codes + at, p.q.scales + (size_t)nb * p.q.sp + m0, p.q.pitch, left, P, r, g);
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
// neighbouring waves.  147456 rows of 128 x 512 in bf16: 35 us, 4.9 TB/s.
constexpr int RW = 16, RM = 2;            // waves of a block, tiles of 16 rows of a wave

template <int OUT>
__global__ __launch_bounds__(RW * 64) void fp8_linear_resident_kernel(LinearParams p, LinearGrid q) {
  extern __shared__ __attribute__((aligned(16))) uint8_t fp8_smem[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int nbs = (p.outputs + GROUP - 1) / GROUP, kbs = (p.inputs + GROUP - 1) / GROUP;
  // blocks of the same rows and other subsets share an XCD (blocks are dealt out to 8 in turn)
  const int index = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3), subset = index % q.subsets, blk = index / q.subsets;
  if (blk >= q.blocks) return;
  const int nb0 = subset * q.per, per = min(q.per, nbs - nb0);
  float* bias = reinterpret_cast<float*>(fp8_smem + (size_t)q.per * kbs * WTILE);
  for (int i = wave; i < per * kbs * 16; i += RW)
    w_stage<OUT>(fp8_smem + (i >> 4) * WTILE, p.w, p.x.pitch, p.outputs, nb0 + (i >> 4) / kbs, (i >> 4) % kbs, i & 15, lane);
  for (int i = threadIdx.x; i < per * GROUP; i += RW * 64)
    bias[i] = p.bias && nb0 * GROUP + i < p.outputs ? p.bias[nb0 * GROUP + i] : 0.f;
  // The scales too: a load from memory between the products would have to wait for the stores before it.
  uint8_t* wscales = reinterpret_cast<uint8_t*>(bias + q.per * GROUP);
  for (int i = threadIdx.x; i < per * kbs; i += RW * 64) wscales[i] = p.ws[nb0 * kbs + i];
  // this block's units, of (rows / 32) x per, and the wave's first; a unit is (row tile, output group)
  const long long units = ((long long)p.rows + 16 * RM - 1) / (16 * RM) * per;
  const int u0 = (int)(units * blk / q.blocks), u1 = (int)(units * (blk + 1) / q.blocks);
  const int i16 = n_of<OUT>(0, r);
  const int wl = i16 * GROUP + ((g ^ key_of<OUT>(i16)) << 4);     // the other half of the columns: ^ 64
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
    const uint8_t* const ws = wscales + nb_now * kbs;
    const float* const bn = bias + nb_now * GROUP;
    int at = nb_now * kbs * WTILE + wl;
    x_zero(x, p, 0);
    mma<OUT, true, false>(acc, fp8_smem + at, fp8_smem + (at ^ 64), x, ws[0], bn, g, [&]() __attribute__((always_inline)) {
      x_load(x, p, (long long)(kbs == 1 ? mt : mt_now) * 16 * RM, kbs == 1 ? 0 : 1, r, g);
    });
    for (int kb = 1; kb < kbs; ++kb) {
      at += WTILE;
      const bool last = kb + 1 == kbs;
      x_zero(x, p, kb);
      mma<OUT, false, false>(acc, fp8_smem + at, fp8_smem + (at ^ 64), x, ws[kb], bn, g, [&]() __attribute__((always_inline)) {
        x_load(x, p, (long long)(last ? mt : mt_now) * 16 * RM, last ? 0 : kb + 1, r, g);
      });
    }
    if constexpr (OUT == OUT_KEPT) finish_kept(acc, p, (long long)mt_now * 16 * RM, nb0 + nb_now, r, g);
    else finish<OUT>(acc, p, (long long)mt_now * 16 * RM, (nb0 + nb_now) * GROUP, r, g);
    if (u >= u1) break;
  }
}

constexpr int SW = 8, SM = 4, MROWS = 16 * SM;   // the streaming kernel's waves, tiles and rows of a wave

// Long reductions: a block of 256 rows and two output groups walks the columns 128 at a time, tiles of both
// operands in two LDS buffers in turn.  One barrier a step; the next step's tiles are under way during this
// one's products.  Blocks on one XCD run through 4 row tiles and then the outputs, so its L2 serves both.  8192 rows of
// 4096 x 4096 in bf16: 199 to 219 us, 1.26 to 1.38 PFLOP/s (a large bf16 library product has 1.2): matrix pipes busy 63 %,
// vector instructions, most of them conversions, 45 %, LDS reads 16 %.
template <int OUT>
__global__ __launch_bounds__(SW * 64, 2) void fp8_linear_stream_kernel(LinearParams p, LinearGrid q) {
  // Two weight tiles and 4 tiles of 64 rows each.  Separate objects: reads of one are then known not to wait
  // for copies into the other.
  constexpr int STAGE = 2 * WTILE + 4 * MROWS * GROUP;
  __shared__ __attribute__((aligned(16))) uint8_t S0[STAGE], S1[STAGE];
  __shared__ __attribute__((aligned(16))) float bias[2 * GROUP];
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
  // A step's copies: 8 rows of 128 bytes an instruction, four of weights and four of x a wave, at uniform bases
  // that move with the step and 32-bit lane offsets.  Rows past the end repeat the last one; the missing
  // half of a half group repeats its first, which x's zeros (below) take out of the sums.  Chunk c of x's
  // row m lies at c ^ (m >> 2 & 7).
  const uint8_t* const wbase = p.w + (size_t)nblk * 2 * GROUP * p.x.pitch;
  const uint8_t* const xbase = p.x.codes + (size_t)mblk * 4 * MROWS * p.x.pitch;
  uint32_t woff[4], xoff[4];    // bit 0: in the upper half of the group
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = (wave * 4 + i) * 8 + (lane >> 3);
    const int cw = (lane & 7) ^ key_of<OUT>(row & (GROUP - 1)), cx = (lane & 7) ^ (row >> 2 & 7);
    woff[i] = __umul24(min(row, p.outputs - 1 - nblk * 2 * GROUP), p.x.pitch) + (cw & 3) * 16 + (cw >> 2);
    xoff[i] = __umul24((int)min((long long)row, p.rows - 1 - (long long)mblk * 4 * MROWS), p.x.pitch) + (cx & 3) * 16 + (cx >> 2);
  }
  // Buffer instructions: after a global load into LDS every wait for LDS becomes a wait for that load too.
  auto stage = [&](uint8_t* dst, int kb) __attribute__((always_inline)) {
#if __HIP_DEVICE_COMPILE__
    const __amdgpu_buffer_rsrc_t wr = __builtin_amdgcn_make_buffer_rsrc((void*)wbase, 0, 0xffffffffu, 0x27000);
    const __amdgpu_buffer_rsrc_t xr = __builtin_amdgcn_make_buffer_rsrc((void*)xbase, 0, 0xffffffffu, 0x27000);
    const uint32_t up = kb * GROUP + 64 < p.x.pitch ? 63 : -1;     // uniform
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      __builtin_amdgcn_raw_ptr_buffer_load_lds(wr, dst + (wave * 4 + i) * 1024, 16, woff[i] + (woff[i] & 1) * up, kb * GROUP, 0, 0);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(xr, dst + 2 * WTILE + (wave * 4 + i) * 1024, 16,
                                               xoff[i] + (xoff[i] & 1) * up, kb * GROUP, 0, 0);
    }
#else
    (void)wbase;
    (void)xbase;
    (void)dst;
    (void)kb;
#endif
  };
  const int i16 = n_of<OUT>(0, r);
  const int wl = wn * WTILE + i16 * GROUP + ((g ^ key_of<OUT>(i16)) << 4), wlx = wl ^ 64;
  // rows 4 r + t: chunk g ^ (r & 7)
  const int xl = 2 * WTILE + wm * MROWS * GROUP + r * 4 * GROUP + ((g ^ (r & 7)) << 4), xlx = xl ^ 64;
  const long long srow = min(m0 + 4 * r, (long long)p.x.sp - 4);
  stage(S0, 0);
  __syncthreads();     // the biases
  f4 acc[8][SM];
#pragma unroll
  for (int t = 0; t < 8; ++t)
#pragma unroll
    for (int q = 0; q < SM; ++q) acc[t][q] = *reinterpret_cast<const f4*>(bias + wn * GROUP + n_of<OUT>(t, 4 * g));
  // the step's scales are loaded a step ahead too, before its copies: a wait for them is no wait for those
  uint32_t scale = *reinterpret_cast<const uint32_t*>(p.x.scales + srow);
  const uint8_t* const ws = p.ws + (size_t)nbl * kbs;
  int wscale = ws[0];
  auto step = [&](int kb, const uint8_t* buf, uint8_t* other) __attribute__((always_inline)) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();     // step kb in LDS for every wave; every wave done with the other buffer
    const int kn = min(kb + 1, kbs - 1);
    XFrag<SM> x;
    x.scale = scale;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      x.v[t][0] = *reinterpret_cast<const u32x4*>(buf + xl + t * GROUP);
      x.v[t][1] = *reinterpret_cast<const u32x4*>(buf + xlx + t * GROUP);
    }
    x_zero(x, p, kb);
    const int wnow = wscale;
    scale = *reinterpret_cast<const uint32_t*>(p.x.scales + (size_t)kn * p.x.sp + srow);
    wscale = ws[kn];
    __builtin_amdgcn_sched_barrier(0);
    stage(other, kn);
    __builtin_amdgcn_sched_barrier(0);     // the copies are under way first, the fragments come one by one
    mma<OUT, false, false>(acc, buf + wl, buf + wlx, x, wnow, bias, g, []() {});
    // products touch no memory: without this they would be moved past the next step's barrier
#pragma unroll
    for (int t = 0; t < 8; ++t)
#pragma unroll
      for (int q = 0; q < SM; ++q) asm volatile("" : "+v"(acc[t][q]));
  };
  int kb = 0;
  for (; kb + 1 < kbs; kb += 2) {
    step(kb, S0, S1);
    step(kb + 1, S1, S0);
  }
  if (kb < kbs) step(kb, S0, S1);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the last copy, which nothing reads
  if (m0 >= p.rows || nb >= nbs) return;
  if constexpr (OUT == OUT_KEPT) finish_kept(acc, p, m0, nb, r, g);
  else finish<OUT>(acc, p, m0, nb * GROUP, r, g);
}

// Small products: what counts is the time to the last byte.  A block computes 32 rows by one run of outputs,
// its waves a group of columns each, in turn, fragments straight from memory, sums joined in LDS.  256 rows of
// 384 x 1536 in bf16: 4.3 us, where a block that stages its weights first takes 10.
//
// Every block reads its weights and its rows from L2 again, so products of more than one block of rows and many
// outputs take the other kernels.  In
// tiles of 32 x 32 outputs the times cross between 1600 (1024 x 256) and 3500 (64 x 256) for resident
// weights (f32: 1300 and 3500), and for streamed ones between 3000 (1536 x 1536) and 6300 (4096 x 4096) (f32: 2300 and
// 4300).  bf16, us, small and other: 384 x 1536: 1024 rows 7.4 and 10.5, 4096 rows 22 and 13; 128 x 512: 2048 rows
// 3.9 and 7.1, 16384 rows 16 and 10; 4096 x 4096: 512 rows 60 and 174, 2048 rows 230 and 178.
constexpr int FW = 8, FM = 2;             // most waves of a block, tiles of 16 rows
constexpr int FEW_TILES = 1500, FEW_TILES_LONG = 3000;

template <int OUT>
__global__ __launch_bounds__(FW * 64) void fp8_linear_few_kernel(LinearParams p) {
  constexpr int NT = Run<OUT>::PER;
  __shared__ f4 part[FW - 1][NT][FM][64];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int waves = blockDim.x >> 6, kbs = (p.inputs + GROUP - 1) / GROUP;
  const int n0 = blockIdx.x * 16 * NT;
  const long long m0 = (long long)blockIdx.y * 16 * FM;
  const uint8_t* const wbase = p.w + (size_t)n0 * p.x.pitch;
  const uint8_t* const ws = p.ws + (size_t)(n0 / GROUP) * kbs;
  uint32_t woff[NT];
  f4 acc[NT][FM], bias[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    woff[t] = __umul24(min(n_of<OUT>(t, r), p.outputs - 1 - n0), p.x.pitch) + 16 * g;
#pragma unroll
    for (int q = 0; q < FM; ++q) acc[t][q] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 4; ++j) bias[t][j] = p.bias ? p.bias[min(n0 + n_of<OUT>(t, 4 * g) + j, p.outputs - 1)] : 0.f;
  }
  struct Step {
    XFrag<FM> x;
    u32x4 w[NT][2];
    int ws;
  };
  auto load = [&](Step& s, int kb) __attribute__((always_inline)) {
    const int second = kb * GROUP + 64 < p.x.pitch ? 64 : 0;    // uniform
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      s.w[t][0] = *reinterpret_cast<const u32x4*>(wbase + kb * GROUP + woff[t]);
      s.w[t][1] = *reinterpret_cast<const u32x4*>(wbase + kb * GROUP + second + woff[t]);
    }
    x_load(s.x, p, m0, kb, r, g);
    s.ws = ws[kb];
  };
  auto multiply = [&](Step& s, int kb) __attribute__((always_inline)) {
    x_zero(s.x, p, kb);
#pragma unroll
    for (int t = 0; t < NT; ++t) mma_frag(acc[t], s.w[t], s.x, s.ws);
  };
  for (int kb = wave; kb < kbs; kb += 2 * waves) {
    Step a, b;
    load(a, kb);
    load(b, min(kb + waves, kbs - 1));
    multiply(a, kb);
    if (kb + waves < kbs) multiply(b, kb + waves);
  }
  if (wave > 0) {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int q = 0; q < FM; ++q) part[wave - 1][t][q][lane] = acc[t][q];
  }
  __syncthreads();
  if (wave > 0) return;
  for (int k = 1; k < waves; ++k)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int q = 0; q < FM; ++q) acc[t][q] += part[k - 1][t][q][lane];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int q = 0; q < FM; ++q) acc[t][q] += bias[t];
  finish<OUT>(acc, p, m0, n0, r, g);
}

namespace {

template <int OUT>
int go(lf_context* ctx, const LinearParams& p) {
  const int nbs = (p.outputs + GROUP - 1) / GROUP, kbs = (p.inputs + GROUP - 1) / GROUP;
  const int cus = ctx->num_cus;
  LinearGrid q{};
  if constexpr (OUT != OUT_KEPT) {
    const long long mt = ((long long)p.rows + 16 * FM - 1) / (16 * FM), tiles = mt * ((p.outputs + 31) / 32);
    if (mt == 1 || tiles <= (kbs <= RESIDENT_TILES ? FEW_TILES : FEW_TILES_LONG)) {
      const dim3 grid((p.outputs + 16 * Run<OUT>::PER - 1) / (16 * Run<OUT>::PER), (unsigned)mt);
      hipLaunchKernelGGL((fp8_linear_few_kernel<OUT>), grid, dim3(std::min(kbs, FW) * 64), 0, ctx->stream, p);
      return check_hip(hipGetLastError(), "fp8 linear launch");
    }
  }
  if (kbs <= RESIDENT_TILES) {
    const long long mt = ((long long)p.rows + 16 * RM - 1) / (16 * RM);
    // as many output groups a block as fit, but no more than keep every wave of the chip in units
    const int fit = RESIDENT_TILES / kbs;
    const long long busy = std::max<long long>(1, mt * nbs / ((long long)cus * RW));
    q.per = (int)std::min<long long>(std::min(fit, nbs), busy);
    q.subsets = (nbs + q.per - 1) / q.per;
    // a unit for every SIMD before a second one: 8192 rows of 128 x 512 in 8.2 us, in blocks of 16 units 11.4
    q.blocks = (int)std::min<long long>((mt * q.per + 3) / 4, std::max(1, cus / q.subsets));
    static const bool lds = hipFuncSetAttribute(reinterpret_cast<const void*>(&fp8_linear_resident_kernel<OUT>),
                                                hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024) == hipSuccess;
    if (!lds) return set_error(LF_ERR_DEVICE, "fp8 linear: the device refuses the LDS it needs");
    const size_t smem = (size_t)q.per * (kbs * WTILE + GROUP * 4 + kbs);
    const unsigned grid = (unsigned)((q.blocks * q.subsets + 7) / 8 * 8);
    hipLaunchKernelGGL((fp8_linear_resident_kernel<OUT>), dim3(grid), dim3(RW * 64), smem, ctx->stream, p, q);
    return check_hip(hipGetLastError(), "fp8 linear launch");
  }
  const long long mt = ((long long)p.rows + MROWS - 1) / MROWS;
  q.subsets = (nbs + 1) / 2;
  q.blocks = (int)((mt + 3) / 4);
  const unsigned grid = (unsigned)(((long long)q.blocks + 31) / 32 * 32 * q.subsets);
  hipLaunchKernelGGL((fp8_linear_stream_kernel<OUT>), dim3(grid), dim3(SW * 64), 0, ctx->stream, p, q);
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
