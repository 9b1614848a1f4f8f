// Products of 4-bit operands (lf_mx4_linear): out[m][n] = sum_k x[m][k] w[n][k], with bias, ReLU and residual.
//
// w is the instruction's first operand, so a lane's sums are outputs of one row.  Operands go by sets of 64
// rows, four tiles of 16: row i of tile t is row 4 f(i) + t of the set, so that the scale bytes of a lane's four tiles are
// one word of memory.
#include <algorithm>

#include "lf_mx4.h"

namespace lf {

namespace {

constexpr int KEPT = 3;          // beside DT_F32, DT_F16, DT_BF16: x is packed
constexpr int LDS_BYTES = 160 * 1024;

struct MxLinear {
  Mx x;                          // KEPT
  const void* act;               // or activations [rows][inputs]
  Mx w;
  int rows, inputs, outputs, steps;   // steps of 128 columns
  const float* bias;
  int relu;
  const void* residual;
  void* out;
  float* partial;                // split: [parts][rows][outputs]
};

// Which row of a set row i of the first operand's tiles belongs to: f puts the 16 outputs of a lane in runs of 16 bytes
// (PER_RUN outputs), four lanes' runs side by side.
template <int OUT>
__device__ __forceinline__ int mx_f(int i) {
  return OUT == DT_F32 ? (i & 3) * 4 + (i >> 2) : (i & 2) * 4 + (i >> 2) * 2 + (i & 1);
}

// One set of outputs from n0 on, rows m0 + MT r + q, stored.
template <int OUT, int MT>
__device__ __forceinline__ void mx_finish(const f4 (&acc)[4][MT], const MxLinear& p, long long m0, int n0, int r, int g) {
  typedef typename Act<OUT>::T T;
  constexpr int L = OUT == DT_F32 ? 4 : 8, RUNS = 16 / L;
#pragma unroll
  for (int q = 0; q < MT; ++q) {
    const long long m = m0 + MT * r + q;
    if (m >= p.rows) continue;
#pragma unroll
    for (int a = 0; a < RUNS; ++a) {
      const int n = n0 + (OUT == DT_F32 ? 16 * a + 4 * g : 32 * a + 8 * g), left = p.outputs - n;
      const size_t at = (size_t)m * p.outputs + n;
      T* const out = static_cast<T*>(p.out) + at;
      const T* const res = static_cast<const T*>(p.residual) + at;
      float v[8];
#pragma unroll
      for (int e = 0; e < L; ++e) {
        v[e] = OUT == DT_F32 ? acc[e][q][a] : acc[e & 3][q][2 * a + (e >> 2)];
        if (p.relu) v[e] = __builtin_elementwise_maximum(v[e], 0.f);   // keeps NaN
      }
      if constexpr (L == 8) {
        if (p.residual) {
          float w[8];
          load8<OUT>(res, left, w);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] += w[e];
        }
        store8<OUT>(out, left, v);
      } else if (left >= 4) {
        float4 w = make_float4(v[0], v[1], v[2], v[3]);
        if (p.residual) {
          float4 s;
          __builtin_memcpy(&s, res, 16);
          w = make_float4(w.x + s.x, w.y + s.y, w.z + s.z, w.w + s.w);
        }
        __builtin_memcpy(out, &w, 16);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (e < left) out[e] = p.residual ? v[e] + res[e] : v[e];
      }
    }
  }
}

// ---- weights resident: short reductions ------------------------------------------------------------

// A block copies its sets of outputs, all their columns, to LDS once, in the order in which a wave reads them: a tile's 64
// lanes side by side.  Its 16 waves then take 32 rows each in turn with no barrier, quantise them in registers (a lane
// holds whole groups) and run through the sets.
constexpr int RW = 16, RM = 2, MOST_STEPS = 4;
struct MxResident {
  int per, subsets, blocks;      // sets of a block, blocks that share the outputs, blocks of a subset
};

// Rows 2 r + q of m0 on, columns 32 g on of every step; rows past the end repeat the last one.
template <int SRC>
__device__ __forceinline__ void mx_rows_load(u32x4 (&v)[RM], uint32_t& scale, const MxLinear& p, long long m0, int kb, int r, int g) {
  if constexpr (SRC == KEPT) {
#pragma unroll
    for (int q = 0; q < RM; ++q)
      v[q] = *reinterpret_cast<const u32x4*>(p.x.codes + (size_t)min(m0 + RM * r + q, (long long)p.rows - 1) * p.x.pitch + kb * 64 + 16 * g);
    scale = *reinterpret_cast<const uint16_t*>(p.x.scales + (size_t)(4 * kb + g) * p.x.sp + min(m0 + RM * r, ((long long)p.rows - 1) & ~1LL));
  } else {
    typedef typename Act<SRC>::T T;
    MxRaw<SRC> raw[RM];
#pragma unroll
    for (int q = 0; q < RM; ++q) {
      const int c = kb * 128 + 32 * g;
      raw[q].load(static_cast<const T*>(p.act) + (size_t)min(m0 + RM * r + q, (long long)p.rows - 1) * p.inputs + c, p.inputs - c);
    }
    scale = 0;
#pragma unroll
    for (int q = 0; q < RM; ++q) scale |= (uint32_t)raw[q].quantise(v[q]) << (8 * q);
  }
}

template <int SRC, int OUT>
__global__ __launch_bounds__(RW * 64) void mx4_resident_kernel(MxLinear p, MxResident q) {
  extern __shared__ __attribute__((aligned(16))) uint8_t mx_smem[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int kbs = p.steps, sets = (p.outputs + 63) / 64;
  // blocks of the same rows and other subsets share an XCD (blocks are dealt out to 8 in turn)
  const int index = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3), subset = index % q.subsets, blk = index / q.subsets;
  if (blk >= q.blocks) return;
  const int set0 = subset * q.per, per = min(q.per, sets - set0);
  uint32_t* const ws = reinterpret_cast<uint32_t*>(mx_smem + (size_t)q.per * kbs * 4096);
  float* const bias = reinterpret_cast<float*>(ws + q.per * kbs * 64);
  for (int i = wave; i < per * kbs * 4; i += RW) {
    const int set = (i >> 2) / kbs, kb = (i >> 2) % kbs;
    const int n = min((set0 + set) * 64 + 4 * mx_f<OUT>(r) + (i & 3), p.outputs - 1);
    const uint8_t* src = p.w.codes + (size_t)n * p.w.pitch + kb * 64 + 16 * g;
#if __HIP_DEVICE_COMPILE__
    __builtin_amdgcn_global_load_lds(src, mx_smem + i * 1024, 16, 0, 0);
#else
    (void)src;
#endif
  }
  for (int i = wave; i < per * kbs; i += RW) {     // scale rows are whole sixteens
    const int set = i / kbs, kb = i % kbs, n = min((set0 + set) * 64 + 4 * mx_f<OUT>(r), (p.outputs - 1) & ~3);
    ws[i * 64 + lane] = *reinterpret_cast<const uint32_t*>(p.w.scales + (size_t)(4 * kb + g) * p.w.sp + n);
  }
  for (int i = threadIdx.x; i < per * 64; i += RW * 64) {     // [set][tile][row of a tile]
    const int n = (set0 + (i >> 6)) * 64 + 4 * mx_f<OUT>(i & 15) + ((i >> 4) & 3);
    bias[i] = p.bias && n < p.outputs ? p.bias[n] : 0.f;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  const long long units = ((long long)p.rows + 16 * RM - 1) / (16 * RM);
  for (long long u = (long long)blk * RW + wave; u < units; u += (long long)q.blocks * RW) {
    const long long m0 = u * 16 * RM;
    u32x4 x[MOST_STEPS][RM];
    uint32_t xs[MOST_STEPS];
#pragma unroll
    for (int kb = 0; kb < MOST_STEPS; ++kb)
      if (kb < kbs) mx_rows_load<SRC>(x[kb], xs[kb], p, m0, kb, r, g);
    for (int set = 0; set < per; ++set) {
      f4 acc[4][RM];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const f4 b = *reinterpret_cast<const f4*>(bias + set * 64 + t * 16 + 4 * g);
#pragma unroll
        for (int k = 0; k < RM; ++k) acc[t][k] = b;
      }
#pragma unroll
      for (int kb = 0; kb < MOST_STEPS; ++kb) {
        if (kb >= kbs) break;
        const uint8_t* at = mx_smem + (size_t)(set * kbs + kb) * 4096 + lane * 16;
        u32x4 a[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) a[t] = *reinterpret_cast<const u32x4*>(at + t * 1024);
        mx_mma_set<RM>(acc, a, x[kb], ws[(set * kbs + kb) * 64 + lane], xs[kb]);
      }
      mx_finish<OUT, RM>(acc, p, m0, (set0 + set) * 64, r, g);
    }
  }
}

// ---- streamed: long reductions ---------------------------------------------------------------------

// A block of WN WM waves computes WN NT 16 outputs by WM 64 rows, 128 columns a step.  Each wave copies one set of 64 rows
// of an operand, its codes in the order in which the waves read them (a tile's 64 lanes side by side) and its
// scale words, to one of four LDS buffers, three steps ahead; one barrier a step.
// Split: a block takes part of the steps and stores f32 sums to p.partial, joined by mx4_join_kernel.
struct MxStream {
  int mtiles, ntiles, parts;
};

template <int OUT, int NT, int WN, int WM, bool PART>
__global__ __launch_bounds__(WN * WM * 64, 2) void mx4_stream_kernel(MxLinear p, MxStream q) {
  constexpr int BN = WN * NT * 16, BM = WM * 64, SETS = WN * WM, AHEAD = 3, LOADS = 5;
  static_assert(SETS * 64 == BN + BM, "a wave copies a set");
  constexpr int STAGE = SETS * (4096 + 256);
  // Separate objects: reads of one are then known not to wait for copies into another.
  __shared__ __attribute__((aligned(16))) uint8_t S0[STAGE], S1[STAGE], S2[STAGE], S3[STAGE];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  int mt, nt, part;
  if constexpr (PART) {      // the tiles of a part on one XCD, whose L2 then reads that part once
    const int slot = blockIdx.x >> 3, tiles = q.mtiles * q.ntiles, tile = slot % tiles;
    part = slot / tiles * 8 + (blockIdx.x & 7);
    mt = tile % q.mtiles;
    nt = tile / q.mtiles;
    if (part >= q.parts) return;
  } else {                   // blocks on one XCD run through 4 tiles of rows and then the outputs
    const int slot = blockIdx.x >> 3, turn = slot / (4 * q.ntiles), in = slot % (4 * q.ntiles);
    mt = (turn * 4 + in % 4) * 8 + (blockIdx.x & 7);
    nt = in / 4;
    part = 0;
    if (mt >= q.mtiles) return;
  }
  const int s0 = (int)((long long)p.steps * part / q.parts), s1 = (int)((long long)p.steps * (part + 1) / q.parts);
  const long long m0 = (long long)mt * BM;
  const int n0 = nt * BN;
  // what this wave copies
  const bool of_w = wave < BN / 64;
  const Mx& src = of_w ? p.w : p.x;
  const long long first = of_w ? n0 + wave * 64 : m0 + (wave - BN / 64) * 64, last = (of_w ? p.outputs : p.rows) - 1;
  const long long base = min(first, last);
  const uint8_t* const codes = src.codes + (size_t)base * src.pitch;
  const int i0 = of_w ? 4 * mx_f<OUT>(r) : 4 * r;
  uint32_t off[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) off[t] = (uint32_t)(min(first + i0 + t, last) - base) * (uint32_t)src.pitch + 16 * g;
  const uint32_t soff = (uint32_t)(g * src.sp + min(first + i0, last & ~3LL));
  const uint32_t sstep = (uint32_t)(4 * src.sp);
  auto stage = [&](uint8_t* dst, int s) __attribute__((always_inline)) {
#if __HIP_DEVICE_COMPILE__
    const __amdgpu_buffer_rsrc_t cr = __builtin_amdgcn_make_buffer_rsrc((void*)codes, 0, 0xffffffffu, 0x27000);
    const __amdgpu_buffer_rsrc_t sr = __builtin_amdgcn_make_buffer_rsrc((void*)src.scales, 0, 0xffffffffu, 0x27000);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(sr, dst + SETS * 4096 + wave * 256, 4, soff, s * sstep, 0, 0);
#pragma unroll
    for (int t = 0; t < 4; ++t)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(cr, dst + wave * 4096 + t * 1024, 16, off[t], s * 64, 0, 0);
#else
    (void)codes, (void)dst, (void)s, (void)soff, (void)sstep;
#endif
  };
  const int wn = wave % WN, wm = wave / WN;
  f4 acc[NT / 4][4][4];
#pragma unroll
  for (int h = 0; h < NT / 4; ++h)
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      f4 b = {0.f, 0.f, 0.f, 0.f};
      if (!PART && p.bias) {
#pragma unroll
        for (int j = 0; j < 4; ++j) b[j] = p.bias[min(n0 + (wn * NT / 4 + h) * 64 + 4 * mx_f<OUT>(4 * g + j) + t, p.outputs - 1)];
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[h][t][k] = b;
    }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  stage(S0, s0);
  stage(S1, min(s0 + 1, s1 - 1));
  stage(S2, min(s0 + 2, s1 - 1));
  auto step = [&](int s, const uint8_t* buf, uint8_t* next) __attribute__((always_inline)) {
    // step s in LDS for every wave; every wave done with `next`, which held step s - 1
    static_assert((AHEAD - 1) * LOADS == 10, "the wait below");
    asm volatile("s_waitcnt vmcnt(10)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    stage(next, min(s + AHEAD, s1 - 1));      // past the end the last step again, which nothing reads
    __builtin_amdgcn_sched_barrier(0);
    u32x4 b[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) b[k] = *reinterpret_cast<const u32x4*>(buf + (BN / 16 + wm * 4 + k) * 1024 + lane * 16);
    const uint32_t sb = *reinterpret_cast<const uint32_t*>(buf + SETS * 4096 + (BN / 64 + wm) * 256 + lane * 4);
#pragma unroll
    for (int h = 0; h < NT / 4; ++h) {
      u32x4 a[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) a[t] = *reinterpret_cast<const u32x4*>(buf + (wn * NT + h * 4 + t) * 1024 + lane * 16);
      const uint32_t sa = *reinterpret_cast<const uint32_t*>(buf + SETS * 4096 + (wn * NT / 4 + h) * 256 + lane * 4);
      mx_mma_set<4>(acc[h], a, b, sa, sb);
    }
    // products touch no memory: without this they would be moved past the next step's barrier
#pragma unroll
    for (int h = 0; h < NT / 4; ++h)
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int k = 0; k < 4; ++k) asm volatile("" : "+v"(acc[h][t][k]));
  };
  int s = s0;
  for (; s + 3 < s1; s += 4) {
    step(s, S0, S3);
    step(s + 1, S1, S0);
    step(s + 2, S2, S1);
    step(s + 3, S3, S2);
  }
  if (s < s1) step(s, S0, S3);
  if (s + 1 < s1) step(s + 1, S1, S0);
  if (s + 2 < s1) step(s + 2, S2, S1);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the last copies, which nothing reads
#pragma unroll
  for (int h = 0; h < NT / 4; ++h) {
    const int n = n0 + (wn * NT / 4 + h) * 64;
    if (n >= p.outputs) continue;
    MxLinear o = p;
    if constexpr (PART) {
      o.relu = 0;
      o.residual = nullptr;
      o.out = p.partial + (size_t)part * p.rows * p.outputs;
    }
    mx_finish<OUT, 4>(acc[h], o, m0 + wm * 64, n, r, g);
  }
}

// The parts' sums, bias, ReLU, residual.
template <int OUT>
__global__ __launch_bounds__(256) void mx4_join_kernel(MxLinear p, int parts) {
  typedef typename Act<OUT>::T T;
  const size_t count = (size_t)p.rows * p.outputs;
  const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= count) return;
  float v = p.bias ? p.bias[i % p.outputs] : 0.f;
  for (int k = 0; k < parts; ++k) v += p.partial[k * count + i];
  if (p.relu) v = __builtin_elementwise_maximum(v, 0.f);
  if (p.residual) v += Act<OUT>::ld(static_cast<const T*>(p.residual) + i);
  Act<OUT>::st(static_cast<T*>(p.out) + i, v);
}

// ---- few rows or outputs -----------------------------------------------------------------------------

// What counts is the time to the last byte: a block computes 32 rows by 16 outputs, its waves steps of the columns in
// turn, operands straight from memory, sums joined in LDS.
constexpr int FW = 8;

template <int SRC, int OUT>
__global__ __launch_bounds__(FW * 64) void mx4_few_kernel(MxLinear p) {
  __shared__ f4 part[FW - 1][RM][64];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int waves = blockDim.x >> 6, n0 = blockIdx.x * 16;
  const long long m0 = (long long)blockIdx.y * 16 * RM;
  const int n = min(n0 + r, p.outputs - 1);
  const uint8_t* const wrow = p.w.codes + (size_t)n * p.w.pitch + 16 * g;
  const uint8_t* const wscale = p.w.scales + (size_t)g * p.w.sp + n;
  f4 acc[RM];
#pragma unroll
  for (int q = 0; q < RM; ++q) acc[q] = f4{0.f, 0.f, 0.f, 0.f};
  for (int kb = wave; kb < p.steps; kb += waves) {
    const u32x4 a = *reinterpret_cast<const u32x4*>(wrow + (size_t)kb * 64);
    const uint32_t sa = wscale[(size_t)4 * kb * p.w.sp];
    u32x4 b[RM];
    uint32_t sb;
    mx_rows_load<SRC>(b, sb, p, m0, kb, r, g);
    acc[0] = mx_mma<0, 0>(a, b[0], acc[0], sa, sb);
    acc[1] = mx_mma<0, 1>(a, b[1], acc[1], sa, sb);
  }
  if (wave > 0) {
#pragma unroll
    for (int q = 0; q < RM; ++q) part[wave - 1][q][lane] = acc[q];
  }
  __syncthreads();
  if (wave > 0) return;
  typedef typename Act<OUT>::T T;
#pragma unroll
  for (int q = 0; q < RM; ++q) {
    for (int k = 1; k < waves; ++k) acc[q] += part[k - 1][q][lane];
    const long long m = m0 + RM * r + q;
    if (m >= p.rows) continue;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int o = n0 + 4 * g + j;
      if (o >= p.outputs) continue;
      float v = acc[q][j] + (p.bias ? p.bias[o] : 0.f);
      if (p.relu) v = __builtin_elementwise_maximum(v, 0.f);
      const size_t at = (size_t)m * p.outputs + o;
      if (p.residual) v += Act<OUT>::ld(static_cast<const T*>(p.residual) + at);
      Act<OUT>::st(static_cast<T*>(p.out) + at, v);
    }
  }
}

// ---- which kernel ------------------------------------------------------------------------------------

enum { FEW, RESIDENT, STREAM };
struct MxPlan {
  int kind;
  bool wide;                 // STREAM: 256 x 256 tiles, else 128 x 128
  int parts;
};
constexpr int CUS = 256, FEW_TILES = 1500, FEW_STEPS = 64;

MxPlan mx_plan(long long rows, int steps, long long outputs) {
  const long long few = (rows + 31) / 32 * ((outputs + 15) / 16);
  if (few <= FEW_TILES && steps <= FEW_STEPS) return {FEW, false, 1};
  if (steps <= MOST_STEPS) return {RESIDENT, false, 1};
  const long long wide = (rows + 255) / 256 * ((outputs + 255) / 256);
  if (wide >= CUS / 2) return {STREAM, true, 1};
  const long long tiles = (rows + 127) / 128 * ((outputs + 127) / 128);
  // a part of 8 steps at least
  const int parts = (int)std::max<long long>(1, std::min<long long>(2 * CUS / tiles, steps / 8));
  return {STREAM, false, parts};
}

size_t up256(size_t n) { return (n + 255) & ~size_t(255); }

template <int OUT, int NT, int WN, int WM, bool PART>
void go_stream(lf_context* ctx, const MxLinear& p, int parts) {
  MxStream q{(p.rows + WM * 64 - 1) / (WM * 64), (p.outputs + WN * NT * 16 - 1) / (WN * NT * 16), parts};
  const long long blocks = PART ? (parts + 7LL) / 8 * 8 * q.mtiles * q.ntiles : (q.mtiles + 31LL) / 32 * 32 * q.ntiles;
  hipLaunchKernelGGL((mx4_stream_kernel<OUT, NT, WN, WM, PART>), dim3((unsigned)blocks), dim3(WN * WM * 64), 0, ctx->stream, p, q);
}

template <int SRC, int OUT>
int go_resident(lf_context* ctx, const MxLinear& p) {
  const int sets = (p.outputs + 63) / 64, set_bytes = p.steps * (4096 + 256) + 256;
  const long long units = ((long long)p.rows + 16 * RM - 1) / (16 * RM);
  MxResident q;
  // as many sets a block as fit, but no more than keep every wave of the chip busy
  const long long busy = std::max<long long>(1, units * sets / (CUS * RW));
  q.per = (int)std::min<long long>(std::min(LDS_BYTES / set_bytes, sets), busy);
  q.subsets = (sets + q.per - 1) / q.per;
  q.blocks = (int)std::min<long long>((units + 3) / 4, std::max(1, CUS / q.subsets));
  static const hipError_t lds = hipFuncSetAttribute(reinterpret_cast<const void*>(&mx4_resident_kernel<SRC, OUT>),
                                                    hipFuncAttributeMaxDynamicSharedMemorySize, LDS_BYTES);
  LF_TRY(check_hip(lds, "4-bit product LDS"));
  const unsigned grid = (unsigned)((q.blocks * q.subsets + 7) / 8 * 8);
  hipLaunchKernelGGL((mx4_resident_kernel<SRC, OUT>), dim3(grid), dim3(RW * 64), (size_t)q.per * set_bytes, ctx->stream, p, q);
  return LF_OK;
}

template <int SRC, int OUT>
int go_small(lf_context* ctx, const MxLinear& p, const MxPlan& plan) {
  if (plan.kind == RESIDENT) return go_resident<SRC, OUT>(ctx, p);
  hipLaunchKernelGGL((mx4_few_kernel<SRC, OUT>), dim3((p.outputs + 15) / 16, (p.rows + 31) / 32), dim3(std::min(p.steps, FW) * 64), 0,
                     ctx->stream, p);
  return LF_OK;
}

template <int OUT>
int go(lf_context* ctx, const MxLinear& p, const MxPlan& plan, int act_dtype) {
  if (plan.kind != STREAM) {
    LaunchScope ls(ctx, "mx4.linear");
    if (!p.act) LF_TRY((go_small<KEPT, OUT>(ctx, p, plan)));
    else if (act_dtype == LF_F32) LF_TRY((go_small<DT_F32, OUT>(ctx, p, plan)));
    else if (act_dtype == LF_F16) LF_TRY((go_small<DT_F16, OUT>(ctx, p, plan)));
    else LF_TRY((go_small<DT_BF16, OUT>(ctx, p, plan)));
    return check_hip(hipGetLastError(), "4-bit product launch");
  }
  {
    LaunchScope ls(ctx, "mx4.linear");
    if (plan.wide) go_stream<OUT, 8, 2, 4, false>(ctx, p, 1);
    else if (plan.parts == 1) go_stream<OUT, 4, 2, 2, false>(ctx, p, 1);
    else go_stream<DT_F32, 4, 2, 2, true>(ctx, p, plan.parts);
    LF_TRY(check_hip(hipGetLastError(), "4-bit product launch"));
  }
  if (plan.parts == 1) return LF_OK;
  LaunchScope ls(ctx, "mx4.join");
  const size_t count = (size_t)p.rows * p.outputs;
  hipLaunchKernelGGL((mx4_join_kernel<OUT>), dim3((unsigned)((count + 255) / 256)), dim3(256), 0, ctx->stream, p, plan.parts);
  return check_hip(hipGetLastError(), "4-bit join launch");
}

}  // namespace

size_t mx4_linear_bytes(int rows, int inputs, int outputs, bool from_act) {
  const MxPlan plan = mx_plan(rows, (int)(LF_MX4_PITCH(inputs) / 128), outputs);
  size_t n = 0;
  if (plan.kind == STREAM && from_act) n += up256((size_t)rows * LF_MX4_PITCH(inputs) / 2) + up256(LF_MX4_GROUPS(inputs) * LF_MX4_SCALE_PITCH(rows));
  if (plan.parts > 1) n += (size_t)plan.parts * rows * outputs * sizeof(float);
  return n;
}

int run_mx4_linear(lf_context* ctx, const lf_mx4_linear_args& a, void* scratch) {
  MxLinear p{};
  p.w = mx_view(*a.w);
  p.rows = a.rows;
  p.inputs = a.w->cols;
  p.outputs = a.w->rows;
  p.steps = (int)(LF_MX4_PITCH(p.inputs) / 128);
  p.bias = a.bias;
  p.relu = a.relu;
  p.residual = a.residual;
  p.out = a.out;
  const MxPlan plan = mx_plan(p.rows, p.steps, p.outputs);
  char* at = static_cast<char*>(scratch);
  if (a.kept) {
    p.x = mx_view(*a.kept);
  } else if (plan.kind != STREAM) {
    p.act = a.act;
  } else {
    const size_t codes = up256((size_t)p.rows * LF_MX4_PITCH(p.inputs) / 2);
    const lf_mx4 packed{p.rows, p.inputs, at, at + codes};
    at += codes + up256(LF_MX4_GROUPS(p.inputs) * LF_MX4_SCALE_PITCH(p.rows));
    lf_mx4_pack_args k{};
    k.rows = p.rows;
    k.cols = p.inputs;
    k.act_dtype = a.act_dtype;
    k.act = a.act;
    k.out = &packed;
    LF_TRY(run_mx4_pack(ctx, k, nullptr));
    p.x = mx_view(packed);
  }
  p.partial = reinterpret_cast<float*>(at);
  if (a.out_dtype == LF_F32) return go<DT_F32>(ctx, p, plan, a.act_dtype);
  if (a.out_dtype == LF_F16) return go<DT_F16>(ctx, p, plan, a.act_dtype);
  return go<DT_BF16>(ctx, p, plan, a.act_dtype);
}

}  // namespace lf
