// Products of 4-bit operands (lf_mx4_linear): out[m][n] = sum_k x[m][k] w[n][k], with bias, ReLU and residual.
//
// x is the instruction's first operand, w its second: a lane's sums are outputs of the column that it has of w.  w goes by
// sets of 64 rows, four tiles of 16, row i of tile t being row 4 i + t of the set: a lane then holds four
// neighbouring outputs, 16 lanes a run of 64 (one line of 16-bit outputs), and the scale bytes of its tiles are one word of
// memory.  x goes the same way, by 64 or 32 rows.
#include <algorithm>
#include <climits>

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

// One set of outputs from n0 on, rows m0 + MT i + q, stored.
template <int OUT>
struct MxFour {
  typename Act<OUT>::T v[4];
};
// SOON: the next kernel reads it.
template <int OUT, int MT, bool SOON = false>
__device__ __forceinline__ void mx_finish(const f4 (&acc)[4][MT], const MxLinear& p, long long m0, int n0, int r, int g) {
  typedef typename Act<OUT>::T T;
  const int rows = (int)min((long long)16 * MT, p.rows - m0), outputs = p.outputs - n0;
  const size_t first = (size_t)m0 * p.outputs + n0;
  T* const out = static_cast<T*>(p.out) + first;
  const T* const res = static_cast<const T*>(p.residual) + first;
  if (rows == 16 * MT && outputs >= 64 && p.outputs <= 1 << 20) {     // uniform; offsets fit 32 bits
    const uint32_t row = (uint32_t)p.outputs * sizeof(T), at = 4 * MT * g * row + 4 * r * (uint32_t)sizeof(T);
    char* const ob = reinterpret_cast<char*>(out);
    const char* const rb = reinterpret_cast<const char*>(res);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      __builtin_amdgcn_sched_barrier(0);   // few registers: some rows of a lane at a time
      MxFour<OUT> o[MT];
      if (p.residual) {
#pragma unroll
        for (int q = 0; q < MT; ++q) __builtin_memcpy(&o[q], rb + (at + (MT * j + q) * row), sizeof(o[q]));
#pragma unroll
        for (int q = 0; q < MT; ++q)
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const float v = p.relu ? __builtin_elementwise_maximum(acc[t][q][j], 0.f) : acc[t][q][j];   // keeps NaN
            Act<OUT>::st(o[q].v + t, v + Act<OUT>::ld(o[q].v + t));
          }
      } else {
#pragma unroll
        for (int q = 0; q < MT; ++q)
#pragma unroll
          for (int t = 0; t < 4; ++t) Act<OUT>::st(o[q].v + t, p.relu ? __builtin_elementwise_maximum(acc[t][q][j], 0.f) : acc[t][q][j]);
      }
#pragma unroll
      for (int q = 0; q < MT; ++q) {
        if constexpr (SOON) __builtin_memcpy(ob + (at + (MT * j + q) * row), &o[q], sizeof(o[q]));
        else stream_out(ob + (at + (MT * j + q) * row), o[q]);
      }
    }
    return;
  }
  asm volatile("" : "+v"(r), "+v"(g));     // or the offsets of this rare path would be kept in registers throughout
#pragma unroll
  for (int q = 0; q < MT; ++q)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      __builtin_amdgcn_sched_barrier(0);
      const int m = MT * (4 * g + j) + q;
      if (m >= rows) continue;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        if (4 * r + t >= outputs) continue;
        const size_t at = (size_t)m * p.outputs + 4 * r + t;
        float v = acc[t][q][j];
        if (p.relu) v = __builtin_elementwise_maximum(v, 0.f);
        Act<OUT>::st(out + at, p.residual ? v + Act<OUT>::ld(res + at) : v);
      }
    }
}

// ---- weights resident: short reductions ------------------------------------------------------------

// A block copies its sets of outputs, all their columns, to LDS once, in the order in which a wave reads them: a tile's 64
// lanes side by side.  Its waves then take 32 rows each in turn with no barrier, quantise them in registers (a lane holds
// whole groups; the next rows are under way meanwhile, where registers allow) and run through the sets.  Bound by what it
// writes: 147456 rows of 128 x 512 in bf16 take 46 us, 4.1 TB/s.
constexpr int RM = 2;            // tiles of 16 rows of a wave
struct MxResident {
  int per, subsets, blocks;      // sets of a block, blocks that share the outputs, blocks of a subset
};

// One step's rows MT r + q of m0 on, columns 32 g on; rows past the end repeat the last one.
template <int SRC, int MT>
struct MxRows {
  MxRaw<SRC> raw[MT];
  __device__ __forceinline__ void load(const MxLinear& p, long long m0, int kb, int r, int g) {
    const int c = kb * 128 + 32 * g;
#pragma unroll
    for (int q = 0; q < MT; ++q)
      raw[q].load(static_cast<const typename Act<SRC>::T*>(p.act) + (size_t)min(m0 + MT * r + q, (long long)p.rows - 1) * p.inputs + c,
                  p.inputs - c);
  }
  __device__ __forceinline__ void take(u32x4 (&v)[MT], uint32_t& scale) const {
    scale = 0;
#pragma unroll
    for (int q = 0; q < MT; ++q) scale |= (uint32_t)raw[q].quantise(v[q]) << (8 * q);
  }
};
template <int MT>
struct MxRows<KEPT, MT> {
  u32x4 codes[MT];
  uint32_t scales;
  __device__ __forceinline__ void load(const MxLinear& p, long long m0, int kb, int r, int g) {
#pragma unroll
    for (int q = 0; q < MT; ++q)
      codes[q] = *reinterpret_cast<const u32x4*>(p.x.codes + (size_t)min(m0 + MT * r + q, (long long)p.rows - 1) * p.x.pitch + kb * 64 + 16 * g);
    const uint8_t* const s = p.x.scales + (size_t)(4 * kb + g) * p.x.sp + min(m0 + MT * r, ((long long)p.rows - 1) & ~(MT - 1LL));
    scales = MT == 2 ? *reinterpret_cast<const uint16_t*>(s) : *s;
  }
  __device__ __forceinline__ void take(u32x4 (&v)[MT], uint32_t& scale) const {
#pragma unroll
    for (int q = 0; q < MT; ++q) v[q] = codes[q];
    scale = scales;
  }
};

// 16 waves of 128 registers hide memory's latency best; where those do not hold the rows, 8 of 256.
constexpr int resident_waves(int src, int steps) { return steps > 2 || (steps == 2 && src == DT_F32) ? 8 : 16; }

// STEPS: 1, 2, 4 or 8, at least p.steps.
template <int SRC, int OUT, int STEPS>
__global__ __launch_bounds__(resident_waves(SRC, STEPS) * 64) void mx4_resident_kernel(MxLinear p, MxResident q) {
  constexpr int RW = resident_waves(SRC, STEPS);
  constexpr bool EARLY = STEPS == 1 && SRC != DT_F32;
  extern __shared__ __attribute__((aligned(16))) uint8_t mx_smem[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int kbs = STEPS <= 2 ? STEPS : p.steps, sets = (p.outputs + 63) / 64;
  // blocks of the same rows and other subsets share an XCD (blocks are dealt out to 8 in turn)
  const int index = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3), subset = index % q.subsets, blk = index / q.subsets;
  if (blk >= q.blocks) return;
  const int set0 = subset * q.per, per = min(q.per, sets - set0);
  uint32_t* const ws = reinterpret_cast<uint32_t*>(mx_smem + (size_t)q.per * kbs * 4096);
  float* const bias = reinterpret_cast<float*>(ws + q.per * kbs * 64);
  for (int i = wave; i < per * kbs * 4; i += RW) {
    const int set = (i >> 2) / kbs, kb = (i >> 2) % kbs;
    const int n = min((set0 + set) * 64 + 4 * r + (i & 3), p.outputs - 1);
    const uint8_t* src = p.w.codes + (size_t)n * p.w.pitch + kb * 64 + 16 * g;
#if __HIP_DEVICE_COMPILE__
    __builtin_amdgcn_global_load_lds(src, mx_smem + i * 1024, 16, 0, 0);
#else
    (void)src;
#endif
  }
  for (int i = wave; i < per * kbs; i += RW) {     // scale rows are whole sixteens
    const int set = i / kbs, kb = i % kbs, n = min((set0 + set) * 64 + 4 * r, (p.outputs - 1) & ~3);
    ws[i * 64 + lane] = *reinterpret_cast<const uint32_t*>(p.w.scales + (size_t)(4 * kb + g) * p.w.sp + n);
  }
  for (int i = threadIdx.x; i < per * 64; i += RW * 64) bias[i] = p.bias && set0 * 64 + i < p.outputs ? p.bias[set0 * 64 + i] : 0.f;
  const long long units = ((long long)p.rows + 16 * RM - 1) / (16 * RM), stride = (long long)q.blocks * RW;
  long long u = (long long)blk * RW + wave;
  MxRows<SRC, RM> rows[EARLY ? STEPS : 1];
  if constexpr (EARLY) {
#pragma unroll
    for (int kb = 0; kb < STEPS; ++kb) rows[kb].load(p, min(u, units - 1) * 16 * RM, kb, r, g);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  for (; u < units; u += stride) {
    const long long m0 = u * 16 * RM;
    u32x4 x[STEPS][RM];
    uint32_t xs[STEPS];
    if constexpr (EARLY) {
#pragma unroll
      for (int kb = 0; kb < STEPS; ++kb) rows[kb].take(x[kb], xs[kb]);
#pragma unroll
      for (int kb = 0; kb < STEPS; ++kb) rows[kb].load(p, min(u + stride, units - 1) * 16 * RM, kb, r, g);
    } else {
#pragma unroll
      for (int kb = 0; kb < STEPS; ++kb)
        if (kb < kbs) {
          rows[0].load(p, m0, kb, r, g);
          rows[0].take(x[kb], xs[kb]);
        }
    }
    for (int set = 0; set < per; ++set) {
      f4 acc[4][RM];
      const f4 b = *reinterpret_cast<const f4*>(bias + set * 64 + 4 * r);
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int k = 0; k < RM; ++k) acc[t][k] = f4{b[t], b[t], b[t], b[t]};
#pragma unroll
      for (int kb = 0; kb < STEPS; ++kb) {
        if (kb >= kbs) break;
        const uint8_t* at = mx_smem + (size_t)(set * kbs + kb) * 4096 + lane * 16;
        u32x4 a[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) a[t] = *reinterpret_cast<const u32x4*>(at + t * 1024);
        mx_mma_set<RM>(acc, x[kb], a, xs[kb], ws[(set * kbs + kb) * 64 + lane]);
      }
      mx_finish<OUT, RM>(acc, p, m0, (set0 + set) * 64, r, g);
    }
  }
}

// ---- streamed: long reductions ---------------------------------------------------------------------

// A block of 2 by WM waves of NT by 4 tiles of 16, 256 columns a step: whole lines of memory.  Each wave copies
// sets of 64 rows of an operand to one of two LDS buffers a step ahead, its instructions 8 rows of 128 bytes: four
// neighbouring lanes read 64 bytes (lanes in the order of the fragments, 16 bytes of a row each, made the copies what
// the kernel waited for: 98 us instead of 63 for 8192 rows of 4096 x 4096, which take 68 to 72 on different cards,
// 3.8 to 4.0 PFLOP/s).  Tile t's rows lie side by side in LDS, their
// 16-byte chunks c at c ^ (row & 7): no conflicts.  Fragments of 128 columns are read half a step ahead, so that the products
// do not wait for LDS.
// Split: a block takes part of the steps and stores f32 sums to p.partial, joined by mx4_join_kernel.
struct MxStream {
  int mtiles, ntiles, parts;
};

// A pointer that every lane has, in scalar registers.
__device__ __forceinline__ const uint8_t* uniform(const uint8_t* p) {
  const uint64_t v = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
  return reinterpret_cast<const uint8_t*>((uint64_t)hi << 32 | lo);
}

template <int OUT, int NT, int WM, bool PART>
__global__ __launch_bounds__(128 * WM, 2) void mx4_stream_kernel(MxLinear p, MxStream q) {
  constexpr int BN = 2 * NT * 16, BM = WM * 64, SETS = (BN + BM) / 64, MINE = SETS / (2 * WM);
  constexpr int CODES = 64 * 128, STAGE = SETS * (CODES + 2 * 256);
  static_assert(MINE * 2 * WM == SETS && BN / 64 % MINE == 0, "a wave copies whole sets of one operand");
  // Separate objects: reads of one are then known not to wait for copies into the other.
  __shared__ __attribute__((aligned(16))) uint8_t S0[STAGE], S1[STAGE];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  int r = lane & 15, g = lane >> 4, mt, nt, part;
  {      // an XCD takes a run of blocks, parts first, then 4 tiles of rows and all outputs, so that its L2 reads little twice
    const long long tiles = (long long)q.mtiles * q.ntiles, blocks = tiles * q.parts;
    const long long id = (blockIdx.x & 7) * ((blocks + 7) / 8) + (blockIdx.x >> 3);
    if (id >= blocks) return;
    part = PART ? (int)(id / tiles) : 0;
    const int tile = (int)(PART ? id % tiles : id), turn = tile / (4 * q.ntiles), in = tile - turn * 4 * q.ntiles;
    const int tall = min(4, q.mtiles - turn * 4);
    mt = turn * 4 + in % tall;
    nt = in / tall;
  }
  const int all = p.steps / 2;             // steps of 256 columns; a last 128 come at the end
  const int s0 = (int)((long long)all * part / q.parts), s1 = (int)((long long)all * (part + 1) / q.parts);
  const long long m0 = (long long)mt * BM;
  const int n0 = nt * BN;
  // what this wave copies: MINE sets of one operand; rows past the end repeat the last one
  const bool of_w = wave * MINE < BN / 64;
  const Mx src = {of_w ? p.w.codes : p.x.codes, of_w ? p.w.scales : p.x.scales, 0, 0, of_w ? p.w.pitch : p.x.pitch,
                  of_w ? p.w.sp : p.x.sp};
  const long long first = of_w ? n0 + wave * MINE * 64 : m0 + (wave * MINE - BN / 64) * 64, last = (of_w ? p.outputs : p.rows) - 1;
  const long long base = min(first, last);
  const uint8_t* const codes = uniform(src.codes + (size_t)base * src.pitch);
  const uint8_t* const scales = uniform(src.scales);
  const uint32_t pitch = (uint32_t)src.pitch, sstep = (uint32_t)(4 * src.sp), chunk = 16 * ((lane & 7) ^ (lane >> 3));
  const int lane_row = (int)(first - base) + 4 * (lane >> 3), last_row = (int)min(last - base, (long long)INT_MAX);
  uint32_t soff[MINE];
#pragma unroll
  for (int i = 0; i < MINE; ++i) soff[i] = (uint32_t)(g * src.sp + min(first + i * 64 + 4 * r, last & ~3LL));
  auto stage = [&](uint8_t* dst, int s) __attribute__((always_inline)) {
#if __HIP_DEVICE_COMPILE__
    const __amdgpu_buffer_rsrc_t cr = __builtin_amdgcn_make_buffer_rsrc((void*)codes, 0, 0xffffffffu, 0x27000);
    const __amdgpu_buffer_rsrc_t sr = __builtin_amdgcn_make_buffer_rsrc((void*)scales, 0, 0xffffffffu, 0x27000);
#pragma unroll
    for (int l = 0; l < 10 * MINE; ++l) {
      const int i = l / 10, k = l % 10 - 2;
      if (k < 0) {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(sr, dst + SETS * CODES + (wave * MINE + i) * 512 + (k + 2) * 256, 4, soff[i],
                                                 (2 * s + k + 2) * sstep, 0, 0);
      } else {       // LDS row 8 k + lane / 8: tile k / 2, its row 8 (k % 2) + lane / 8
        const uint32_t row = (uint32_t)min(lane_row + i * 64 + 32 * (k & 1) + (k >> 1), last_row);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(cr, dst + (wave * MINE + i) * CODES + k * 1024, 16, row * pitch + chunk, s * 128, 0, 0);
      }
    }
#else
    (void)codes, (void)scales, (void)dst, (void)s, (void)soff, (void)sstep, (void)pitch, (void)chunk, (void)lane_row, (void)last_row;
#endif
  };
  const int wn = wave & 1, wm = wave >> 1;
  constexpr int H = NT / 4, UNITS = 2 * H;     // units of a step: a half of its columns times a set of outputs
  f4 acc[H][4][4];
#pragma unroll
  for (int h = 0; h < H; ++h)
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const float b = !PART && p.bias ? p.bias[min(n0 + (wn * H + h) * 64 + 4 * r + t, p.outputs - 1)] : 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[h][t][k] = f4{b, b, b, b};
    }
  u32x4 x[2][4], w[2][4];
  uint32_t sx[2], sw[2];
  const int at0 = r * 128 + ((g ^ (r & 7)) << 4), at1 = at0 ^ 64;
  auto read_set = [&](u32x4 (&v)[4], uint32_t& scale, const uint8_t* buf, int set, int half) __attribute__((always_inline)) {
    scale = *reinterpret_cast<const uint32_t*>(buf + SETS * CODES + set * 512 + half * 256 + lane * 4);
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = *reinterpret_cast<const u32x4*>(buf + set * CODES + k * 2048 + (half ? at1 : at0));
  };
  auto read = [&](const uint8_t* buf, int unit) __attribute__((always_inline)) {
    const int half = unit / H, h = unit % H;
    if (h == 0) read_set(x[half], sx[half], buf, BN / 64 + wm, half);
    read_set(w[unit & 1], sw[unit & 1], buf, wn * H + h, half);
  };
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  if (s0 < s1) {
    stage(S0, s0);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    stage(S1, min(s0 + 1, s1 - 1));
    read(S0, 0);
  }
  // Step s: its first unit is read, it is in `buf`, and step s + 1 on its way to `other`.
  auto step = [&](int s, uint8_t* buf, uint8_t* other) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      if (u + 1 < UNITS) {
        read(buf, u + 1);
      } else {
        // every wave's copies of s + 1 are there, and every wave has read s
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        read(other, 0);
        stage(buf, min(s + 2, s1 - 1));      // past the end the last step again, which nothing uses
      }
      mx_mma_set<4>(acc[u % H], x[u / H], w[u & 1], sx[u / H], sw[u & 1]);
      __builtin_amdgcn_sched_barrier(0);   // products touch no memory: they would be moved past the next barrier
    }
  };
  int s = s0;
  for (; s + 1 < s1; s += 2) {
    step(s, S0, S1);
    step(s + 1, S1, S0);
  }
  if (s < s1) step(s, S0, S1);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the last copies, which nothing reads
  asm volatile("" : "+v"(r), "+v"(g));     // or the offsets of what follows would be kept in registers throughout
  if ((p.steps & 1) && part == q.parts - 1) {         // the last 128 columns, straight from memory
    const int kb = p.steps - 1;
    const long long m = m0 + wm * 64 + 4 * r;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      x[0][k] = *reinterpret_cast<const u32x4*>(p.x.codes + (size_t)min(m + k, p.rows - 1LL) * p.x.pitch + kb * 64 + 16 * g);
    sx[0] = *reinterpret_cast<const uint32_t*>(p.x.scales + (size_t)(4 * kb + g) * p.x.sp + min(m, (p.rows - 1LL) & ~3LL));
#pragma unroll
    for (int h = 0; h < H; ++h) {
      const int n = n0 + (wn * H + h) * 64 + 4 * r;
#pragma unroll
      for (int t = 0; t < 4; ++t)
        w[0][t] = *reinterpret_cast<const u32x4*>(p.w.codes + (size_t)min(n + t, p.outputs - 1) * p.w.pitch + kb * 64 + 16 * g);
      sw[0] = *reinterpret_cast<const uint32_t*>(p.w.scales + (size_t)(4 * kb + g) * p.w.sp + min(n, (p.outputs - 1) & ~3));
      mx_mma_set<4>(acc[h], x[0], w[0], sx[0], sw[0]);
    }
  }
#pragma unroll
  for (int h = 0; h < H; ++h) {
    const int n = n0 + (wn * H + h) * 64;
    if (n >= p.outputs) continue;
    MxLinear o = p;
    if constexpr (PART) {
      o.relu = 0;
      o.residual = nullptr;
      o.out = p.partial + (size_t)part * p.rows * p.outputs;
    }
    mx_finish<OUT, 4, PART>(acc[h], o, m0 + wm * 64, n, r, g);
  }
}

// The parts' sums in a fixed order, bias, ReLU, residual: a thread sums V elements in a row, P threads share them.
template <int OUT, int P, int V>
__global__ __launch_bounds__(256) void mx4_join_kernel(MxLinear p, int parts) {
  typedef typename Act<OUT>::T T;
  typedef float fv __attribute__((ext_vector_type(V), aligned(4)));      // a part begins at any element
  constexpr int E = 256 / P;
  __shared__ float sm[P > 1 ? P : 1][P > 1 ? E * V : 1];
  const size_t count = (size_t)p.rows * p.outputs;
  const int e = threadIdx.x % E, k0 = threadIdx.x / E;
  const size_t i = ((size_t)blockIdx.x * E + e) * V;
  float v[V] = {};
  const int first = parts * k0 / P, end = parts * (k0 + 1) / P;
  if (i + V <= count) {
#pragma unroll 4
    for (int k = first; k < end; ++k) {
      const fv t = *reinterpret_cast<const fv*>(p.partial + k * count + i);
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] += t[j];
    }
  } else {
    for (int k = first; k < end; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (i + j < count) v[j] += p.partial[k * count + i + j];
  }
  if constexpr (P > 1) {
#pragma unroll
    for (int j = 0; j < V; ++j) sm[k0][j * E + e] = v[j];
    __syncthreads();
    if (k0 > 0) return;
#pragma unroll
    for (int k = 1; k < P; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] += sm[k][j * E + e];
  }
#pragma unroll
  for (int j = 0; j < V; ++j) {
    if (i + j >= count) return;
    float s = v[j];
    if (p.bias) s += p.bias[(i + j) % p.outputs];
    if (p.relu) s = __builtin_elementwise_maximum(s, 0.f);
    if (p.residual) s += Act<OUT>::ld(static_cast<const T*>(p.residual) + i + j);
    Act<OUT>::st(static_cast<T*>(p.out) + i + j, s);
  }
}

// ---- few rows or outputs -----------------------------------------------------------------------------

// What counts is the time to the last byte: a block computes 16 MT rows by 16 outputs, its waves steps of the columns in
// turn, two at a time, operands straight from memory, sums joined in LDS.  One row of 4096 x 4096: 5.7 us, 1.6 TB/s of
// weights; a launch and one trip to memory are most of it.
constexpr int few_waves(int src, int mt) { return src == DT_F32 && mt == 2 ? 8 : 16; }    // registers

template <int SRC, int OUT, int MT>
__global__ __launch_bounds__(few_waves(SRC, MT) * 64) void mx4_few_kernel(MxLinear p) {
  constexpr int FW = few_waves(SRC, MT);
  __shared__ f4 part[FW][MT][64];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int waves = blockDim.x >> 6, n0 = blockIdx.x * 16;
  const long long m0 = (long long)blockIdx.y * 16 * MT;
  const int n = min(n0 + r, p.outputs - 1);
  const uint8_t* const wrow = p.w.codes + (size_t)n * p.w.pitch + 16 * g;
  const uint8_t* const wscale = p.w.scales + (size_t)g * p.w.sp + n;
  f4 acc[MT];
#pragma unroll
  for (int q = 0; q < MT; ++q) acc[q] = f4{0.f, 0.f, 0.f, 0.f};
  struct Step {
    u32x4 w;
    uint32_t ws;
    MxRows<SRC, MT> x;
  };
  auto load = [&](Step& s, int kb) __attribute__((always_inline)) {
    s.w = *reinterpret_cast<const u32x4*>(wrow + (size_t)kb * 64);
    s.ws = wscale[(size_t)4 * kb * p.w.sp];
    s.x.load(p, m0, kb, r, g);
  };
  auto multiply = [&](const Step& s) __attribute__((always_inline)) {
    u32x4 x[MT];
    uint32_t sx;
    s.x.take(x, sx);
    acc[0] = mx_mma<0, 0>(x[0], s.w, acc[0], sx, s.ws);
    if constexpr (MT == 2) acc[1] = mx_mma<1, 0>(x[1], s.w, acc[1], sx, s.ws);
  };
  for (int kb = wave; kb < p.steps; kb += 2 * waves) {
    Step a, b;
    load(a, kb);
    load(b, min(kb + waves, p.steps - 1));
    multiply(a);
    if (kb + waves < p.steps) multiply(b);
  }
#pragma unroll
  for (int q = 0; q < MT; ++q) part[wave][q][lane] = acc[q];
  __syncthreads();
  typedef typename Act<OUT>::T T;
  // thread: output n0 + e % 16 of row MT i + q, i = 4 (lane / 16) + j of the lane that holds it
  for (int e = threadIdx.x; e < MT * 256; e += blockDim.x) {
    const int row = e >> 4, q = row % MT, i = row / MT, o = n0 + (e & 15);
    const float* const at = reinterpret_cast<const float*>(&part[0][q][(i >> 2) * 16 + (e & 15)]) + (i & 3);
    float v = at[0];
    for (int k = 1; k < waves; ++k) v += at[k * MT * 256];
    const long long m = m0 + row;
    if (m >= p.rows || o >= p.outputs) continue;
    if (p.bias) v += p.bias[o];
    if (p.relu) v = __builtin_elementwise_maximum(v, 0.f);
    const size_t to = (size_t)m * p.outputs + o;
    if (p.residual) v += Act<OUT>::ld(static_cast<const T*>(p.residual) + to);
    Act<OUT>::st(static_cast<T*>(p.out) + to, v);
  }
}

// ---- which kernel ------------------------------------------------------------------------------------

enum { FEW, RESIDENT, STREAM };
struct MxPlan {
  int kind;
  bool wide;                 // STREAM: 256 x 256 tiles, else 128 x 128
  int parts;
};
constexpr int CUS = 256;

constexpr int set_bytes(int steps) { return steps * (4096 + 256) + 256; }

MxPlan mx_plan(long long rows, int steps, long long outputs) {
  // Few: in runs of 32 rows by 16 outputs the times cross at 2300 for one step (128 x 512 in bf16: 1500 runs 8.1 us and 10.5
  // resident, 3000 12.6 and 11.0), near 1100 for more (512 x 128: 700 9.2 and 12.2, 1500 16.6 and 12.3; 1024 x 256: 700 15
  // and 22, 1500 28 and 22), and near 400 for streamed ones (1024 x 1024: 300 6.9 and 8.5, 700 15 and 8.7; 4096 x 4096: 300
  // 11.5 and 12.5, 700 22 and 13.5).  Past 8192 columns the parts of a streamed product share them.
  const bool resident = steps <= 4 || (steps <= 8 && (outputs + 63) / 64 * set_bytes(steps) <= LDS_BYTES);
  const long long few = (rows + 31) / 32 * ((outputs + 15) / 16);
  if (few <= (steps == 1 ? 2300 : resident ? 1100 : 400) && steps <= 64) return {FEW, false, 1};
  if (resident) return {RESIDENT, false, 1};
  const long long wide = (rows + 255) / 256 * ((outputs + 255) / 256);
  if (wide >= 128) return {STREAM, true, 1};
  // P parts take 0.34 / P us a step of 128 columns and 0.044 P us a tile for their sums' way through memory, so that
  // sqrt(8 steps / tiles) is best: 128 x 128 outputs of 147456 columns take 359 us in one part, 23 in 16, 13 in 64, 14 in
  // 128; 256 x 512 of them 388, 34, 26, 37; 480 x 1024 of 24576 columns 67 in one, 25 in 4, 23 in 8, 24 in 16.  A part has
  // 1024 columns at least.
  const long long tiles = (rows + 127) / 128 * ((outputs + 127) / 128);
  int parts = 1;
  while (parts < 64 && parts < steps / 8 && (parts + 1LL) * (parts + 1) * tiles <= 8LL * steps) ++parts;
  return {STREAM, false, parts};
}

size_t up256(size_t n) { return (n + 255) & ~size_t(255); }

template <int OUT, int NT, int WM, bool PART>
void go_stream(lf_context* ctx, const MxLinear& p, int parts) {
  constexpr int BM = WM * 64, BN = 2 * NT * 16;
  MxStream q{(int)(((long long)p.rows + BM - 1) / BM), (p.outputs + BN - 1) / BN, parts};
  const long long blocks = ((long long)q.mtiles * q.ntiles * parts + 7) / 8 * 8;
  hipLaunchKernelGGL((mx4_stream_kernel<OUT, NT, WM, PART>), dim3((unsigned)blocks), dim3(128 * WM), 0, ctx->stream, p, q);
}

template <int OUT, int P>
void go_join(lf_context* ctx, const MxLinear& p, int parts) {
  constexpr int V = 4;
  const size_t count = (size_t)p.rows * p.outputs, each = 256 / P * V;
  hipLaunchKernelGGL((mx4_join_kernel<OUT, P, V>), dim3((unsigned)((count + each - 1) / each)), dim3(256), 0, ctx->stream, p, parts);
}

template <int SRC, int OUT, int STEPS>
int go_resident(lf_context* ctx, const MxLinear& p) {
  constexpr int RW = resident_waves(SRC, STEPS);
  const int sets = (p.outputs + 63) / 64, each = set_bytes(p.steps);
  const long long units = ((long long)p.rows + 16 * RM - 1) / (16 * RM);
  MxResident q;
  // as many sets a block as fit, but no more than keep every wave of the chip busy
  const long long busy = std::max<long long>(1, units * sets / (CUS * RW));
  q.per = (int)std::min<long long>(std::min(LDS_BYTES / each, sets), busy);
  q.subsets = (sets + q.per - 1) / q.per;
  q.blocks = (int)std::min<long long>((units + 3) / 4, std::max(1, CUS / q.subsets));
  static const hipError_t lds = hipFuncSetAttribute(reinterpret_cast<const void*>(&mx4_resident_kernel<SRC, OUT, STEPS>),
                                                    hipFuncAttributeMaxDynamicSharedMemorySize, LDS_BYTES);
  LF_TRY(check_hip(lds, "4-bit product LDS"));
  const unsigned grid = (unsigned)((q.blocks * q.subsets + 7) / 8 * 8);
  hipLaunchKernelGGL((mx4_resident_kernel<SRC, OUT, STEPS>), dim3(grid), dim3(RW * 64), (size_t)q.per * each, ctx->stream, p, q);
  return LF_OK;
}

template <int SRC, int OUT>
int go_small(lf_context* ctx, const MxLinear& p, const MxPlan& plan) {
  if (plan.kind == RESIDENT) {
    if (p.steps == 1) return go_resident<SRC, OUT, 1>(ctx, p);
    if (p.steps == 2) return go_resident<SRC, OUT, 2>(ctx, p);
    if (p.steps <= 4) return go_resident<SRC, OUT, 4>(ctx, p);
    return go_resident<SRC, OUT, 8>(ctx, p);
  }
  if (p.rows <= 16)
    hipLaunchKernelGGL((mx4_few_kernel<SRC, OUT, 1>), dim3((p.outputs + 15) / 16), dim3(std::min(p.steps, few_waves(SRC, 1)) * 64), 0,
                       ctx->stream, p);
  else
    hipLaunchKernelGGL((mx4_few_kernel<SRC, OUT, 2>), dim3((p.outputs + 15) / 16, (p.rows + 31) / 32),
                       dim3(std::min(p.steps, few_waves(SRC, 2)) * 64), 0, ctx->stream, p);
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
    if (plan.wide) go_stream<OUT, 8, 4, false>(ctx, p, 1);
    else if (plan.parts == 1) go_stream<OUT, 4, 2, false>(ctx, p, 1);
    else go_stream<DT_F32, 4, 2, true>(ctx, p, plan.parts);
    LF_TRY(check_hip(hipGetLastError(), "4-bit product launch"));
  }
  if (plan.parts == 1) return LF_OK;
  LaunchScope ls(ctx, "mx4.join");
  if (plan.parts > 16) go_join<OUT, 16>(ctx, p, plan.parts);
  else if (plan.parts > 4) go_join<OUT, 4>(ctx, p, plan.parts);
  else go_join<OUT, 1>(ctx, p, plan.parts);
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
