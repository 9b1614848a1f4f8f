// Weight gradients of 8-bit operands: out[i][j] = sum_m a[m][i] b[m][j], a and b checkpoints of the same
// rows, and the column sums of one of them (the bias gradient).
//
// The reduction runs over the rows, along which each value has a scale of its own, so the codes are turned
// into bf16 (exactly) as they are staged into LDS, and the fragments, whose lanes need 8 rows of a column,
// are read from there by transposing reads.  A block of three teams of four waves computes a tile of
// 128 x 128 outputs over its share of the rows, the teams on steps of 32 rows in turn, joined in LDS; the
// blocks' partial sums are added in order by a second kernel.  Column sums are a product with ones.
//
// 196608 rows, 1024 x 256: 126 to 154 us from card to card (670 to 820 TFLOP/s; its bytes alone are 49 us); 147456 rows,
// 512 x 128 and 128 x 512 in one launch: 56 us.  Nothing is full: matrix pipes, LDS and issue are each busy about 40 % of
// the time, and overlap only as far as waves differ.  12 waves that load three steps ahead beat 16 of 128
// registers that load two ahead: in turn on one card, medians with the join, 131 us and 137, 147456 rows of 512 x 128
// 36.5 us and 38.1, 90601 rows of 128 x 128 22.3 us and 22.9.  Before those, 8 waves took 140 us and 78 us in two
// launches, and forms that fetch fragments a step ahead 149 to 164 us and 63 us.  Codes in LDS, converted after the
// read, halve its traffic but double the conversions: 166 us.
#include <algorithm>

#include "lf_train.h"

namespace lf {

typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef short s4v __attribute__((ext_vector_type(4)));

constexpr int GN = GROUP;                 // outputs of a block, either way: one group of both operands
constexpr int GSTEP = 32;                 // rows of a step: one matrix instruction's
constexpr int TEAMS = 3;                  // of four waves, on steps in turn
constexpr int GWAVES = 4 * TEAMS;

struct GradParams {
  Kept a, b;
  float* partial;                         // [splits][a.cols][b.cols]; null: one split, straight to out
  float* colsum;                          // [splits][cols of the summed one], or null
  int sum_of;                             // 0: no column sums, 1: of a, 2: of b
  int splits, tiles, tiles_j, per_xcd;
  long long rows_per;                     // rows of a split, a multiple of TEAMS GSTEP
  void *out, *bias;
  int dt, swapped;                        // out is [b.cols][a.cols]
};

// Products of the same rows that share a launch, blocks dealt out in order.
struct GradBatch {
  GradParams w[2];
  unsigned first[2];                      // of the products' blocks
  unsigned join[2];                       // of the blocks that join them
};

constexpr int PITCH = GN * 2 + 32;        // LDS bytes of a row of bf16: 4 rows apart by 32 bytes mod 128
constexpr int BUF = 2 * GSTEP * PITCH;    // one team's buffer: rows of a, then of b
constexpr size_t GRAD_SMEM = TEAMS * 2 * BUF;
static_assert(GRAD_SMEM >= 18 * 256 * 16 && GRAD_SMEM <= 160 * 1024, "the join of two teams at a time; LDS");

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
__device__ __forceinline__ b8 tr_frag(const uint8_t* p) {
  uint32_t w[4], h[2];
  tr_read(h, p);
  w[0] = h[0];
  w[1] = h[1];
  tr_read(h, p + 16 * PITCH);
  w[2] = h[0];
  w[3] = h[1];
  b8 o;
  __builtin_memcpy(&o, w, 16);
  return o;
}

template <bool SUMS>
__global__ __launch_bounds__(GWAVES * 64) void weight_grad_kernel(GradBatch batch) {
  extern __shared__ __attribute__((aligned(16))) uint8_t grad_smem[];
  const int op = blockIdx.x >= batch.first[1] ? 1 : 0;
  const GradParams& p = batch.w[op];
  const unsigned block = blockIdx.x - batch.first[op];
  // tiles of the same rows share an XCD (blocks are dealt out to 8 in turn, and products begin at multiples of 8)
  const int index = (block & 7) * p.per_xcd + (block >> 3), tile = index % p.tiles, split = index / p.tiles;
  if (split >= p.splits) return;
  const int i0 = tile / p.tiles_j * GN, j0 = tile % p.tiles_j * GN;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int team = wave >> 2, wi = (wave >> 1) & 1, wj = wave & 1, tid = threadIdx.x & 255;
  const long long m0 = split * p.rows_per;
  const int n = (int)min(p.a.rows - m0, p.rows_per);            // rows of the split
  const int steps = (n + TEAMS * GSTEP - 1) / (TEAMS * GSTEP);
  uint8_t* const mine = grad_smem + team * 2 * BUF;

  // A step is 16 codes a lane of a and of b, at a uniform base that moves with the step and a 32-bit lane
  // offset.  The loads have no condition, or the compiler could not count those in flight: rows past the
  // end read the last one, and are made zeros when they are stored; columns past the pitch read the last
  // ones, for outputs that do not exist.
  const int row = tid >> 3, pc = tid & 7;
  const uint8_t* const code[2] = {p.a.codes + (size_t)m0 * p.a.pitch, p.b.codes + (size_t)m0 * p.b.pitch};
  const uint8_t* const scale[2] = {p.a.scales + (size_t)(i0 / GROUP) * p.a.sp + m0, p.b.scales + (size_t)(j0 / GROUP) * p.b.sp + m0};
  const int pitch[2] = {p.a.pitch, p.b.pitch};
  const int col[2] = {min(i0 + pc * 16, pitch[0] - 16), min(j0 + pc * 16, pitch[1] - 16)};
  u32x4 raw[2][2];        // [step][a, b]
  int sc[2][2];
  // 24-bit products: the 64-bit multiply-add that the compiler would take reads a register pair whose other
  // half may be a load in flight, and waits for it
  auto load = [&](int s, int ring, int k) __attribute__((always_inline)) {
    const int m = (int)min(((uint32_t)s * TEAMS + team) * GSTEP, (uint32_t)n - 1), r = min(row, n - 1 - m);
    raw[ring][k] = *reinterpret_cast<const u32x4*>(code[k] + (size_t)m * pitch[k] + (__umul24(r, pitch[k]) + col[k]));
    sc[ring][k] = (scale[k] + m)[(uint32_t)r];
  };
  // A lane's 16 values are two 16-byte pieces; in the upper half of a row they lie the other way round, so
  // that the 8 lanes of a row store to all banks at once.
  const int dst = row * PITCH + pc * 32 + (pc & 4 ? 16 : 0);
  auto store = [&](int s, int ring, int k) __attribute__((always_inline)) {
    const bool ok = row < (int)(n - ((uint32_t)s * TEAMS + team) * GSTEP);
    const float f = scale_value(sc[ring][k]);
    uint32_t w[8];
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      const int c = ok ? (int)raw[ring][k][d] : 0;
      w[2 * d] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, f, false));
      w[2 * d + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, f, true));
    }
    uint8_t* const to = mine + (s & 1) * BUF + k * GSTEP * PITCH;
    *reinterpret_cast<u32x4*>(to + dst) = u32x4{w[0], w[1], w[2], w[3]};
    *reinterpret_cast<u32x4*>(to + (dst ^ 16)) = u32x4{w[4], w[5], w[6], w[7]};
  };

  // A wave has a 64 x 64 part of the tile.  Its fragments are numbered so that fragments 0 and 2 of the two
  // waves that share them are different ones: each sums those.
  f4 acc[4][4], sums[2];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = f4{0.f, 0.f, 0.f, 0.f};
  sums[0] = sums[1] = f4{0.f, 0.f, 0.f, 0.f};
  const int of = SUMS ? p.sum_of : 0;
  const bool sum_a = of == 1 && j0 == 0, sum_b = of == 2 && i0 == 0;     // blocks at the other operand's first tile
  b8 ones;
#pragma unroll
  for (int k = 0; k < 8; ++k) ones[k] = (__bf16)1.0f;
  const int xi = of == 1 ? wj : 0, xj = of == 2 ? wi : 0;
  const int g = lane >> 4, l16 = lane & 15;
  const uint8_t* const from = mine + (4 * g + (l16 >> 2)) * PITCH;
  const uint8_t* const from_a = from + wi * 128 + ((l16 & 3) * 8 ^ wi * 16) + xi * 32;
  const uint8_t* const from_b = from + GSTEP * PITCH + wj * 128 + ((l16 & 3) * 8 ^ wj * 16) + xj * 32;
  const int odd_a = (1 - 2 * xi) * 32, odd_b = (1 - 2 * xj) * 32;

  // Step s is multiplied while step s + 1 is converted and stored; steps s + 2 and s + 3 are under way.
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    load(0, 0, k);
    load(1, 1, k);
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    store(0, 0, k);
    load(2, 0, k);
  }
  for (int s0 = 0; s0 < steps; s0 += 2) {     // past the last step: zeros
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      __syncthreads();
      const int at = u * BUF;
      b8 fa[4], fb[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) fb[j] = tr_frag(from_b + (j & 1 ? at + (j - 1) * 32 + odd_b : at + j * 32));
#pragma unroll
      for (int i = 0; i < 4; ++i) fa[i] = tr_frag(from_a + (i & 1 ? at + (i - 1) * 32 + odd_a : at + i * 32));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa[i], fb[j], acc[i][j], 0, 0, 0);
        if (i & 1) {
          store(s0 + u + 1, 1 - u, i >> 1);
          load(s0 + u + 3, 1 - u, i >> 1);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      if constexpr (SUMS) {
        if (sum_a) {
#pragma unroll
          for (int f = 0; f < 2; ++f) sums[f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa[2 * f], ones, sums[f], 0, 0, 0);
        } else if (sum_b) {
#pragma unroll
          for (int f = 0; f < 2; ++f) sums[f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, fb[2 * f], sums[f], 0, 0, 0);
        }
      }
    }
  }

  // the other teams' sums are added to the first's, in order
  f4* const join = reinterpret_cast<f4*>(grad_smem) + (wi * 2 + wj) * 64 + lane;   // [18][4 waves][64]
#pragma unroll 1
  for (int t = 1; t < TEAMS; ++t) {
    __syncthreads();
    if (team == t) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) join[(i * 4 + j) * 256] = acc[i][j];
      join[16 * 256] = sums[0];
      join[17 * 256] = sums[1];
    }
    __syncthreads();
    if (team == 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] += join[(i * 4 + j) * 256];
      sums[0] += join[16 * 256];
      sums[1] += join[17 * 256];
    }
  }
  if (team != 0) return;
  const int ca = p.a.cols, cb = p.b.cols;
  float* part = p.partial ? p.partial + (size_t)split * ca * cb : nullptr;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int ci = i0 + wi * 64 + (i ^ xi) * 16 + 4 * g, cj = j0 + wj * 64 + (j ^ xj) * 16 + l16;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (ci + k < ca && cj < cb) {
          if (part) part[(size_t)(ci + k) * cb + cj] = acc[i][j][k];
          else store_act(p.out, p.dt, p.swapped ? (size_t)cj * ca + ci + k : (size_t)(ci + k) * cb + cj, acc[i][j][k]);
        }
    }
  if (!sum_a && !sum_b) return;
  // of a: lane group g has columns 4g .. 4g + 3 of a fragment, in every lane; of b: lane l16 column l16
  const int cn = sum_a ? ca : cb;
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int c = sum_a ? i0 + wi * 64 + (2 * h + xi) * 16 + 4 * g + k : j0 + wj * 64 + (2 * h + xj) * 16 + l16;
      if ((sum_a ? l16 == 0 : g == 0 && k == 0) && c < cn) {
        if (part) p.colsum[(size_t)split * cn + c] = sums[h][k];
        else store_act(p.bias, p.dt, c, sums[h][k]);
      }
    }
}

// Partial sums added in order: 64 outputs a block, 16 runs of the splits at a time.
__global__ __launch_bounds__(256) void weight_grad_join_kernel(GradBatch batch) {
  const int op = blockIdx.x >= batch.join[1] ? 1 : 0;
  const GradParams& p = batch.w[op];
  const unsigned block = blockIdx.x - batch.join[op];
  const long long n = (long long)p.a.cols * p.b.cols;
  const int cn = p.sum_of == 1 ? p.a.cols : p.b.cols;     // blocks for it are there only if it is summed
  __shared__ f4 sm[16][16];
  const int c = threadIdx.x & 15, run = threadIdx.x >> 4;
  const long long blocks_n = (n + 63) / 64;
  const bool main = block < blocks_n;
  const long long len = main ? n : cn, i = ((long long)block - (main ? 0 : blocks_n)) * 64 + c * 4;
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
  int tiles, tiles_j, splits;
  long long rows_per;
};
int tiles_of(int n, int k) { return (n + GN - 1) / GN * ((k + GN - 1) / GN); }
// How many ways the rows are split: the blocks' turns, at 0.95 us a step of the three teams, steps in twos, against the
// partial sums, 64 KB a block written and read, and the join's launch (5 us).
GradPlan grad_plan(long long rows, int ci, int cj, int all_tiles) {
  GradPlan q{};
  q.tiles_j = (cj + GN - 1) / GN;
  q.tiles = tiles_of(ci, cj);
  const long long turns = (rows + TEAMS * GSTEP - 1) / (TEAMS * GSTEP);
  double least = 1e300;
  for (int w = 1; w <= 256 && w <= turns; ++w) {
    const long long per = (turns + w - 1) / w, blocks = (long long)all_tiles * w;
    const double cost = 0.95 * ((per + 1) & ~1ll) * ((blocks + 255) / 256) + (w > 1 ? 5 + 0.033 * blocks : 0);
    if (cost < least) {
      least = cost;
      q.rows_per = per * (TEAMS * GSTEP);
    }
  }
  q.splits = (int)((rows + q.rows_per - 1) / q.rows_per);
  return q;
}

template <bool SUMS>
int go(lf_context* ctx, const GradBatch& b, unsigned grid) {
  static const bool lds = hipFuncSetAttribute(reinterpret_cast<const void*>(&weight_grad_kernel<SUMS>),
                                              hipFuncAttributeMaxDynamicSharedMemorySize, (int)GRAD_SMEM) == hipSuccess;
  if (!lds) return set_error(LF_ERR_DEVICE, "weight gradient: the device refuses the LDS it needs");
  hipLaunchKernelGGL((weight_grad_kernel<SUMS>), dim3(grid), dim3(GWAVES * 64), GRAD_SMEM, ctx->stream, b);
  return check_hip(hipGetLastError(), "weight gradient launch");
}

size_t up16(size_t n) { return (n + 15) & ~size_t(15); }

size_t partial_bytes(int splits, int outputs, int inputs) {
  return up16((size_t)splits * outputs * inputs * sizeof(float)) + up16((size_t)splits * std::max(outputs, inputs) * sizeof(float));
}

}  // namespace

size_t weight_grad_partials(int rows, int outputs, int inputs, int products) {
  const int splits =
      grad_plan(rows, std::max(outputs, inputs), std::min(outputs, inputs), products * tiles_of(outputs, inputs)).splits;
  return splits == 1 ? 0 : products * partial_bytes(splits, outputs, inputs);
}
size_t weight_grad_scratch(int rows, int outputs, int inputs) {
  return std::max(weight_grad_partials(rows, outputs, inputs), partial_bytes(1, outputs, inputs));
}

int run_weight_grads(lf_context* ctx, const WeightGrad* w, int count, int dt, void* scratch, const char* label) {
  GradBatch batch{};
  int all = 0;
  for (int k = 0; k < count; ++k) all += tiles_of(w[k].a.cols, w[k].b.cols);
  unsigned grid = 0, joins = 0;
  bool sums = false;
  char* at = static_cast<char*>(scratch);
  for (int k = 0; k < 2; ++k) {
    batch.first[k] = grid;
    batch.join[k] = joins;
    if (k >= count) break;
    GradParams& p = batch.w[k];
    p.swapped = w[k].a.cols < w[k].b.cols;
    p.a = p.swapped ? w[k].b : w[k].a;
    p.b = p.swapped ? w[k].a : w[k].b;
    const GradPlan q = grad_plan(p.a.rows, p.a.cols, p.b.cols, all);
    p.sum_of = !w[k].bias ? 0 : w[k].bias_of_b == (p.swapped != 0) ? 1 : 2;
    p.splits = q.splits;
    p.tiles = q.tiles;
    p.tiles_j = q.tiles_j;
    p.rows_per = q.rows_per;
    p.out = w[k].out;
    p.bias = w[k].bias;
    p.dt = dt;
    sums = sums || p.sum_of != 0;
    p.per_xcd = (q.splits * q.tiles + 7) / 8;
    grid += 8u * p.per_xcd;
    if (q.splits == 1) continue;
    const size_t n = (size_t)p.a.cols * p.b.cols;
    const int cn = p.sum_of == 0 ? 0 : p.sum_of == 1 ? p.a.cols : p.b.cols;
    p.partial = reinterpret_cast<float*>(at);
    at += up16(q.splits * n * sizeof(float));
    p.colsum = reinterpret_cast<float*>(at);
    at += up16((size_t)q.splits * cn * sizeof(float));
    joins += (unsigned)((n + 63) / 64 + (cn + 63) / 64);
  }
  if (count == 1) batch.first[1] = batch.join[1] = ~0u;
  {
    LaunchScope ls(ctx, label);
    LF_TRY(sums ? go<true>(ctx, batch, grid) : go<false>(ctx, batch, grid));
  }
  if (joins == 0) return LF_OK;
  LaunchScope ls(ctx, "fp8.weight_grad_join");
  hipLaunchKernelGGL(weight_grad_join_kernel, dim3(joins), dim3(256), 0, ctx->stream, batch);
  return check_hip(hipGetLastError(), "weight gradient join launch");
}

}  // namespace lf
