// A learned row per relative position added to every pair, and its gradient (lf_relative_position,
// lf_relative_position_backward).  Bound by memory: one addition a value.
#include <algorithm>

#include "lf_step.h"

namespace lf {

// Number of the nb ascending boundaries that are at most d.  64 bits: differences of positions need 33.
__device__ __forceinline__ int bucket_of(long long d, const int* boundaries, int nb) {
  int lo = 0, hi = nb;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (boundaries[mid] <= d) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

// The table's row of a pair, -1 for padding.
__device__ __forceinline__ int row_of(const lf_relative_pairs& p, int qp, int qs, int key, const int* boundaries) {
  if (p.key_segments) {
    const int ks = p.key_segments[key];
    if (qs < 0 || ks < 0) return -1;
    if (qs != ks) return p.boundary_count + 1;
  }
  return bucket_of((long long)qp - p.key_positions[key], boundaries, p.boundary_count);
}

// A block adds rows to `tile` (at most 256) keys of one query: the rows' numbers once a pair, in LDS, then 8
// channels a lane.
template <int ACT, int TAB>
__global__ __launch_bounds__(256) void position_kernel(lf_relative_pairs p, int channels, const typename Act<TAB>::T* table,
                                                       const float* bias, const typename Act<ACT>::T* act,
                                                       typename Act<ACT>::T* out, int tile, int tiles,
                                                       long long blocks) {
  __shared__ int rows[256];
  extern __shared__ int boundaries[];
  for (int i = threadIdx.x; i < p.boundary_count; i += 256) boundaries[i] = p.boundaries[i];
  const int chunks = (channels + 7) / 8;
  for (long long b = blockIdx.x; b < blocks; b += gridDim.x) {
    const int query = (int)(b / tiles), k0 = (int)(b % tiles) * tile, keys = min(tile, p.keys - k0);
    __syncthreads();
    if ((int)threadIdx.x < keys)
      rows[threadIdx.x] = row_of(p, p.query_positions[query], p.query_segments ? p.query_segments[query] : 0,
                                 k0 + threadIdx.x, boundaries);
    __syncthreads();
    const size_t first = ((size_t)query * p.keys + k0) * channels;
    for (int i = threadIdx.x; i < keys * chunks; i += 256) {
      const int key = i / chunks, c = (i - key * chunks) * 8, n = channels - c;
      const int row = rows[key];
      const size_t at = first + (size_t)key * channels + c;
      float v[8] = {};
      if (row >= 0) {
        load8<TAB>(table + (size_t)row * channels + c, n, v);
        if (bias) {
          float d[8];
          load8<DT_F32>(bias + c, n, d);
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k] += d[k];
        }
      }
      if (act) {
        float d[8];
        load8<ACT>(act + at, n, d);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = d[k] + v[k];
      }
      store8<ACT>(out + at, n, v);
    }
  }
}

// ---- gradient ----------------------------------------------------------------------------------

// A lane sums two channels of the keys that its team of L lanes takes, in registers while the table's row stays
// the same (most pairs are beyond the last boundary, where it does) and into the team's own rows in LDS when it
// changes: no two lanes share an address, so the order of the sums is fixed.
struct PositionGrid {
  int chunks;               // units of 64 keys of a query
  long long units;
  int blocks, slices;       // blocks of a slice of 2 L channels
  int row0, rows;           // the table's rows that this launch sums
  int all;                  // rows of the table
};

template <int ACT, int L, bool EVEN>
__global__ __launch_bounds__(256) void position_grad_kernel(lf_relative_pairs p, int channels, const typename Act<ACT>::T* grad,
                                                            float* partial, PositionGrid q) {
  typedef typename Act<ACT>::T T;
  constexpr int TEAMS = 64 / L, WIDE = 2 * L, BATCH = 16;
  extern __shared__ float sums[];
  const int waves = blockDim.x >> 6, wave = threadIdx.x >> 6, lane = threadIdx.x & 63, team = lane / L, tl = lane % L;
  const int slice = blockIdx.x / q.blocks, blk = blockIdx.x % q.blocks;
  const int c = slice * WIDE + 2 * tl;
  const int copies = waves * TEAMS;
  int* const boundaries = reinterpret_cast<int*>(sums + (size_t)copies * q.rows * WIDE);
  for (int i = threadIdx.x; i < p.boundary_count; i += blockDim.x) boundaries[i] = p.boundaries[i];
  for (int i = threadIdx.x; i < copies * q.rows * WIDE; i += blockDim.x) sums[i] = 0.f;
  __syncthreads();
  float* const mine = sums + (size_t)(wave * TEAMS + team) * q.rows * WIDE + 2 * tl;
  const int c0 = min(c, channels - (EVEN ? 2 : 1)), c1 = min(c + 1, channels - 1);
  const long long w = (long long)blk * waves + wave, all = (long long)q.blocks * waves;
  const long long u1 = q.units * (w + 1) / all;
  int cur = -1;
  float a0 = 0.f, a1 = 0.f;
  for (long long u = q.units * w / all; u < u1; ++u) {
    const int query = (int)(u / q.chunks), k0 = (int)(u % q.chunks) * 64, left = min(64, p.keys - k0);
    int row = -1;
    if (lane < left) {
      row = row_of(p, p.query_positions[query], p.query_segments ? p.query_segments[query] : 0, k0 + lane, boundaries) - q.row0;
      if (row < 0 || row >= q.rows) row = -1;
    }
    const T* const g = grad + ((size_t)query * p.keys + k0) * channels;
    for (int s0 = 0; s0 < L; s0 += BATCH) {
      if (s0 * TEAMS >= left) break;
      float v0[BATCH], v1[BATCH];
#pragma unroll
      for (int s = 0; s < BATCH; ++s) {
        const int key = min((s0 + s) * TEAMS + team, left - 1);
        const T* const at = g + (size_t)key * channels;
        if constexpr (EVEN) {
          T both[2];
          __builtin_memcpy(both, at + c0, sizeof(both));
          v0[s] = Act<ACT>::ld(both);
          v1[s] = Act<ACT>::ld(both + 1);
        } else {
          v0[s] = Act<ACT>::ld(at + c0);
          v1[s] = Act<ACT>::ld(at + c1);
        }
      }
#pragma unroll
      for (int s = 0; s < BATCH; ++s) {
        if (s0 + s >= L) break;
        const int r = __shfl(row, (s0 + s) * TEAMS + team);    // -1 past the last key
        if (r != cur) {
          if (cur >= 0) {
            mine[cur * WIDE] += a0;
            mine[cur * WIDE + 1] += a1;
          }
          cur = r;
          a0 = a1 = 0.f;
        }
        a0 += v0[s];
        a1 += v1[s];
      }
    }
  }
  if (cur >= 0) {
    mine[cur * WIDE] += a0;
    mine[cur * WIDE + 1] += a1;
  }
  __syncthreads();
  // the block's rows [all + 1][channels], the last one the sum of them all (over the launches of a table)
  float* const dst = partial + (size_t)blk * (q.all + 1) * channels;
  const int cn = min(WIDE, channels - slice * WIDE);
  for (int i = threadIdx.x; i < q.rows * WIDE; i += blockDim.x) {
    float t = 0.f;
    for (int k = 0; k < copies; ++k) t += sums[(size_t)k * q.rows * WIDE + i];
    sums[i] = t;      // this thread alone reads and writes the first copy's i
    if (i % WIDE < cn) dst[(size_t)(q.row0 + i / WIDE) * channels + slice * WIDE + i % WIDE] = t;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < cn; i += blockDim.x) {
    float t = 0.f;
    for (int r = 0; r < q.rows; ++r) t += sums[r * WIDE + i];
    float* const total = dst + (size_t)q.all * channels + slice * WIDE + i;
    *total = q.row0 ? *total + t : t;
  }
}

// out[e] = sum over p of partial[p][e]: 16 sums a block, 16 parts of each, joined in order; elements from `split`
// on go to out2.
template <int DT>
__global__ __launch_bounds__(256) void join_kernel(const float* partial, int count, long long width, long long split, void* out,
                                                   void* out2) {
  __shared__ double sm[16][16];
  const int part = threadIdx.x >> 4, lane = threadIdx.x & 15;
  const long long e = (long long)blockIdx.x * 16 + lane;
  double t = 0;
  if (e < width) {
    const int p1 = (int)((long long)count * (part + 1) / 16);
#pragma unroll 4
    for (int i = (int)((long long)count * part / 16); i < p1; ++i) t += partial[(size_t)i * width + e];
  }
  sm[part][lane] = t;
  __syncthreads();
  if (part == 0 && e < width) {
#pragma unroll
    for (int i = 1; i < 16; ++i) t += sm[i][lane];
    typedef typename Act<DT>::T T;
    if (e < split) Act<DT>::st(static_cast<T*>(out) + e, (float)t);
    else if (out2) Act<DT>::st(static_cast<T*>(out2) + (e - split), (float)t);
  }
}

int run_join(lf_context* ctx, const float* partial, int count, long long width, long long split, void* out, void* out2, int dt,
             const char* label) {
  LaunchScope ls(ctx, label);
  const dim3 grid((unsigned)((width + 15) / 16)), block(256);
  if (dt == LF_F32) hipLaunchKernelGGL((join_kernel<DT_F32>), grid, block, 0, ctx->stream, partial, count, width, split, out, out2);
  else if (dt == LF_F16) hipLaunchKernelGGL((join_kernel<DT_F16>), grid, block, 0, ctx->stream, partial, count, width, split, out, out2);
  else hipLaunchKernelGGL((join_kernel<DT_BF16>), grid, block, 0, ctx->stream, partial, count, width, split, out, out2);
  return check_hip(hipGetLastError(), "join launch");
}

namespace {

template <int ACT, int TAB>
void go_position(const lf_relative_position_args& a, int tile, int tiles, hipStream_t s) {
  const long long blocks = (long long)a.pairs->queries * tiles;
  hipLaunchKernelGGL((position_kernel<ACT, TAB>), dim3((unsigned)std::min(blocks, 1LL << 20)), dim3(256),
                     a.pairs->boundary_count * sizeof(int), s, *a.pairs, a.channels,
                     static_cast<const typename Act<TAB>::T*>(a.table), a.bias,
                     static_cast<const typename Act<ACT>::T*>(a.act), static_cast<typename Act<ACT>::T*>(a.out), tile, tiles, blocks);
}
template <int ACT>
void go_position(const lf_relative_position_args& a, int tile, int tiles, hipStream_t s) {
  if (a.table_dtype == LF_F32) go_position<ACT, DT_F32>(a, tile, tiles, s);
  else if (a.table_dtype == LF_F16) go_position<ACT, DT_F16>(a, tile, tiles, s);
  else go_position<ACT, DT_BF16>(a, tile, tiles, s);
}

constexpr int LDS_BYTES = 160 * 1024;

struct PositionPlan {
  int team, slices, chunks, waves, window, blocks;
  long long units;
};
PositionPlan position_plan(int queries, int keys, int channels, int rows) {
  PositionPlan p;
  p.team = channels > 64 ? 64 : channels > 32 ? 32 : channels > 16 ? 16 : 8;
  p.slices = (channels + 2 * p.team - 1) / (2 * p.team);
  p.chunks = (keys + 63) / 64;
  p.units = (long long)queries * p.chunks;
  // a wave's rows in LDS: 64 lanes of two sums each
  const int budget = (LDS_BYTES - rows * 4) / 512;
  p.waves = std::min(4, std::max(1, budget / rows));
  p.window = std::min(rows, budget / p.waves);
  const long long want = std::max(1, 256 / p.slices);
  p.blocks = (int)std::min(want, (p.units + p.waves - 1) / p.waves);
  return p;
}

template <int ACT, int L, bool EVEN>
int go_grad(lf_context* ctx, const lf_relative_position_backward_args& a, const PositionPlan& p, int rows, float* partial) {
  const auto kernel = position_grad_kernel<ACT, L, EVEN>;
  static const hipError_t lds_set = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                                        hipFuncAttributeMaxDynamicSharedMemorySize, LDS_BYTES);
  LF_TRY(check_hip(lds_set, "position gradient LDS"));
  for (int r0 = 0; r0 < rows; r0 += p.window) {
    const PositionGrid q{p.chunks, p.units, p.blocks, p.slices, r0, std::min(p.window, rows - r0), rows};
    const size_t lds = (size_t)p.waves * q.rows * 512 + a.pairs->boundary_count * 4;
    LaunchScope ls(ctx, "position.grad");
    hipLaunchKernelGGL(kernel, dim3(p.blocks * p.slices), dim3(p.waves * 64), lds, ctx->stream, *a.pairs, a.channels,
                       static_cast<const typename Act<ACT>::T*>(a.grad), partial, q);
    LF_TRY(check_hip(hipGetLastError(), "position gradient launch"));
  }
  return LF_OK;
}
template <int ACT, int L>
int go_grad(lf_context* ctx, const lf_relative_position_backward_args& a, const PositionPlan& p, int rows, float* partial) {
  return a.channels % 2 ? go_grad<ACT, L, false>(ctx, a, p, rows, partial) : go_grad<ACT, L, true>(ctx, a, p, rows, partial);
}
template <int ACT>
int go_grad(lf_context* ctx, const lf_relative_position_backward_args& a, const PositionPlan& p, int rows, float* partial) {
  if (p.team == 64) return go_grad<ACT, 64>(ctx, a, p, rows, partial);
  if (p.team == 32) return go_grad<ACT, 32>(ctx, a, p, rows, partial);
  if (p.team == 16) return go_grad<ACT, 16>(ctx, a, p, rows, partial);
  return go_grad<ACT, 8>(ctx, a, p, rows, partial);
}

}  // namespace

int run_relative_position(lf_context* ctx, const lf_relative_position_args& a) {
  // few pairs: small tiles, so that they fill the chip
  const long long pairs = (long long)a.pairs->queries * a.pairs->keys;
  const int tile = pairs >= 256 * 512 ? 256 : pairs >= 64 * 512 ? 64 : 16;
  const int tiles = (a.pairs->keys + tile - 1) / tile;
  LaunchScope ls(ctx, "position");
  if (a.act_dtype == LF_F32) go_position<DT_F32>(a, tile, tiles, ctx->stream);
  else if (a.act_dtype == LF_F16) go_position<DT_F16>(a, tile, tiles, ctx->stream);
  else go_position<DT_BF16>(a, tile, tiles, ctx->stream);
  return check_hip(hipGetLastError(), "position launch");
}

size_t relative_partials(int queries, int keys, int channels, int rows) {
  return (size_t)position_plan(queries, keys, channels, rows).blocks * (rows + 1) * channels * sizeof(float);
}

int run_relative_position_backward(lf_context* ctx, const lf_relative_position_backward_args& a, void* scratch) {
  const int rows = LF_RELATIVE_ROWS(a.pairs);
  const PositionPlan p = position_plan(a.pairs->queries, a.pairs->keys, a.channels, rows);
  float* const partial = static_cast<float*>(scratch);
  if (a.act_dtype == LF_F32) LF_TRY(go_grad<DT_F32>(ctx, a, p, rows, partial));
  else if (a.act_dtype == LF_F16) LF_TRY(go_grad<DT_F16>(ctx, a, p, rows, partial));
  else LF_TRY(go_grad<DT_BF16>(ctx, a, p, rows, partial));
  return run_join(ctx, partial, p.blocks, (long long)(rows + 1) * a.channels, (long long)rows * a.channels, a.grad_table,
                  a.grad_bias, a.grad_dtype, "position.join");
}

}  // namespace lf
