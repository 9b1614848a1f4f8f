// A learned row per relative position added to every pair, and its gradient (lf_relative_position,
// lf_relative_position_backward).  Bound by memory: one addition a value.
#include <algorithm>
#include <climits>

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

// A block adds rows to tiles of `tile` (at most 256) keys of one query: the rows' numbers once a pair, in LDS, then 8
// channels a lane, FLIGHT loads under way.  Many pairs: blocks that stay, with the table and the bias added up in LDS once
// (TABLE_LDS), so that a pair costs its own bytes alone: 825 x 825 pairs of 128 channels in bf16, read and written, 62 us,
// 5.6 TB/s.  A table that LDS does not hold comes from the caches at the same rate (130 rows of it 64 us, 66 63.5).
struct PositionTiles {
  int tile, tiles;             // keys of a tile, tiles of a query
  long long count;             // tiles in all
  int rows;                    // of the table
};

template <int ACT, int TAB, bool TABLE_LDS>
__global__ __launch_bounds__(512, 4) void position_kernel(lf_relative_pairs p, int channels, const typename Act<TAB>::T* table,
                                                          const float* bias, const typename Act<ACT>::T* act,
                                                          typename Act<ACT>::T* out, PositionTiles q) {
  constexpr int FLIGHT = 4;
  __shared__ int rows[256];
  extern __shared__ __attribute__((aligned(16))) float position_smem[];
  const int chunks = (channels + 7) / 8, wide = chunks * 8, threads = blockDim.x;
  int* const boundaries = reinterpret_cast<int*>(position_smem + (TABLE_LDS ? q.rows * wide : 0));
  for (int i = threadIdx.x; i < p.boundary_count; i += threads) boundaries[i] = p.boundaries[i];
  // a thread's items of a tile: (key, chunk), `threads` apart
  const int key0 = threadIdx.x / chunks, chunk0 = threadIdx.x % chunks, dkey = threads / chunks, dchunk = threads % chunks;
  if constexpr (TABLE_LDS) {
    for (int row = key0, c = chunk0; row < q.rows;) {
      float v[8], d[8];
      load8<TAB>(table + (size_t)row * channels + c * 8, channels - c * 8, v);
      if (bias) {
        load8<DT_F32>(bias + c * 8, channels - c * 8, d);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] += d[k];
      }
      float4* const at = reinterpret_cast<float4*>(position_smem + row * wide + c * 8);
      at[0] = make_float4(v[0], v[1], v[2], v[3]);
      at[1] = make_float4(v[4], v[5], v[6], v[7]);
      row += dkey;
      c += dchunk;
      if (c >= chunks) {
        c -= chunks;
        ++row;
      }
    }
  }
  for (long long b = blockIdx.x; b < q.count; b += gridDim.x) {
    const int query = (int)(b / q.tiles), k0 = (int)(b % q.tiles) * q.tile, keys = min(q.tile, p.keys - k0);
    __syncthreads();
    if ((int)threadIdx.x < keys)
      rows[threadIdx.x] = row_of(p, p.query_positions[query], p.query_segments ? p.query_segments[query] : 0,
                                 k0 + threadIdx.x, boundaries);
    __syncthreads();
    const size_t first = ((size_t)query * p.keys + k0) * channels;
    int key = key0, chunk = chunk0;
    for (int i0 = threadIdx.x; i0 < keys * chunks; i0 += FLIGHT * threads) {
      float a[FLIGHT][8];
      int ks[FLIGHT], cs[FLIGHT];
#pragma unroll
      for (int f = 0; f < FLIGHT; ++f) {
        ks[f] = key;
        cs[f] = chunk * 8;
        key += dkey;
        chunk += dchunk;
        if (chunk >= chunks) {
          chunk -= chunks;
          ++key;
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) a[f][k] = 0.f;
        if (act && ks[f] < keys) load8<ACT>(act + first + (size_t)ks[f] * channels + cs[f], channels - cs[f], a[f]);
      }
#pragma unroll
      for (int f = 0; f < FLIGHT; ++f) {
        if (ks[f] >= keys) continue;
        const int row = rows[ks[f]], c = cs[f];
        if (row >= 0) {
          float v[8];
          if constexpr (TABLE_LDS) {
            const float4* const at = reinterpret_cast<const float4*>(position_smem + row * wide + c);
            const float4 x = at[0], y = at[1];
            v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w, v[4] = y.x, v[5] = y.y, v[6] = y.z, v[7] = y.w;
          } else {
            load8<TAB>(table + (size_t)row * channels + c, channels - c, v);
            if (bias) {
              float d[8];
              load8<DT_F32>(bias + c, channels - c, d);
#pragma unroll
              for (int k = 0; k < 8; ++k) v[k] += d[k];
            }
          }
#pragma unroll
          for (int k = 0; k < 8; ++k) a[f][k] += v[k];
        }
        typename Act<ACT>::T* const at = out + first + (size_t)ks[f] * channels + c;
        if (channels - c >= 8) {
          uint4 w[sizeof(*at) / 2];
          pack8<ACT>(a[f], w);
#pragma unroll
          for (int k = 0; k < (int)sizeof(*at) / 2; ++k) stream_out(reinterpret_cast<uint4*>(at) + k, w[k]);
        } else {
          store8<ACT>(at, channels - c, a[f]);
        }
      }
    }
  }
}

// ---- gradient ----------------------------------------------------------------------------------

// A lane sums two channels of the keys that its team of L lanes takes, in registers while the table's row stays
// the same (most pairs are beyond the last boundary, where it does) and into the team's own rows in LDS when it
// changes: no two lanes share an address, so the order of the sums is fixed.  Those rows, 512 bytes of each a wave, leave
// room for 4 waves a CU where there are 66 (80 for 3, 39 and fewer for all 8, more than about 300 for a part of the table
// at a time, with a pass over the gradient each): a wave has the next 32 loads under way while it adds up the last ones.
// (LDS's own float additions took twice as long as reading and writing: 39 us instead of 23 for 384 x 384 pairs of 128
// channels in bf16.)  Those take 20 now, 1.9 TB/s: bound by the waves that LDS has room for, each waiting for its loads.
struct PositionGrid {
  int chunks;               // units of a query
  long long units;
  int blocks, slices;       // blocks of a slice of 2 L channels
  int row0, rows;           // the table's rows that this launch sums
  int all;                  // rows of the table
};
constexpr int STEPS = 32;                                             // loads of a unit
constexpr int position_keys(int team) { return STEPS * (64 / team); }    // keys of a unit

template <int ACT, int L, bool EVEN>
__global__ __launch_bounds__(512) void position_grad_kernel(lf_relative_pairs p, int channels, const typename Act<ACT>::T* grad,
                                                            float* partial, PositionGrid q) {
  typedef typename Act<ACT>::T T;
  constexpr int TEAMS = 64 / L, WIDE = 2 * L, KEYS = position_keys(L), REGS = (KEYS + 63) / 64;
  struct Two {
    T v[2];
  };
  extern __shared__ __attribute__((aligned(16))) float position_smem[];
  float* const sums = position_smem;
  const int waves = blockDim.x >> 6, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int team = lane / L, tl = lane % L;
  const int slice = blockIdx.x / q.blocks, blk = blockIdx.x % q.blocks;
  const int c = slice * WIDE + 2 * tl;
  const int copies = waves * TEAMS, size = q.rows * WIDE;
  int* const boundaries = reinterpret_cast<int*>(sums + (size_t)copies * size);
  for (int i = threadIdx.x; i < p.boundary_count; i += blockDim.x) boundaries[i] = p.boundaries[i];
  for (int i = threadIdx.x; i < copies * size / 4; i += blockDim.x) reinterpret_cast<float4*>(sums)[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  __syncthreads();
  float* const mine = sums + (size_t)(wave * TEAMS + team) * size + 2 * tl;
  const int c0 = min(c, channels - (EVEN ? 2 : 1)), c1 = min(c + 1, channels - 1);
  const long long w = (long long)blk * waves + wave, all = (long long)q.blocks * waves;
  const long long u0 = q.units * w / all, u1 = q.units * (w + 1) / all;
  const int nb = p.boundary_count, b0 = nb ? boundaries[0] : INT_MIN, b1 = nb ? boundaries[nb - 1] : INT_MIN;
  const uint32_t row_bytes = (uint32_t)channels * sizeof(T);
  Two in[STEPS];
  int kp[REGS], ks[REGS], qp = 0, qs = 0, left = 0;
  int query = (int)(u0 / q.chunks), chunk = (int)(u0 % q.chunks);      // of the next unit to load
  // The loads of a unit: gradients, and the positions that its rows come from.
  auto load = [&]() __attribute__((always_inline)) {
    qp = p.query_positions[query];
    qs = p.query_segments ? p.query_segments[query] : 0;
    const int k0 = chunk * KEYS;
    left = min(KEYS, p.keys - k0);
#pragma unroll
    for (int i = 0; i < REGS; ++i) {
      const int key = k0 + min(i * 64 + lane, left - 1);
      kp[i] = p.key_positions[key];
      ks[i] = p.key_segments ? p.key_segments[key] : 0;
    }
    const char* const g = reinterpret_cast<const char*>(grad + ((size_t)query * p.keys + k0) * channels);
    const uint32_t most = (uint32_t)(left - 1) * row_bytes;      // keys past the end repeat the last one
    uint32_t at = (uint32_t)team * row_bytes;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const uint32_t row = min(at, most);
      if constexpr (EVEN) {
        __builtin_memcpy(&in[s], g + (row + c0 * (uint32_t)sizeof(T)), sizeof(Two));
      } else {
        in[s].v[0] = *reinterpret_cast<const T*>(g + (row + c0 * (uint32_t)sizeof(T)));
        in[s].v[1] = *reinterpret_cast<const T*>(g + (row + c1 * (uint32_t)sizeof(T)));
      }
      at += TEAMS * row_bytes;
    }
    if (++chunk == q.chunks) {
      chunk = 0;
      ++query;
    }
  };
  int cur = -1;
  float a0 = 0.f, a1 = 0.f, all0 = 0.f, all1 = 0.f;      // of the row, of all rows
  auto flush = [&]() __attribute__((always_inline)) {
    if (cur >= 0) {
      float2* const at = reinterpret_cast<float2*>(mine + cur * WIDE);
      const float2 old = *at;
      *at = make_float2(old.x + a0, old.y + a1);
      all0 += a0;
      all1 += a1;
    }
  };
  if (u0 < u1) load();
  for (long long u = u0; u < u1; ++u) {
    int row[REGS];
    bool same = true;
#pragma unroll
    for (int i = 0; i < REGS; ++i) {
      const long long d = (long long)qp - kp[i];
      // beyond the boundaries, as most are, there is nothing to search
      int r = d >= b1 ? nb : 0;
      if (__any(d >= b0 && d < b1)) r = bucket_of(d, boundaries, nb);
      if (p.key_segments) r = qs < 0 || ks[i] < 0 ? -1 : qs != ks[i] ? nb + 1 : r;
      r -= q.row0;
      row[i] = r < 0 || r >= q.rows || i * 64 + lane >= left ? -1 : r;
      const int first = __builtin_amdgcn_readfirstlane(row[0]);
      if (i * 64 + lane < KEYS) same = same && row[i] == first;
    }
    float v0[STEPS], v1[STEPS];
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      v0[s] = Act<ACT>::ld(in[s].v);
      v1[s] = Act<ACT>::ld(in[s].v + 1);
    }
    if (u + 1 < u1) load();
    if (__all(same)) {             // a unit of one row
      const int r = __builtin_amdgcn_readfirstlane(row[0]);
      if (r != cur) {
        flush();
        cur = r;
        a0 = a1 = 0.f;
      }
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        a0 += v0[s];
        a1 += v1[s];
      }
      continue;
    }
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const int k = s * TEAMS;
      const int r = TEAMS == 1 ? __builtin_amdgcn_readlane(row[k / 64], k % 64) : __shfl(row[k / 64], k % 64 + team);
      if (r != cur) {
        flush();
        cur = r;
        a0 = a1 = 0.f;
      }
      a0 += v0[s];
      a1 += v1[s];
    }
  }
  flush();
  __syncthreads();
  // the block's rows [all + 1][channels], the last one the sum of them all (over the launches of a table)
  float* const dst = partial + (size_t)blk * (q.all + 1) * channels + slice * WIDE;
  const int cn = min(WIDE, channels - slice * WIDE);
  for (int i = threadIdx.x; i < size / 4; i += blockDim.x) {
    float4 t = reinterpret_cast<const float4*>(sums)[i];
#pragma unroll 4
    for (int k = 1; k < copies; ++k) {
      const float4 v = *reinterpret_cast<const float4*>(sums + (size_t)k * size + 4 * i);
      t = make_float4(t.x + v.x, t.y + v.y, t.z + v.z, t.w + v.w);
    }
    const int row = 4 * i / WIDE, col = 4 * i % WIDE;
    float* const at = dst + (size_t)(q.row0 + row) * channels + col;
    if (col + 4 <= cn) {
      __builtin_memcpy(at, &t, 16);
    } else {
      if (col < cn) at[0] = t.x;
      if (col + 1 < cn) at[1] = t.y;
      if (col + 2 < cn) at[2] = t.z;
    }
  }
  __syncthreads();
  sums[(wave * TEAMS + team) * WIDE + 2 * tl] = all0;
  sums[(wave * TEAMS + team) * WIDE + 2 * tl + 1] = all1;
  __syncthreads();
  for (int i = threadIdx.x; i < cn; i += blockDim.x) {
    float t = 0.f;
    for (int k = 0; k < copies; ++k) t += sums[k * WIDE + i];
    float* const total = dst + (size_t)q.all * channels + i;
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

constexpr int TABLE_MOST = 64 * 1024;      // two blocks a CU

template <int ACT, int TAB>
int go_position(const lf_relative_position_args& a, hipStream_t s) {
  const long long pairs = (long long)a.pairs->queries * a.pairs->keys;
  PositionTiles q;
  // few pairs: small tiles, so that they fill the chip
  q.tile = pairs >= 256 * 512 ? 256 : pairs >= 64 * 512 ? 64 : 16;
  q.tiles = (int)(((long long)a.pairs->keys + q.tile - 1) / q.tile);     // 2^31 - 1 keys rounded up are more than an int
  q.count = (long long)a.pairs->queries * q.tiles;
  q.rows = LF_RELATIVE_ROWS(a.pairs);
  const size_t marks = a.pairs->boundary_count * sizeof(int), table = (size_t)q.rows * ((a.channels + 7) / 8 * 8) * sizeof(float);
  const auto* t = static_cast<const typename Act<TAB>::T*>(a.table);
  const auto* act = static_cast<const typename Act<ACT>::T*>(a.act);
  auto* out = static_cast<typename Act<ACT>::T*>(a.out);
  // what stays has to be read by every block first: worth it where a block adds many times as much
  if (table + marks <= TABLE_MOST && (size_t)pairs * a.channels >= 2 * 512 * 8 * (size_t)q.rows * a.channels) {
    const auto kernel = position_kernel<ACT, TAB, true>;
    static const hipError_t lds = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, TABLE_MOST);
    LF_TRY(check_hip(lds, "position LDS"));
    hipLaunchKernelGGL(kernel, dim3(512), dim3(512), table + marks, s, *a.pairs, a.channels, t, a.bias, act, out, q);
  } else {
    hipLaunchKernelGGL((position_kernel<ACT, TAB, false>), dim3((unsigned)std::min(q.count, 1LL << 20)), dim3(q.tile > 64 ? 512 : 256),
                       marks, s, *a.pairs, a.channels, t, a.bias, act, out, q);
  }
  return check_hip(hipGetLastError(), "position launch");
}
template <int ACT>
int go_position(const lf_relative_position_args& a, hipStream_t s) {
  if (a.table_dtype == LF_F32) return go_position<ACT, DT_F32>(a, s);
  if (a.table_dtype == LF_F16) return go_position<ACT, DT_F16>(a, s);
  return go_position<ACT, DT_BF16>(a, s);
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
  const int unit = position_keys(p.team);
  p.chunks = (int)(((long long)keys + unit - 1) / unit);
  p.units = (long long)queries * p.chunks;
  // a wave's rows in LDS: 64 lanes of two sums each
  const int budget = (LDS_BYTES - rows * 4) / 512;
  p.waves = std::min(8, std::max(1, budget / rows));
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
  LaunchScope ls(ctx, "position");
  if (a.act_dtype == LF_F32) return go_position<DT_F32>(a, ctx->stream);
  if (a.act_dtype == LF_F16) return go_position<DT_F16>(a, ctx->stream);
  return go_position<DT_BF16>(a, ctx->stream);
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
