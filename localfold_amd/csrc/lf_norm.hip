// LayerNorm forward and backward.
//
//   m = E[x], v = E[(x - m)^2] (or E[x^2] - m^2), r = 1 / sqrt(v + eps), y = (x - m) r s + o
//   h = (x - m) r, g = dy s:  dx = r (g - E[g] - h E[g h]),  ds = sum dy h,  do = sum dy
//
// Both are bound by memory: a row is read once into registers, 8 consecutive channels a lane and
// vector, and its sums go over a team of L lanes (L * NV * 8 >= channels) by permutes.  The team is
// small, so that narrow rows share a wave (team_of); rows past 1024 channels take the whole block, whose four
// waves join their sums in LDS.
#include <algorithm>
#include <type_traits>

#include "lf_train.h"

namespace lf {

struct NormParams {
  const void* x;
  const float *scale, *offset;
  void* out;
  float *mean, *rstd;
  Kept xk, yk;                  // codes null: not wanted
  int rows, C;
  float eps;
  int fast_var;
};

struct NormGradParams {
  const void *dy, *x, *resid;
  Kept xk;                      // read where x is null
  const float *mean, *rstd, *scale;
  void* out;
  float* partial;               // [blocks][2][C], or null
  int rows, C;
};

// Sum over a row's lanes: a team within a wave, or the whole block (L = 256), which takes a slot of
// `sm` (4 floats) that no other sum of the same barrier interval uses.
template <int L>
__device__ __forceinline__ float row_sum(float v, float* sm) {
  if constexpr (L <= 64) {
    return team_reduce<L, OpSum>(v);
  } else {
    v = team_reduce<64, OpSum>(v);
    if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = v;
    __syncthreads();
    return (sm[0] + sm[1]) + (sm[2] + sm[3]);
  }
}

template <int ACT, int L, int NV>
__global__ __launch_bounds__(256) void norm_kernel(NormParams p) {
  typedef typename Act<ACT>::T T;
  __shared__ float sm[8];
  constexpr int SLOTS = 256 / L;
  const int lr = threadIdx.x % L;
  const long long row0 = (long long)blockIdx.x * SLOTS + threadIdx.x / L;
  const bool valid = row0 < p.rows;
  const size_t row = valid ? (size_t)row0 : (size_t)p.rows - 1;
  const int C = p.C;
  const T* src = static_cast<const T*>(p.x) + row * (size_t)C;
  float x[NV][8];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int c0 = (v * L + lr) * 8;
    load8<ACT>(src + c0, C - c0, x[v]);
  }
  float s = 0.f;
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int k = 0; k < 8; ++k) s += x[v][k];
  const float n = (float)C;
  const float mean = row_sum<L>(s, sm) / n;
  float q = 0.f;
  if (p.fast_var) {
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int k = 0; k < 8; ++k) q += x[v][k] * x[v][k];
    q = row_sum<L>(q, sm + 4) / n - mean * mean;
    q = q < 0.f ? 0.f : q;      // the difference of two roundings
  } else {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c0 = (v * L + lr) * 8;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float d = c0 + k < C ? x[v][k] - mean : 0.f;
        q += d * d;
      }
    }
    q = row_sum<L>(q, sm + 4) / n;
  }
  const float r = 1.0f / sqrtf(q + p.eps);
  if (valid && lr == 0 && p.mean) {
    p.mean[row] = mean;
    p.rstd[row] = r;
  }
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int c0 = (v * L + lr) * 8;
    if (p.xk.codes) keep8<(L < 16 ? L : 16)>(p.xk, row, c0, x[v], valid);
    if (p.out || p.yk.codes) {
      float g[8], o[8], y[8];
      load8<DT_F32>(p.scale + c0, C - c0, g);
      load8<DT_F32>(p.offset + c0, C - c0, o);
#pragma unroll
      for (int k = 0; k < 8; ++k) y[k] = c0 + k < C ? (x[v][k] - mean) * r * g[k] + o[k] : 0.f;
      if (p.yk.codes) keep8<(L < 16 ? L : 16)>(p.yk, row, c0, y, valid);
      if (p.out && valid) store8<ACT>(static_cast<T*>(p.out) + row * (size_t)C + c0, C - c0, y);
    }
  }
}

// Rows are dealt out to a fixed number of blocks, whose lanes add up their columns' ds and do in
// registers; a block joins its teams in LDS and writes one row of partial sums.
template <int ACT, int L, int NV, int DY>
__global__ __launch_bounds__(256) void norm_grad_kernel(NormGradParams p) {
  typedef typename Act<ACT>::T T;
  constexpr int SLOTS = 256 / L;
  __shared__ float sm[16];
  __shared__ float cols[L <= 64 ? SLOTS * L * 8 : 8];
  const int lr = threadIdx.x % L, slot = threadIdx.x / L;
  const int C = p.C;
  const float n = (float)C;
  float ds[NV][8] = {}, dof[NV][8] = {};
  int parity = 0;
  for (long long base = (long long)blockIdx.x * SLOTS; base < p.rows; base += (long long)gridDim.x * SLOTS) {
    const bool valid = base + slot < p.rows;
    const size_t row = valid ? (size_t)(base + slot) : (size_t)p.rows - 1;
    const float mean = p.mean[row], r = p.rstd[row];
    float dy[NV][8], h[NV][8], a = 0.f, b = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c0 = (v * L + lr) * 8;
      load8<DY>(static_cast<const typename Act<DY>::T*>(p.dy) + row * (size_t)C + c0, C - c0, dy[v]);
      if (p.x) {
        load8<ACT>(static_cast<const T*>(p.x) + row * (size_t)C + c0, C - c0, h[v]);
      } else {
        uint2 w = make_uint2(0, 0);
        float sc = 1.f;
        if (c0 < p.xk.pitch) {
          w = *reinterpret_cast<const uint2*>(p.xk.codes + row * (size_t)p.xk.pitch + c0);
          sc = scale_value(p.xk.scales[(size_t)(c0 / GROUP) * p.xk.sp + row]);
        }
        decode4(w.x, sc, h[v]);
        decode4(w.y, sc, h[v] + 4);
      }
    }
    float g[NV][8];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c0 = (v * L + lr) * 8;
      load8<DT_F32>(p.scale + c0, C - c0, g[v]);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        h[v][k] = c0 + k < C ? (h[v][k] - mean) * r : 0.f;
        if (valid) {
          ds[v][k] += dy[v][k] * h[v][k];
          dof[v][k] += dy[v][k];
        }
        g[v][k] *= dy[v][k];
        a += g[v][k];
        b += g[v][k] * h[v][k];
      }
    }
    if (!p.out) continue;       // uniform
    // the block's sums alternate between two sets of slots: a wave may still read the last row's
    a = row_sum<L>(a, sm + 8 * parity) / n;
    b = row_sum<L>(b, sm + 8 * parity + 4) / n;
    parity ^= 1;
    if (valid) {
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int c0 = (v * L + lr) * 8;
        float o[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k] = 0.f;
        if (p.resid) load8<ACT>(static_cast<const T*>(p.resid) + row * (size_t)C + c0, C - c0, o);
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k] += r * (g[v][k] - a - h[v][k] * b);
        store8<ACT>(static_cast<T*>(p.out) + row * (size_t)C + c0, C - c0, o);
      }
    }
  }
  if (!p.partial) return;
  float* dst = p.partial + (size_t)blockIdx.x * 2 * C;
  if constexpr (L > 64) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c0 = (v * L + lr) * 8;
      store8<DT_F32>(dst + c0, C - c0, ds[v]);
      store8<DT_F32>(dst + C + c0, C - c0, dof[v]);
    }
  } else {
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 8; ++k) cols[(slot * L + lr) * 8 + k] = half ? dof[v][k] : ds[v][k];
        __syncthreads();
        for (int c = threadIdx.x; c < L * 8; c += 256) {
          const int col = v * L * 8 + c;
          float t = 0.f;
          for (int i = 0; i < SLOTS; ++i) t += cols[i * L * 8 + c];
          if (col < C) dst[half * C + col] = t;
        }
      }
  }
}

// Columns of [blocks][2 C] partial sums added in order of the blocks: 16 columns a block, four a lane, in 256
// runs of the blocks, then 16 of 16 runs, then those.  Few columns a block, so that many read: 1024 rows of 256
// sums take 4.2 us, with 64 columns a block 4.4.
template <int OUT>
__global__ __launch_bounds__(1024) void norm_join_kernel(const float* partial, int blocks, int C, void* ds, void* dof) {
  __shared__ f4 sm[256][4];
  const int lane = threadIdx.x & 3, run = threadIdx.x >> 2, c = blockIdx.x * 16 + lane * 4;
  const int per = (blocks + 255) / 256, b0 = run * per, b1 = min(blocks, b0 + per);
  f4 t = {0.f, 0.f, 0.f, 0.f};
  if (c + 4 <= 2 * C) {
#pragma unroll 4
    for (int b = b0; b < b1; ++b) {
      f4 v;
      __builtin_memcpy(&v, partial + (size_t)b * 2 * C + c, 16);   // rows may be unaligned
      t += v;
    }
  } else {
    for (int b = b0; b < b1; ++b)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (c + k < 2 * C) t[k] += partial[(size_t)b * 2 * C + c + k];
  }
  sm[run][lane] = t;
  __syncthreads();
  if (run < 16) {
    t = sm[run * 16][lane];
#pragma unroll
    for (int i = 1; i < 16; ++i) t += sm[run * 16 + i][lane];
    sm[run * 16][lane] = t;
  }
  __syncthreads();
  if (run != 0) return;
#pragma unroll
  for (int i = 1; i < 16; ++i) t += sm[i * 16][lane];
  typedef typename Act<OUT>::T T;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (c + k < C) Act<OUT>::st(static_cast<T*>(ds) + c + k, t[k]);
    else if (c + k < 2 * C) Act<OUT>::st(static_cast<T*>(dof) + c + k - C, t[k]);
  }
}

namespace {

// A team and vectors a lane for a width: see the head of this file.  bf16, us: 147456 rows of 64 forward and
// backward 9 and 16, where a wave of two vectors a row takes 81 and 113; of 128 16 and 24 for 79 and 113; 100000 rows of
// 384 29 and 51 for 57 and 81.  Three vectors a lane are faster forward (29 us, two of a team of 32 36) and
// slower backward (55 us for 51), which holds three times as many.  196608 rows of 256: 33 and 47, with one vector of
// 32 lanes 36 and 50.
struct Team {
  int lanes, vectors;
};
Team team_of(int C, bool backward) {
  if (C <= 64) return {8, 1};
  if (C <= 128) return {16, 1};
  if (C <= 256) return {16, 2};
  if (C <= 384 && !backward) return {16, 3};
  if (C <= 512) return {32, 2};
  if (C <= 1024) return {64, 2};
  if (C <= 2048) return {256, 1};
  return {256, 2};
}

// At most; four a CU.  196608 rows of 256 from kept activations: 60 us, with 768 blocks 64, with 2048 62 and a join of
// 5.8 us for 4.8.
constexpr int GRAD_BLOCKS = 1024;

int grad_blocks(int rows, int C) {
  const int slots = 256 / team_of(C, true).lanes;
  return (int)std::min<long long>(((long long)rows + slots - 1) / slots, GRAD_BLOCKS);
}

template <template <int, int, int> class F, int ACT, class P>
void by_team(const Team& t, const P& p, dim3 grid, hipStream_t s) {
  if constexpr (std::is_same<P, NormParams>::value)
    if (t.vectors == 3) return F<ACT, 16, 3>::go(p, grid, s);
  if (t.lanes == 8) F<ACT, 8, 1>::go(p, grid, s);
  else if (t.lanes == 16 && t.vectors == 1) F<ACT, 16, 1>::go(p, grid, s);
  else if (t.lanes == 16 && t.vectors == 2) F<ACT, 16, 2>::go(p, grid, s);
  else if (t.lanes == 32) F<ACT, 32, 2>::go(p, grid, s);
  else if (t.lanes == 64) F<ACT, 64, 2>::go(p, grid, s);
  else if (t.vectors == 1) F<ACT, 256, 1>::go(p, grid, s);
  else F<ACT, 256, 2>::go(p, grid, s);
}
template <template <int, int, int> class F, class P>
void by_type(int dt, const Team& t, const P& p, dim3 grid, hipStream_t s) {
  if (dt == LF_F32) by_team<F, DT_F32>(t, p, grid, s);
  else if (dt == LF_F16) by_team<F, DT_F16>(t, p, grid, s);
  else by_team<F, DT_BF16>(t, p, grid, s);
}
template <int ACT, int L, int NV>
struct GoNorm {
  static void go(const NormParams& p, dim3 grid, hipStream_t s) {
    hipLaunchKernelGGL((norm_kernel<ACT, L, NV>), grid, dim3(256), 0, s, p);
  }
};
template <int ACT, int L, int NV>
struct GoNormGrad {
  static void go(const NormGradParams& p, dim3 grid, hipStream_t s) {
    hipLaunchKernelGGL((norm_grad_kernel<ACT, L, NV, ACT>), grid, dim3(256), 0, s, p);
  }
};
template <int ACT, int L, int NV>
struct GoNormGradWide {     // from a gradient in f32
  static void go(const NormGradParams& p, dim3 grid, hipStream_t s) {
    hipLaunchKernelGGL((norm_grad_kernel<ACT, L, NV, DT_F32>), grid, dim3(256), 0, s, p);
  }
};

}  // namespace

int run_layer_norm(lf_context* ctx, const lf_layer_norm_args& a) {
  NormParams p{};
  p.x = a.act;
  p.scale = a.scale;
  p.offset = a.offset;
  p.out = a.out;
  p.mean = a.mean;
  p.rstd = a.rstd;
  if (a.act_kept) p.xk = kept_view(*a.act_kept);
  if (a.out_kept) p.yk = kept_view(*a.out_kept);
  p.rows = a.rows;
  p.C = a.channels;
  p.eps = a.epsilon;
  p.fast_var = a.fast_variance;
  const Team t = team_of(a.channels, false);
  const int slots = 256 / t.lanes;
  LaunchScope ls(ctx, "layer_norm");
  by_type<GoNorm>(a.act_dtype, t, p, dim3((unsigned)(((long long)a.rows + slots - 1) / slots)), ctx->stream);
  return check_hip(hipGetLastError(), "layer_norm launch");
}

size_t layer_norm_partials(int rows, int channels) {
  return (size_t)grad_blocks(rows, channels) * 2 * channels * sizeof(float);
}

int run_layer_norm_backward(lf_context* ctx, const lf_layer_norm_backward_args& a, void* scratch, bool wide) {
  NormGradParams p{};
  p.dy = a.grad;
  p.x = a.act;
  p.resid = a.residual;
  if (a.act_kept) p.xk = kept_view(*a.act_kept);
  p.mean = a.mean;
  p.rstd = a.rstd;
  p.scale = a.scale;
  p.out = a.out;
  p.partial = a.grad_scale ? static_cast<float*>(scratch) : nullptr;
  p.rows = a.rows;
  p.C = a.channels;
  const int blocks = grad_blocks(a.rows, a.channels);
  {
    LaunchScope ls(ctx, "layer_norm.backward");
    const Team t = team_of(a.channels, true);
    if (wide) by_type<GoNormGradWide>(a.act_dtype, t, p, dim3(blocks), ctx->stream);
    else by_type<GoNormGrad>(a.act_dtype, t, p, dim3(blocks), ctx->stream);
  }
  LF_TRY(check_hip(hipGetLastError(), "layer_norm backward launch"));
  if (!a.grad_scale) return LF_OK;
  return run_norm_join(ctx, p.partial, blocks, a.channels, a.grad_scale, a.grad_offset, a.grad_dtype);
}

int run_norm_join(lf_context* ctx, const float* partial, int blocks, int channels, void* grad_scale, void* grad_offset,
                  int dt) {
  LaunchScope ls(ctx, "layer_norm.join");
  const dim3 grid((2 * channels + 15) / 16);
  auto k = dt == LF_F32 ? norm_join_kernel<DT_F32> : dt == LF_F16 ? norm_join_kernel<DT_F16> : norm_join_kernel<DT_BF16>;
  hipLaunchKernelGGL(k, grid, dim3(1024), 0, ctx->stream, partial, blocks, channels, grad_scale, grad_offset);
  return check_hip(hipGetLastError(), "layer_norm join launch");
}

}  // namespace lf
