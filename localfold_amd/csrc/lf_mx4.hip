// Matrices of 4 bits: pack, unpack and products (lf_mx4_pack, lf_mx4_unpack, lf_mx4_linear).
#include <algorithm>

#include "lf_mx4.h"

namespace lf {

// ---- pack and unpack: bound by memory ------------------------------------------------------------

// Four lanes pack a group of a row, 8 columns each.
template <int ACT>
__global__ __launch_bounds__(256) void mx4_pack_kernel(const typename Act<ACT>::T* x, Mx k) {
  const long long item = (long long)blockIdx.x * 256 + threadIdx.x;
  const int chunks = (int)(k.pitch / 4);            // of 8 columns
  const long long total = (long long)k.rows * chunks;
  const bool valid = item < total;
  const long long i = valid ? item : total - 1;
  const size_t row = (size_t)(i / chunks);
  const int c0 = (int)(i % chunks) * 8;
  float v[8];
  load8<ACT>(x + row * (size_t)k.cols + c0, k.cols - c0, v);
  const int b = mx_scale_byte(quad_max(amax_bits8(v)));
  if (!valid) return;
  *reinterpret_cast<uint32_t*>(k.codes + row * k.pitch + c0 / 2) = mx_encode8(v, mx_scale_value(b));
  if (c0 % MX_GROUP == 0) k.scales[(size_t)(c0 / MX_GROUP) * k.sp + row] = (uint8_t)b;
}

// A block reads a tile of 128 rows by 64 columns once and packs it along the columns (k.codes, if given), along
// the rows (t.codes, if given), and adds up its rows (partial [row tiles][cols], if given).
template <int ACT>
__global__ __launch_bounds__(256) void mx4_pack_both_kernel(const typename Act<ACT>::T* x, int rows, int cols, Mx k, Mx t,
                                                            float* partial, int col_tiles) {
  __shared__ float tile[128][64];
  __shared__ float sm[4][64];
  const int rt = blockIdx.x / col_tiles, r0 = rt * 128, c0 = blockIdx.x % col_tiles * 64;
#pragma unroll
  for (int pass = 0; pass < 4; ++pass) {
    const int r = pass * 32 + (threadIdx.x >> 3), c = (threadIdx.x & 7) * 8;
    float v[8] = {};
    if (r0 + r < rows && c0 + c < cols) load8<ACT>(x + (size_t)(r0 + r) * cols + c0 + c, cols - c0 - c, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) tile[r][c + j] = v[j];
    if (k.codes) {
      const int b = mx_scale_byte(quad_max(amax_bits8(v)));
      if (r0 + r < rows) {
        *reinterpret_cast<uint32_t*>(k.codes + (size_t)(r0 + r) * k.pitch + (c0 + c) / 2) = mx_encode8(v, mx_scale_value(b));
        if (c % MX_GROUP == 0) k.scales[(size_t)((c0 + c) / MX_GROUP) * k.sp + r0 + r] = (uint8_t)b;
      }
    }
  }
  __syncthreads();
  const int c = threadIdx.x & 63, g = threadIdx.x >> 6;      // a column's group of 32 rows
  float v[32];
  uint32_t m = 0;
  float sum = 0.f;
#pragma unroll
  for (int j = 0; j < 32; ++j) {
    v[j] = tile[g * 32 + j][c];
    m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
    sum += v[j];
  }
  if (t.codes && c0 + c < cols) {
    const int b = mx_scale_byte(m);
    const float f = mx_scale_value(b);
    const uint4 w = make_uint4(mx_encode8(v, f), mx_encode8(v + 8, f), mx_encode8(v + 16, f), mx_encode8(v + 24, f));
    *reinterpret_cast<uint4*>(t.codes + (size_t)(c0 + c) * t.pitch + r0 / 2 + g * 16) = w;
    t.scales[(size_t)(r0 / MX_GROUP + g) * t.sp + c0 + c] = (uint8_t)b;
  }
  if (partial) {
    sm[g][c] = sum;
    __syncthreads();
    if (g == 0 && c0 + c < cols) partial[(size_t)rt * cols + c0 + c] = sm[0][c] + sm[1][c] + sm[2][c] + sm[3][c];
  }
}

__device__ __forceinline__ float mx_decode(uint32_t code, float scale) {
  const int e = (code >> 1) & 3, m = code & 1;
  const float v = e ? (float)(2 + m) * __uint_as_float((uint32_t)(e + 125) << 23) : 0.5f * (float)m;
  return (code & 8 ? -v : v) * scale;
}

template <int ACT>
__global__ __launch_bounds__(256) void mx4_unpack_kernel(typename Act<ACT>::T* x, Mx k, int chunks) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= (long long)k.rows * chunks) return;
  const size_t row = (size_t)(i / chunks);
  const int c0 = (int)(i % chunks) * 8;
  const uint32_t w = *reinterpret_cast<const uint32_t*>(k.codes + row * k.pitch + c0 / 2);
  const int b = k.scales[(size_t)(c0 / MX_GROUP) * k.sp + row];
  const float s = b == 255 ? __builtin_nanf("") : b ? scale_value(b) : __uint_as_float(0x400000u);   // 0: 2^-127
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = mx_decode(w >> (4 * j), s);
  store8<ACT>(x + row * (size_t)k.cols + c0, k.cols - c0, v);
}

namespace {
template <int ACT>
void go_pack(const lf_mx4_pack_args& a, float* partial, hipStream_t s) {
  const auto* x = static_cast<const typename Act<ACT>::T*>(a.act);
  if (!a.transposed && !a.sums) {
    const Mx k = mx_view(*a.out);
    hipLaunchKernelGGL((mx4_pack_kernel<ACT>), dim3((unsigned)((k.rows * (k.pitch / 4) + 255) / 256)), dim3(256), 0, s, x, k);
    return;
  }
  const int col_tiles = (int)(LF_MX4_PITCH(a.cols) / 64);
  const long long row_tiles = ((long long)a.rows + 127) / 128;
  hipLaunchKernelGGL((mx4_pack_both_kernel<ACT>), dim3((unsigned)(row_tiles * col_tiles)), dim3(256), 0, s, x, a.rows, a.cols,
                     a.out ? mx_view(*a.out) : Mx{}, a.transposed ? mx_view(*a.transposed) : Mx{}, partial, col_tiles);
}
template <int ACT>
void go_unpack(const lf_mx4_unpack_args& a, hipStream_t s) {
  const Mx k = mx_view(*a.kept);
  const int chunks = (k.cols + 7) / 8;
  hipLaunchKernelGGL((mx4_unpack_kernel<ACT>), dim3((unsigned)(((long long)k.rows * chunks + 255) / 256)), dim3(256), 0, s,
                     static_cast<typename Act<ACT>::T*>(a.act), k, chunks);
}
}  // namespace

size_t mx4_sum_partials(int rows, int cols) { return ((size_t)rows + 127) / 128 * cols * sizeof(float); }

int run_mx4_pack(lf_context* ctx, const lf_mx4_pack_args& a, void* scratch) {
  float* const partial = a.sums ? static_cast<float*>(scratch) : nullptr;
  {
    LaunchScope ls(ctx, "mx4.pack");
    if (a.act_dtype == LF_F32) go_pack<DT_F32>(a, partial, ctx->stream);
    else if (a.act_dtype == LF_F16) go_pack<DT_F16>(a, partial, ctx->stream);
    else go_pack<DT_BF16>(a, partial, ctx->stream);
    LF_TRY(check_hip(hipGetLastError(), "4-bit pack launch"));
  }
  if (!a.sums) return LF_OK;
  return run_join(ctx, partial, (a.rows + 127) / 128, a.cols, a.cols, a.sums, nullptr, a.sums_dtype, "mx4.sums");
}

int run_mx4_unpack(lf_context* ctx, const lf_mx4_unpack_args& a) {
  LaunchScope ls(ctx, "mx4.unpack");
  if (a.act_dtype == LF_F32) go_unpack<DT_F32>(a, ctx->stream);
  else if (a.act_dtype == LF_F16) go_unpack<DT_F16>(a, ctx->stream);
  else go_unpack<DT_BF16>(a, ctx->stream);
  return check_hip(hipGetLastError(), "4-bit unpack launch");
}

// ---- products ------------------------------------------------------------------------------------

struct MxLinear {
  Mx x, w;
  int rows, outputs, steps;      // steps of 128 columns
  const float* bias;
  int relu;
  const void* residual;
  void* out;
};

// w is the instruction's first operand, so a lane's sums are 4 outputs of one row.  Row i of tile t (of 4) of the
// first operand is output 4 f(i) + t: the scale bytes of a lane's four tiles are one word.  f puts the 16 outputs
// that a lane holds in runs of 16 bytes, four lanes' runs side by side.
template <int OUT>
__device__ __forceinline__ int mx_f(int i) {
  return OUT == DT_F32 ? (i & 3) * 4 + (i >> 2) : (i & 2) * 4 + (i >> 2) * 2 + (i & 1);
}

// A wave computes 64 rows by 64 outputs, operands straight from memory.
template <int OUT>
__global__ __launch_bounds__(256) void mx4_linear_kernel(MxLinear p, int out_tiles, long long tiles) {
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const long long tile = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (tile >= tiles) return;
  const long long m0 = tile / out_tiles * 64;
  const int n0 = (int)(tile % out_tiles) * 64;
  const uint8_t *wrow[4], *xrow[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) {     // rows past the end repeat the last one
    wrow[t] = p.w.codes + (size_t)min(n0 + 4 * mx_f<OUT>(r) + t, p.outputs - 1) * p.w.pitch + 16 * g;
    xrow[t] = p.x.codes + (size_t)min(m0 + 4 * r + t, (long long)p.rows - 1) * p.x.pitch + 16 * g;
  }
  // scale rows are whole sixteens: a word of four is in bounds where its first byte's row exists
  const uint8_t* ws = p.w.scales + (size_t)g * p.w.sp + min(n0 + 4 * mx_f<OUT>(r), (p.outputs - 1) & ~3);
  const uint8_t* xs = p.x.scales + (size_t)g * p.x.sp + min(m0 + 4 * r, ((long long)p.rows - 1) & ~3LL);
  f4 acc[4][4];
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int q = 0; q < 4; ++q) acc[t][q] = f4{0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < p.steps; ++s) {
    u32x4 a[4], b[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      a[t] = *reinterpret_cast<const u32x4*>(wrow[t] + (size_t)s * 64);
      b[t] = *reinterpret_cast<const u32x4*>(xrow[t] + (size_t)s * 64);
    }
    const uint32_t sa = *reinterpret_cast<const uint32_t*>(ws + (size_t)4 * s * p.w.sp);
    const uint32_t sb = *reinterpret_cast<const uint32_t*>(xs + (size_t)4 * s * p.x.sp);
#define MX_ROW(T)                                     \
  acc[T][0] = mx_mma<T, 0>(a[T], b[0], acc[T][0], sa, sb); \
  acc[T][1] = mx_mma<T, 1>(a[T], b[1], acc[T][1], sa, sb); \
  acc[T][2] = mx_mma<T, 2>(a[T], b[2], acc[T][2], sa, sb); \
  acc[T][3] = mx_mma<T, 3>(a[T], b[3], acc[T][3], sa, sb);
    MX_ROW(0) MX_ROW(1) MX_ROW(2) MX_ROW(3)
#undef MX_ROW
  }
  typedef typename Act<OUT>::T T;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const long long m = m0 + 4 * r + q;
    if (m >= p.rows) continue;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int n = n0 + 4 * mx_f<OUT>(4 * g + j) + t;
        if (n >= p.outputs) continue;
        float v = acc[t][q][j];
        if (p.bias) v += p.bias[n];
        if (p.relu) v = __builtin_elementwise_maximum(v, 0.f);   // keeps NaN
        const size_t at = (size_t)m * p.outputs + n;
        if (p.residual) v += Act<OUT>::ld(static_cast<const T*>(p.residual) + at);
        Act<OUT>::st(static_cast<T*>(p.out) + at, v);
      }
  }
}

size_t mx4_linear_bytes(int rows, int inputs, int, bool from_act) {
  if (!from_act) return 0;
  return ((size_t)rows * LF_MX4_PITCH(inputs) / 2 + 255) / 256 * 256 + LF_MX4_GROUPS(inputs) * LF_MX4_SCALE_PITCH(rows);
}

int run_mx4_linear(lf_context* ctx, const lf_mx4_linear_args& a, void* scratch) {
  MxLinear p{};
  lf_mx4 packed{};
  if (a.act) {
    packed = {a.rows, a.w->cols, scratch,
              static_cast<char*>(scratch) + ((size_t)a.rows * LF_MX4_PITCH(a.w->cols) / 2 + 255) / 256 * 256};
    lf_mx4_pack_args k{};
    k.rows = a.rows;
    k.cols = a.w->cols;
    k.act_dtype = a.act_dtype;
    k.act = a.act;
    k.out = &packed;
    LF_TRY(run_mx4_pack(ctx, k, nullptr));
  }
  p.x = mx_view(a.act ? packed : *a.kept);
  p.w = mx_view(*a.w);
  p.rows = a.rows;
  p.outputs = a.w->rows;
  p.steps = (int)(LF_MX4_PITCH(a.w->cols) / 128);
  p.bias = a.bias;
  p.relu = a.relu;
  p.residual = a.residual;
  p.out = a.out;
  const int out_tiles = (p.outputs + 63) / 64;
  const long long tiles = ((long long)p.rows + 63) / 64 * out_tiles;
  LaunchScope ls(ctx, "mx4.linear");
  const dim3 grid((unsigned)((tiles + 3) / 4)), block(256);
  if (a.out_dtype == LF_F32) hipLaunchKernelGGL((mx4_linear_kernel<DT_F32>), grid, block, 0, ctx->stream, p, out_tiles, tiles);
  else if (a.out_dtype == LF_F16) hipLaunchKernelGGL((mx4_linear_kernel<DT_F16>), grid, block, 0, ctx->stream, p, out_tiles, tiles);
  else hipLaunchKernelGGL((mx4_linear_kernel<DT_BF16>), grid, block, 0, ctx->stream, p, out_tiles, tiles);
  return check_hip(hipGetLastError(), "4-bit product launch");
}

}  // namespace lf
