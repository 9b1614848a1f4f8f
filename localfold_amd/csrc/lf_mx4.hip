// Matrices of 4 bits: pack and unpack (lf_mx4_pack, lf_mx4_unpack).
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

// A block walks down `chunk` tiles of 128 rows by 64 columns, reads each once and packs it along the columns (k.codes, if
// given), along the rows (t.codes, if given), and adds up its rows (partial [chunks][cols], if given).  Blocks of
// neighbouring columns share an XCD, and a block keeps its columns: what they write meets in lines of one L2.
struct PackBoth {
  int rows, cols, col_tiles, row_tiles, chunk, blocks;
};
template <int ACT>
__global__ __launch_bounds__(256) void mx4_pack_both_kernel(const typename Act<ACT>::T* x, Mx k, Mx t, float* partial, PackBoth q) {
  __shared__ float tile[128][64];
  __shared__ float sm[4][64];
  const int index = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
  if (index >= q.blocks) return;
  const int rc = index / q.col_tiles, c0 = index % q.col_tiles * 64, last = min((rc + 1) * q.chunk, q.row_tiles);
  const int lr = threadIdx.x >> 3, lc = (threadIdx.x & 7) * 8;   // as it reads: row of 32, columns
  const int c = threadIdx.x & 63, g = threadIdx.x >> 6;          // as it packs along the rows: column, group of 32 rows
  float sum = 0.f;
  for (int rt = rc * q.chunk; rt < last; ++rt) {
    const int r0 = rt * 128;
    float in[4][8];
#pragma unroll
    for (int pass = 0; pass < 4; ++pass) {
      const int r = r0 + pass * 32 + lr;
#pragma unroll
      for (int j = 0; j < 8; ++j) in[pass][j] = 0.f;
      if (r < q.rows && c0 + lc < q.cols) load8<ACT>(x + (size_t)r * q.cols + c0 + lc, q.cols - c0 - lc, in[pass]);
    }
    __syncthreads();     // the last tile is read
#pragma unroll
    for (int pass = 0; pass < 4; ++pass) {
      const int r = r0 + pass * 32 + lr;
      *reinterpret_cast<float4*>(&tile[pass * 32 + lr][lc]) = make_float4(in[pass][0], in[pass][1], in[pass][2], in[pass][3]);
      *reinterpret_cast<float4*>(&tile[pass * 32 + lr][lc + 4]) = make_float4(in[pass][4], in[pass][5], in[pass][6], in[pass][7]);
      if (k.codes) {
        const int b = mx_scale_byte(quad_max(amax_bits8(in[pass])));
        if (r < q.rows) {
          *reinterpret_cast<uint32_t*>(k.codes + (size_t)r * k.pitch + (c0 + lc) / 2) = mx_encode8(in[pass], mx_scale_value(b));
          if (lc % MX_GROUP == 0) k.scales[(size_t)((c0 + lc) / MX_GROUP) * k.sp + r] = (uint8_t)b;
        }
      }
    }
    __syncthreads();
    float v[32];
    uint32_t m = 0;
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      v[j] = tile[g * 32 + j][c];
      m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
      s += v[j];
    }
    sum += s;
    if (t.codes && c0 + c < q.cols) {
      const int b = mx_scale_byte(m);
      const float f = mx_scale_value(b);
      const uint4 w = make_uint4(mx_encode8(v, f), mx_encode8(v + 8, f), mx_encode8(v + 16, f), mx_encode8(v + 24, f));
      *reinterpret_cast<uint4*>(t.codes + (size_t)(c0 + c) * t.pitch + r0 / 2 + g * 16) = w;
      t.scales[(size_t)(r0 / MX_GROUP + g) * t.sp + c0 + c] = (uint8_t)b;
    }
  }
  if (partial) {
    sm[g][c] = sum;
    __syncthreads();
    if (g == 0 && c0 + c < q.cols) partial[(size_t)rc * q.cols + c0 + c] = sm[0][c] + sm[1][c] + sm[2][c] + sm[3][c];
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

// About 2048 blocks, twice what the chip holds at a time.
PackBoth pack_both(int rows, int cols) {
  PackBoth q;
  q.rows = rows;
  q.cols = cols;
  q.col_tiles = (int)(LF_MX4_PITCH(cols) / 64);
  q.row_tiles = (int)(((long long)rows + 127) / 128);
  const int chunks = std::min(q.row_tiles, std::max(1, 2048 / q.col_tiles));
  q.chunk = (q.row_tiles + chunks - 1) / chunks;
  q.blocks = (q.row_tiles + q.chunk - 1) / q.chunk * q.col_tiles;
  return q;
}

template <int ACT>
void go_pack(const lf_mx4_pack_args& a, float* partial, hipStream_t s) {
  const auto* x = static_cast<const typename Act<ACT>::T*>(a.act);
  if (!a.transposed && !a.sums) {
    const Mx k = mx_view(*a.out);
    hipLaunchKernelGGL((mx4_pack_kernel<ACT>), dim3((unsigned)((k.rows * (k.pitch / 4) + 255) / 256)), dim3(256), 0, s, x, k);
    return;
  }
  const PackBoth q = pack_both(a.rows, a.cols);
  hipLaunchKernelGGL((mx4_pack_both_kernel<ACT>), dim3((q.blocks + 7) / 8 * 8), dim3(256), 0, s, x,
                     a.out ? mx_view(*a.out) : Mx{}, a.transposed ? mx_view(*a.transposed) : Mx{}, partial, q);
}
template <int ACT>
void go_unpack(const lf_mx4_unpack_args& a, hipStream_t s) {
  const Mx k = mx_view(*a.kept);
  const int chunks = (k.cols + 7) / 8;
  hipLaunchKernelGGL((mx4_unpack_kernel<ACT>), dim3((unsigned)(((long long)k.rows * chunks + 255) / 256)), dim3(256), 0, s,
                     static_cast<typename Act<ACT>::T*>(a.act), k, chunks);
}
}  // namespace

size_t mx4_sum_partials(int rows, int cols) {
  const PackBoth q = pack_both(rows, cols);
  return (size_t)(q.blocks / q.col_tiles) * cols * sizeof(float);
}

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
  const PackBoth q = pack_both(a.rows, a.cols);
  return run_join(ctx, partial, q.blocks / q.col_tiles, a.cols, a.cols, a.sums, nullptr, a.sums_dtype, "mx4.sums");
}

int run_mx4_unpack(lf_context* ctx, const lf_mx4_unpack_args& a) {
  LaunchScope ls(ctx, "mx4.unpack");
  if (a.act_dtype == LF_F32) go_unpack<DT_F32>(a, ctx->stream);
  else if (a.act_dtype == LF_F16) go_unpack<DT_F16>(a, ctx->stream);
  else go_unpack<DT_BF16>(a, ctx->stream);
  return check_hip(hipGetLastError(), "4-bit unpack launch");
}

}  // namespace lf
