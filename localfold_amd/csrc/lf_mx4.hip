// Matrices of 4 bits: pack and unpack (lf_mx4_pack, lf_mx4_unpack).
#include <algorithm>

#include "lf_mx4.h"

namespace lf {

// ---- pack and unpack: bound by memory ------------------------------------------------------------

// Four lanes pack a group of a row, 8 columns each.  8192 rows of 4096 in bf16: 16 us, 5.4 TB/s.
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

// A block walks down `chunk` tiles of 128 rows by 128 columns, reads each once, a tile ahead, into LDS and packs it along the
// columns (k.codes, if given) and along the rows (t.codes, if given), a group a thread, and adds up its rows (partial
// [chunks][cols], if given).  Four neighbouring lanes write 64 bytes (where every lane wrote 16 of another line, what both
// wrote of 196608 rows of 1024 in bf16 took 120 us beside the 82 of reading).  Blocks of neighbouring columns share an XCD,
// and a block keeps its columns: halves of lines meet in one L2.  Those packs take 113 us, 5.4 TB/s.
struct PackBoth {
  int rows, cols, col_tiles, row_tiles, chunk, blocks;
};
// BEYOND: the cache behind the L2s does not hold x, loads pass by it.
template <int ACT, bool BEYOND>
__global__ __launch_bounds__(256) void mx4_pack_both_kernel(const typename Act<ACT>::T* x, Mx k, Mx t, float* partial, PackBoth q) {
  typedef typename Act<ACT>::T T;
  constexpr int V = 16 / (int)sizeof(T), LANES = 128 / V, ROWS = 256 / LANES, PASSES = 128 / ROWS;   // as it reads
  // A row's 16 bytes more put neighbouring rows 4 banks apart; groups of 32 rows start 16 columns apart.
  constexpr int PITCH = 128 + V, SKEW = 16;
  __shared__ __attribute__((aligned(16))) T tile[128 * PITCH + 4 * SKEW];
  const int index = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
  if (index >= q.blocks) return;
  const int rc = index / q.col_tiles, c0 = index % q.col_tiles * 128, last = min((rc + 1) * q.chunk, q.row_tiles);
  const int lr = threadIdx.x / LANES, lc = threadIdx.x % LANES * V, left = q.cols - c0 - lc;
  const int item = threadIdx.x >> 2, g = threadIdx.x & 3;        // as it packs: row or column, group
  u32x4 in[PASSES];
  auto load = [&](int rt) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int r = rt * 128 + i * ROWS + lr;
      const T* const at = x + (size_t)r * q.cols + c0 + lc;
      in[i] = u32x4{0, 0, 0, 0};
      if (r < q.rows && left >= V) {
        if constexpr (BEYOND) stream_in(in[i], at);
        else __builtin_memcpy(&in[i], at, 16);
      } else if (r < q.rows && left > 0) {
        T v[V] = {};
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (e < left) v[e] = at[e];
        __builtin_memcpy(&in[i], v, 16);
      }
    }
  };
  float sum[2] = {0.f, 0.f};
  load(rc * q.chunk);
  for (int rt = rc * q.chunk; rt < last; ++rt) {
    const int r0 = rt * 128;
    __syncthreads();     // the last tile is read
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int r = i * ROWS + lr;
      *reinterpret_cast<u32x4*>(&tile[r * PITCH + (r >> 5) * SKEW + lc]) = in[i];
    }
    __syncthreads();
    if (rt + 1 < last) load(rt + 1);
    if (k.codes) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = i * 64 + item;
        const T* const at = &tile[r * PITCH + (r >> 5) * SKEW + g * 32];
        MxRaw<ACT> v;
        u32x4 w;
#pragma unroll
        for (int e = 0; e < MxRaw<ACT>::WORDS / 4; ++e) {
          const u32x4 four = *reinterpret_cast<const u32x4*>(at + e * V);
#pragma unroll
          for (int h = 0; h < 4; ++h) v.w[4 * e + h] = four[h];
        }
        const int b = v.quantise(w);
        if (r0 + r < q.rows) {
          *reinterpret_cast<u32x4*>(k.codes + (size_t)(r0 + r) * k.pitch + c0 / 2 + g * 16) = w;
          k.scales[(size_t)(c0 / MX_GROUP + g) * k.sp + r0 + r] = (uint8_t)b;
        }
      }
    }
    if (t.codes || partial) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int c = i * 64 + item;
        const T* const at = &tile[g * (32 * PITCH + SKEW) + c];
        MxRaw<ACT> v;
#pragma unroll
        for (int j = 0; j < MxRaw<ACT>::WORDS; ++j) {
          if constexpr (ACT == DT_F32) {
            v.w[j] = __float_as_uint(at[j * PITCH]);
          } else {
            uint16_t lo, hi;
            __builtin_memcpy(&lo, at + 2 * j * PITCH, 2);
            __builtin_memcpy(&hi, at + (2 * j + 1) * PITCH, 2);
            v.w[j] = lo | (uint32_t)hi << 16;
          }
        }
        if (t.codes) {
          u32x4 w;
          const int b = v.quantise(w);
          if (c0 + c < q.cols) {
            *reinterpret_cast<u32x4*>(t.codes + (size_t)(c0 + c) * t.pitch + r0 / 2 + g * 16) = w;
            t.scales[(size_t)(r0 / MX_GROUP + g) * t.sp + c0 + c] = (uint8_t)b;
          }
        }
        if (partial) {
          float s = 0.f;
#pragma unroll
          for (int j = 0; j < MxRaw<ACT>::WORDS; ++j) {
            if constexpr (ACT == DT_F32) s += __uint_as_float(v.w[j]);
            else if constexpr (ACT == DT_BF16) s += __uint_as_float(v.w[j] << 16) + __uint_as_float(v.w[j] & 0xffff0000u);
            else s += h2f((uint16_t)v.w[j]) + h2f((uint16_t)(v.w[j] >> 16));
          }
          sum[i] += s;
        }
      }
    }
  }
  if (partial) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int c = c0 + i * 64 + item;
      float s = sum[i] + dpp_f<0xB1>(sum[i]);     // the four groups of a column, in one order
      s += dpp_f<0x4E>(s);
      if (g == 0 && c < q.cols) partial[(size_t)rc * q.cols + c] = s;
    }
  }
}

__device__ __forceinline__ float mx_decode(uint32_t code, float scale) {
  const int e = (code >> 1) & 3, m = code & 1;
  const float v = e ? (float)(2 + m) * __uint_as_float((uint32_t)(e + 125) << 23) : 0.5f * (float)m;
  return (code & 8 ? -v : v) * scale;
}

// Eight columns a thread.  8192 rows of 4096 to bf16: 22 us, 3.9 TB/s; 147456 of 512 40 us, 4.8 TB/s.
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
  PackBoth q{};
  q.rows = rows;
  q.cols = cols;
  q.col_tiles = (int)(LF_MX4_PITCH(cols) / 128);
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
  // That cache has 256 MB.  403 MB of 196608 rows of 1024 in bf16 (packs and products of a backward pass): 249 us, and 265
  // with plain loads; 46 MB of 90601 rows of 128 in f32, which it may still hold from the kernel that wrote them: 48 and 44.
  const bool beyond = (size_t)a.rows * a.cols * act_bytes(a.act_dtype) > (256u << 20);
  const dim3 grid((q.blocks + 7) / 8 * 8), block(256);
  const Mx k = a.out ? mx_view(*a.out) : Mx{}, t = a.transposed ? mx_view(*a.transposed) : Mx{};
  if (beyond) hipLaunchKernelGGL((mx4_pack_both_kernel<ACT, true>), grid, block, 0, s, x, k, t, partial, q);
  else hipLaunchKernelGGL((mx4_pack_both_kernel<ACT, false>), grid, block, 0, s, x, k, t, partial, q);
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
