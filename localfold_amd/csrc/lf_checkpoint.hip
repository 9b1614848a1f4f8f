// Activations kept in 8 bits (pack, unpack) and weights packed for 8-bit products.  Bound by memory.
#include <algorithm>

#include "lf_train.h"

namespace lf {

// A team of L lanes packs one group of one row: 16, or 8 for rows of one half group, of which 16 would idle
// (207872 rows of 64 in bf16: 7.8 us, with 16 lanes 12.7).  680625 rows of 128 in f32: 93 us, 4.7 TB/s.
template <int ACT, int L>
__global__ __launch_bounds__(256) void checkpoint_pack_kernel(const typename Act<ACT>::T* x, Kept k, int groups) {
  const long long item = (long long)blockIdx.x * (256 / L) + threadIdx.x / L;
  const long long total = (long long)k.rows * groups;
  const bool valid = item < total;
  const long long i = valid ? item : total - 1;
  const size_t row = (size_t)(i / groups);
  const int c0 = (int)(i % groups) * GROUP + (threadIdx.x % L) * 8;
  float v[8];
  load8<ACT>(x + row * (size_t)k.cols + c0, k.cols - c0, v);
  keep8<L>(k, row, c0, v, valid);
}

template <int ACT>
__global__ __launch_bounds__(256) void checkpoint_unpack_kernel(typename Act<ACT>::T* x, Kept k, int chunks) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= (long long)k.rows * chunks) return;
  const size_t row = (size_t)(i / chunks);
  const int c0 = (int)(i % chunks) * 8;
  const uint2 w = *reinterpret_cast<const uint2*>(k.codes + row * (size_t)k.pitch + c0);
  const float s = scale_value(k.scales[(size_t)(c0 / GROUP) * k.sp + row]);
  float v[8];
  decode4(w.x, s, v);
  decode4(w.y, s, v + 4);
  store8<ACT>(x + row * (size_t)k.cols + c0, k.cols - c0, v);
}

constexpr int PACK_MOST = 4;
struct PackBatch {
  PackWeight w[PACK_MOST];
  int first[PACK_MOST + 1];     // first block of each matrix
  int count;
};

// One block packs one tile of 128 x 128 of the stored matrix: read once into LDS, 8 consecutive values a
// lane, its largest magnitude, then the codes, 8 consecutive of a packed row a lane.  A matrix has few
// tiles, so a block is as large as it can be: latency is what a pack costs.
template <int ACT>
__device__ __forceinline__ float pack_weight_load(const PackWeight& w, int r0, int c0, float (*tile)[GROUP + 1]) {
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int e = i * 1024 + threadIdx.x, r = e >> 4, c = (e & 15) * 8;
    float v[8] = {};
    if (r0 + r < w.rows)
      load8<ACT>(static_cast<const typename Act<ACT>::T*>(w.data) + (size_t)(r0 + r) * w.cols + c0 + c, w.cols - c0 - c, v);
#pragma unroll
    for (int k = 0; k < 8; ++k) tile[r][c + k] = v[k];
    top = fmaxf(top, amax8_finite(v));
  }
  return top;
}

__global__ __launch_bounds__(1024) void pack_weight_kernel(PackBatch b) {
  __shared__ float tile[GROUP][GROUP + 1];
  __shared__ float sm[16];
  int m = 0;
  while (m + 1 < b.count && (int)blockIdx.x >= b.first[m + 1]) ++m;
  const PackWeight& w = b.w[m];
  const int tc = (w.cols + GROUP - 1) / GROUP;
  const int t = blockIdx.x - b.first[m], r0 = t / tc * GROUP, c0 = t % tc * GROUP;
  float top = w.dtype == DT_F32   ? pack_weight_load<DT_F32>(w, r0, c0, tile)
              : w.dtype == DT_F16 ? pack_weight_load<DT_F16>(w, r0, c0, tile)
                                  : pack_weight_load<DT_BF16>(w, r0, c0, tile);
  top = team_reduce<64, OpMax>(top);
  if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = top;
  __syncthreads();
  top = team_reduce<16, OpMax>(sm[threadIdx.x & 15]);
  const int byte = scale_byte(top);
  const float f = scale_value(byte);
  const int rows = w.transpose ? w.cols : w.rows, cols = w.transpose ? w.rows : w.cols;   // of the packed matrix
  const int p0 = w.transpose ? c0 : r0, q0 = w.transpose ? r0 : c0;
  const int pitch = (int)LF_CHECKPOINT_PITCH(cols);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int e = i * 1024 + threadIdx.x;
    // transposed, neighbouring lanes take neighbouring rows: LDS columns without bank conflicts
    const int r = w.transpose ? e & 127 : e >> 4, c = w.transpose ? (e >> 7) * 8 : (e & 15) * 8;
    if (p0 + r >= rows || q0 + c >= pitch) continue;
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = w.transpose ? tile[c + k][r] : tile[r][c + k];
    *reinterpret_cast<uint2*>(w.codes + (size_t)(p0 + r) * pitch + q0 + c) = encode8(v, f);
  }
  if (threadIdx.x == 0) w.scales[(size_t)(p0 / GROUP) * ((cols + GROUP - 1) / GROUP) + q0 / GROUP] = (uint8_t)byte;
}

namespace {
template <int ACT>
void go_pack(const void* act, const Kept& k, hipStream_t s) {
  typedef typename Act<ACT>::T T;
  const int groups = (k.cols + GROUP - 1) / GROUP, team = k.cols <= 64 ? 8 : 16, per = 256 / team;
  const dim3 grid((unsigned)(((long long)k.rows * groups + per - 1) / per));
  if (team == 8)
    hipLaunchKernelGGL((checkpoint_pack_kernel<ACT, 8>), grid, dim3(256), 0, s, static_cast<const T*>(act), k, groups);
  else
    hipLaunchKernelGGL((checkpoint_pack_kernel<ACT, 16>), grid, dim3(256), 0, s, static_cast<const T*>(act), k, groups);
}
template <int ACT>
void go_unpack(void* act, const Kept& k, hipStream_t s) {
  const int chunks = (k.cols + 7) / 8;
  const dim3 grid((unsigned)(((long long)k.rows * chunks + 255) / 256));
  hipLaunchKernelGGL((checkpoint_unpack_kernel<ACT>), grid, dim3(256), 0, s, static_cast<typename Act<ACT>::T*>(act), k,
                     chunks);
}
}  // namespace

int run_checkpoint_pack(lf_context* ctx, const void* act, int dt, const Kept& k) {
  LaunchScope ls(ctx, "checkpoint.pack");
  if (dt == LF_F32) go_pack<DT_F32>(act, k, ctx->stream);
  else if (dt == LF_F16) go_pack<DT_F16>(act, k, ctx->stream);
  else go_pack<DT_BF16>(act, k, ctx->stream);
  return check_hip(hipGetLastError(), "checkpoint pack launch");
}

int run_checkpoint_unpack(lf_context* ctx, void* act, int dt, const Kept& k) {
  LaunchScope ls(ctx, "checkpoint.unpack");
  if (dt == LF_F32) go_unpack<DT_F32>(act, k, ctx->stream);
  else if (dt == LF_F16) go_unpack<DT_F16>(act, k, ctx->stream);
  else go_unpack<DT_BF16>(act, k, ctx->stream);
  return check_hip(hipGetLastError(), "checkpoint unpack launch");
}

int run_pack_weights(lf_context* ctx, const PackWeight* w, int count) {
  PackBatch b{};
  b.count = count;
  for (int i = 0; i < count; ++i) {
    b.w[i] = w[i];
    b.first[i + 1] = b.first[i] + (int)(LF_CHECKPOINT_GROUPS(w[i].rows) * LF_CHECKPOINT_GROUPS(w[i].cols));
  }
  LaunchScope ls(ctx, "fp8.pack_weight");
  hipLaunchKernelGGL(pack_weight_kernel, dim3(b.first[count]), dim3(1024), 0, ctx->stream, b);
  return check_hip(hipGetLastError(), "fp8 weight pack launch");
}

}  // namespace lf
