// Products of 8-bit operands: out[m][n] = sum_k x[m][k] w[n][k], x a checkpoint (a scale per row and 128
// columns), w packed (a scale per tile of 128 x 128), with bias, ReLU or a ReLU's gradient, residual,
// and an output that is kept in 8 bits itself.
#include <algorithm>

#include "lf_train.h"

namespace lf {

typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));

// Eight codes times a power of two as bf16, exact.
__device__ __forceinline__ b8 codes_bf16(uint2 w, float s) {
  const b2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w.x, s, false);
  const b2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w.x, s, true);
  const b2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w.y, s, false);
  const b2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w.y, s, true);
  return b8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// One block: 16 rows by 128 outputs, one 16 x 16 tile a wave, operands straight from memory.
template <int OUT>
__global__ __launch_bounds__(512) void fp8_linear_kernel(LinearParams p) {
  __shared__ float top[8][16];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, i16 = lane & 15, g = lane >> 4;
  const int nb = (p.outputs + GROUP - 1) / GROUP;
  const size_t m = (size_t)(blockIdx.x / nb) * 16 + i16;
  const int nblk = blockIdx.x % nb, n0 = nblk * GROUP + wave * 16;
  const size_t mr = m < (size_t)p.rows ? m : (size_t)p.rows - 1;
  const int nr = n0 + i16 < p.outputs ? n0 + i16 : p.outputs - 1;
  const int kg = (p.inputs + GROUP - 1) / GROUP, pitch = p.x.pitch;
  f4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int kb = 0; kb < kg; ++kb) {
    const float sx = scale_value(p.x.scales[(size_t)kb * p.x.sp + mr]), sw = scale_value(p.ws[nblk * kg + kb]);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int k = kb * GROUP + q * 32 + g * 8;
      uint2 a = make_uint2(0, 0), b = make_uint2(0, 0);
      if (k < pitch) {
        a = *reinterpret_cast<const uint2*>(p.w + (size_t)nr * pitch + k);
        b = *reinterpret_cast<const uint2*>(p.x.codes + mr * pitch + k);
      }
      acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(codes_bf16(a, sw), codes_bf16(b, sx), acc, 0, 0, 0);
    }
  }
  // lane: outputs n .. n + 3 of row m
  const int n = n0 + 4 * g;
  float v[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float t = acc[j];
    if (n + j < p.outputs) {
      if (p.bias) t += p.bias[n + j];
      if (p.relu) t = t < 0.f ? 0.f : t;
      if (p.relu_of && (int8_t)p.relu_of[mr * p.q.pitch + n + j] <= 0) t = 0.f;
    } else {
      t = 0.f;
    }
    v[j] = t;
  }
  typedef typename Act<OUT>::T T;
  if (p.out) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (m < (size_t)p.rows && n + j < p.outputs) {
        const size_t at = m * p.outputs + n + j;
        if (p.residual) v[j] += Act<OUT>::ld(static_cast<const T*>(p.residual) + at);
        Act<OUT>::st(static_cast<T*>(p.out) + at, v[j]);
      }
    return;
  }
  float f = 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) f = fmaxf(f, fabsf(v[j]) < __builtin_inff() ? fabsf(v[j]) : 0.f);
  f = lanes4_max(f);
  if (g == 0) top[wave][i16] = f;
  __syncthreads();
  f = top[0][i16];
#pragma unroll
  for (int w = 1; w < 8; ++w) f = fmaxf(f, top[w][i16]);
  const int byte = scale_byte(f);
  const float inv = scale_inverse(byte);
  int c = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * inv, v[1] * inv, 0, false);
  c = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * inv, v[3] * inv, c, true);
  if (m < (size_t)p.rows) {
    if (n < p.q.pitch) *reinterpret_cast<int*>(p.q.codes + m * p.q.pitch + n) = c;
    if (wave == 0 && g == 0) p.q.scales[(size_t)nblk * p.q.sp + m] = (uint8_t)byte;
  }
}

int run_fp8_linear(lf_context* ctx, const LinearParams& p, int out_dtype, const char* label) {
  LaunchScope ls(ctx, label);
  const long long blocks = ((long long)p.rows + 15) / 16 * ((p.outputs + GROUP - 1) / GROUP);
  auto k = out_dtype == LF_F32 ? fp8_linear_kernel<DT_F32> : out_dtype == LF_F16 ? fp8_linear_kernel<DT_F16>
                                                                                 : fp8_linear_kernel<DT_BF16>;
  hipLaunchKernelGGL(k, dim3((unsigned)blocks), dim3(512), 0, ctx->stream, p);
  return check_hip(hipGetLastError(), "fp8 linear launch");
}

}  // namespace lf
