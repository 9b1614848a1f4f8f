// Weight gradients of 8-bit operands: out[i][j] = sum_m a[m][i] b[m][j], a and b checkpoints of the same
// rows, and the column sums of one of them (the bias gradient).  The reduction runs over the rows,
// which are many, so it is split over blocks whose partial sums a second kernel adds in order.
#include <algorithm>

#include "lf_train.h"

namespace lf {

struct GradParams {
  Kept a, b;
  float* partial;               // [splits][a.cols][b.cols], then [splits][cols of the summed one]
  float* colsum;                // or null
  int colsum_of_b;
  int rows_per;                 // rows of one split
  int tiles_b;
};

constexpr int GT = 64;          // tile of the output, either way

// One block: a 64 x 64 tile of one split, 4 x 4 outputs a thread, 16 rows at a time in LDS.
__global__ __launch_bounds__(256) void weight_grad_kernel(GradParams p) {
  __shared__ float A[16][GT + 4], B[16][GT + 4];
  const int ta = blockIdx.x / p.tiles_b, tb = blockIdx.x % p.tiles_b, split = blockIdx.y;
  const int i0 = ta * GT, j0 = tb * GT;
  const long long m0 = (long long)split * p.rows_per, m1 = min((long long)p.a.rows, m0 + p.rows_per);
  const int ti = threadIdx.x / 16 * 4, tj = threadIdx.x % 16 * 4;
  float acc[4][4] = {}, sum = 0.f;
  for (long long m = m0; m < m1; m += 16) {
    const int r = threadIdx.x / 16, c = threadIdx.x % 16 * 4;
    float va[4] = {}, vb[4] = {};
    if (m + r < m1) {
      const size_t row = (size_t)(m + r);
      decode4(*reinterpret_cast<const uint32_t*>(p.a.codes + row * p.a.pitch + i0 + c),
              scale_value(p.a.scales[(size_t)(i0 / GROUP) * p.a.sp + row]), va);
      decode4(*reinterpret_cast<const uint32_t*>(p.b.codes + row * p.b.pitch + j0 + c),
              scale_value(p.b.scales[(size_t)(j0 / GROUP) * p.b.sp + row]), vb);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      A[r][c + k] = va[k];
      B[r][c + k] = vb[k];
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 16; ++q) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(A[q][ti + i], B[q][tj + j], acc[i][j]);
    }
    if (threadIdx.x < GT)
      for (int q = 0; q < 16; ++q) sum += p.colsum_of_b ? B[q][threadIdx.x] : A[q][threadIdx.x];
  }
  float* dst = p.partial + (size_t)split * p.a.cols * p.b.cols;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i0 + ti + i < p.a.cols && j0 + tj + j < p.b.cols) dst[(size_t)(i0 + ti + i) * p.b.cols + j0 + tj + j] = acc[i][j];
  if (p.colsum && threadIdx.x < GT && (p.colsum_of_b ? ta : tb) == 0) {
    const int n = p.colsum_of_b ? p.b.cols : p.a.cols, c = (p.colsum_of_b ? j0 : i0) + threadIdx.x;
    if (c < n) p.colsum[(size_t)split * n + c] = sum;
  }
}

template <int OUT>
__global__ __launch_bounds__(256) void weight_grad_join_kernel(const float* partial, long long n, const float* colsum,
                                                               int cn, int splits, void* out, void* bias) {
  typedef typename Act<OUT>::T T;
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= n + cn) return;
  const float* src = i < n ? partial + i : colsum + (i - n);
  const long long step = i < n ? n : cn;
  float t = 0.f;
  for (int s = 0; s < splits; ++s) t += src[(size_t)s * step];
  if (i < n) Act<OUT>::st(static_cast<T*>(out) + i, t);
  else Act<OUT>::st(static_cast<T*>(bias) + (i - n), t);
}

static int grad_splits(int rows, int ca, int cb) {
  const long long tiles = (long long)((ca + GT - 1) / GT) * ((cb + GT - 1) / GT);
  const long long want = std::max<long long>(1, 1024 / tiles), most = std::max<long long>(1, ((long long)rows + 63) / 64);
  return (int)std::min(want, most);
}

size_t weight_grad_partials(int rows, int outputs, int inputs) {
  return (size_t)grad_splits(rows, outputs, inputs) * ((size_t)outputs * inputs + std::max(outputs, inputs)) * sizeof(float);
}

int run_weight_grad(lf_context* ctx, const Kept& a, const Kept& b, void* out, void* bias, bool bias_of_b, int dt,
                    void* scratch, const char* label) {
  GradParams p{};
  p.a = a;
  p.b = b;
  const int splits = grad_splits(a.rows, a.cols, b.cols);
  const long long n = (long long)a.cols * b.cols;
  p.partial = static_cast<float*>(scratch);
  p.colsum = bias ? p.partial + (size_t)splits * n : nullptr;
  p.colsum_of_b = bias_of_b;
  p.rows_per = (int)((((long long)a.rows + splits - 1) / splits + 15) / 16 * 16);
  p.tiles_b = (b.cols + GT - 1) / GT;
  {
    LaunchScope ls(ctx, label);
    hipLaunchKernelGGL(weight_grad_kernel, dim3((a.cols + GT - 1) / GT * p.tiles_b, splits), dim3(256), 0, ctx->stream, p);
  }
  LF_TRY(check_hip(hipGetLastError(), "weight gradient launch"));
  const int cn = !bias ? 0 : bias_of_b ? b.cols : a.cols;
  LaunchScope ls(ctx, "fp8.weight_grad_join");
  auto k = dt == LF_F32 ? weight_grad_join_kernel<DT_F32> : dt == LF_F16 ? weight_grad_join_kernel<DT_F16>
                                                                         : weight_grad_join_kernel<DT_BF16>;
  hipLaunchKernelGGL(k, dim3((unsigned)((n + cn + 255) / 256)), dim3(256), 0, ctx->stream, p.partial, n, p.colsum, cn,
                     splits, out, bias);
  return check_hip(hipGetLastError(), "weight gradient join launch");
}

}  // namespace lf
