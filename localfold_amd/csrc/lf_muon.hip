// Newton-Schulz products (lf_orthogonalize, lf_muon_step): X <- (a I + b G + c G^2) X with G = X X^T, X scaled
// to a Frobenius norm of one at first, on the orientation that makes G small.
//
// Operands are pairs of f16, v = hi + lo: products hi hi + hi lo + lo hi keep 22 bits of each factor and are summed
// in f32.  A power of two per step and matrix, known from the coefficients alone (muon_plan), keeps hi
// within 2^14 and lo's last bit at 2^-38 of the largest value that the matrix can have, so nothing leaves
// f16's range.  Rounding X to bf16, as is usual, would leave 2^-9 of the largest singular values on the
// small ones, which a run of five steps makes a few hundred times larger.
#include <algorithm>
#include <cmath>

#include "lf_step.h"

namespace lf {

namespace {

// A matrix in scratch: hi and lo, [rows][ld] each, rows and ld multiples of 64, zeros behind the matrix.
struct Planes {
  _Float16 *hi, *lo;
  int ld;
  size_t stride;               // between matrices of the batch
};

struct MuonSize {
  int m, n, mp, np;            // the smaller side, the larger, both rounded up to 64
};

__device__ __forceinline__ void split(float v, _Float16& hi, _Float16& lo) {
  hi = (_Float16)v;
  lo = (_Float16)(v - (float)hi);
}

// u of an element, and its momentum stored.
template <int DT>
__device__ __forceinline__ float muon_u(const Muon& a, size_t i, bool write) {
  const float g = Act<DT>::ld(static_cast<const typename Act<DT>::T*>(a.grad) + i);
  if (!a.momentum) return g;
  float m;
  if (write) {
    m = a.momentum_factor * a.momentum[i] + g;
    a.momentum_out[i] = m;
  } else {
    m = a.momentum_out[i];
  }
  return a.nesterov ? g + a.momentum_factor * m : m;
}

constexpr int NORM_MOST = 64;  // blocks that share a matrix

// Sums of squares, in double: f32's largest values do not overflow it.
template <int DT>
__global__ __launch_bounds__(256) void muon_norm_kernel(Muon a, double* partial) {
  __shared__ double sm[4];
  const long long count = (long long)a.rows * a.cols;
  const size_t base = (size_t)blockIdx.y * count;
  double t = 0;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < count; i += (long long)gridDim.x * 256) {
    const double u = muon_u<DT>(a, base + i, true);
    t += u * u;
  }
  for (int o = 32; o > 0; o >>= 1) t += __shfl_xor(t, o, 64);
  if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = t;
  __syncthreads();
  if (threadIdx.x == 0) partial[blockIdx.y * NORM_MOST + blockIdx.x] = sm[0] + sm[1] + sm[2] + sm[3];
}

// X = u / (|u| + epsilon) times 2^e, as X and as its transpose; one block a tile of 64 x 64.
template <int DT>
__global__ __launch_bounds__(256) void muon_start_kernel(Muon a, MuonSize z, const double* partial, int parts, int e, Planes x,
                                                         Planes xt) {
  __shared__ float tile[64][65];
  double t = 0;
  for (int i = 0; i < parts; ++i) t += partial[blockIdx.z * NORM_MOST + i];
  const double f = 1.0 / (sqrt(t) + a.epsilon);
  const size_t base = (size_t)blockIdx.z * a.rows * a.cols;
  const bool tall = a.rows > a.cols;
  const int i0 = blockIdx.y * 64, j0 = blockIdx.x * 64;     // of X
  const int r0 = tall ? j0 : i0, c0 = tall ? i0 : j0;       // of the stored matrix
  for (int k = threadIdx.x; k < 64 * 64; k += 256) {
    const int r = r0 + (k >> 6), c = c0 + (k & 63);
    float v = 0.f;
    if (r < a.rows && c < a.cols) v = ldexpf((float)(muon_u<DT>(a, base + (size_t)r * a.cols + c, false) * f), e);
    tile[k >> 6][k & 63] = v;
  }
  __syncthreads();
  for (int k = threadIdx.x; k < 64 * 64; k += 256) {
    const int p = k >> 6, q = k & 63;
    // [stored row][stored column] is X's plane where the matrix is wide, its transpose's where it is tall
    const Planes& same = tall ? xt : x;
    const Planes& other = tall ? x : xt;
    const size_t s = blockIdx.z * same.stride + (size_t)(r0 + p) * same.ld + c0 + q;
    split(tile[p][q], same.hi[s], same.lo[s]);
    const size_t o = blockIdx.z * other.stride + (size_t)(c0 + p) * other.ld + r0 + q;
    split(tile[q][p], other.hi[o], other.lo[o]);
  }
}

enum { GRAM = 0, SQUARE = 1, APPLY = 2, LAST = 3 };

struct Product {
  Planes a, b;                 // out[i][j] = sum over k of a[i][k] b[j][k]
  int k;
  Planes out, out_t;           // APPLY: X and its transpose; GRAM, SQUARE: a symmetric matrix
  float f;                     // factor of the sum
  float fb, fa;                // SQUARE: of a's own element, and the diagonal's
};

template <int OUT>
__device__ __forceinline__ void muon_store(const Muon& m, size_t at, float o) {
  typedef typename Act<OUT>::T T;
  float v = -m.rate * o;
  if (m.weight) v = m.keep * Act<OUT>::ld(static_cast<const T*>(m.weight) + at) + v;
  Act<OUT>::st(static_cast<T*>(m.out) + at, v);
}

// A wave computes 32 x 32, a block 64 x 64, operands straight from memory.
template <int KIND, int OUT>
__global__ __launch_bounds__(256) void muon_product_kernel(Product p, Muon m, MuonSize z) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
  if ((KIND == GRAM || KIND == SQUARE) && blockIdx.y > blockIdx.x) return;      // symmetric: the upper tiles, mirrored
  const int i0 = blockIdx.y * 64 + (wave >> 1) * 32, j0 = blockIdx.x * 64 + (wave & 1) * 32;
  const size_t za = blockIdx.z * p.a.stride, zb = blockIdx.z * p.b.stride;
  f4 acc[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) acc[i][j] = f4{0.f, 0.f, 0.f, 0.f};
  for (int k = 0; k < p.k; k += 32) {
    h8 ah[2], al[2], bh[2], bl[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const size_t x = za + (size_t)(i0 + 16 * t + r) * p.a.ld + k + 8 * g;
      const size_t y = zb + (size_t)(j0 + 16 * t + r) * p.b.ld + k + 8 * g;
      ah[t] = *reinterpret_cast<const h8*>(p.a.hi + x);
      al[t] = *reinterpret_cast<const h8*>(p.a.lo + x);
      bh[t] = *reinterpret_cast<const h8*>(p.b.hi + y);
      bl[t] = *reinterpret_cast<const h8*>(p.b.lo + y);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        acc[i][j] = mfma16(al[i], bh[j], acc[i][j]);
        acc[i][j] = mfma16(ah[i], bl[j], acc[i][j]);
        acc[i][j] = mfma16(ah[i], bh[j], acc[i][j]);
      }
  }
#pragma unroll
  for (int ti = 0; ti < 2; ++ti)
#pragma unroll
    for (int tj = 0; tj < 2; ++tj)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = i0 + 16 * ti + 4 * g + e, j = j0 + 16 * tj + r;
        float v = acc[ti][tj][e] * p.f;
        if constexpr (KIND == SQUARE) {
          const size_t at = za + (size_t)i * p.a.ld + j;
          v += p.fb * ((float)p.a.hi[at] + (float)p.a.lo[at]);
          if (i == j) v += p.fa;
        }
        if constexpr (KIND == LAST) {
          if (i >= z.m || j >= z.n) continue;
          const size_t at = m.rows > m.cols ? (size_t)j * m.cols + i : (size_t)i * m.cols + j;
          muon_store<OUT>(m, (size_t)blockIdx.z * m.rows * m.cols + at, v);
        } else {
          const Planes& t = KIND == APPLY ? p.out_t : p.out;
          const size_t at = blockIdx.z * p.out.stride + (size_t)i * p.out.ld + j;
          const size_t tt = blockIdx.z * t.stride + (size_t)j * t.ld + i;
          split(v, p.out.hi[at], p.out.lo[at]);
          // a tile on the diagonal holds both halves itself
          if (KIND == APPLY || blockIdx.x != blockIdx.y) split(v, t.hi[tt], t.lo[tt]);
        }
      }
}

MuonSize muon_size(long long rows, long long cols) {
  const int m = (int)std::min(rows, cols), n = (int)std::max(rows, cols);
  return MuonSize{m, n, (m + 63) / 64 * 64, (n + 63) / 64 * 64};
}

template <int DT>
int start(lf_context* ctx, const Muon& a, const MuonSize& z, double* partial, int e, const Planes& x, const Planes& xt) {
  const long long count = (long long)a.rows * a.cols;
  const int parts = (int)std::min<long long>(NORM_MOST, (count + 4095) / 4096);
  {
    LaunchScope ls(ctx, "muon.norm");
    hipLaunchKernelGGL((muon_norm_kernel<DT>), dim3(parts, a.batch), dim3(256), 0, ctx->stream, a, partial);
  }
  LF_TRY(check_hip(hipGetLastError(), "muon norm launch"));
  LaunchScope ls(ctx, "muon.start");
  hipLaunchKernelGGL((muon_start_kernel<DT>), dim3(z.np / 64, z.mp / 64, a.batch), dim3(256), 0, ctx->stream, a, z, partial, parts,
                     e, x, xt);
  return check_hip(hipGetLastError(), "muon start launch");
}

template <int KIND, int OUT = DT_F32>
int product(lf_context* ctx, const Product& p, const Muon& m, const MuonSize& z, const char* label) {
  const int nx = KIND == GRAM || KIND == SQUARE ? z.mp : z.np;
  LaunchScope ls(ctx, label);
  hipLaunchKernelGGL((muon_product_kernel<KIND, OUT>), dim3(nx / 64, z.mp / 64, m.batch), dim3(256), 0, ctx->stream, p, m, z);
  return check_hip(hipGetLastError(), "muon product launch");
}

size_t up256(size_t n) { return (n + 255) & ~size_t(255); }

}  // namespace

size_t muon_bytes(long long batch, long long rows, long long cols) {
  const MuonSize z = muon_size(rows, cols);
  const size_t x = up256(batch * (size_t)z.mp * z.np * 2), g = up256(batch * (size_t)z.mp * z.mp * 2);
  return up256(batch * NORM_MOST * sizeof(double)) + 8 * x + 4 * g;
}

int run_muon(lf_context* ctx, const Muon& m, const MuonPlan& plan, void* scratch) {
  const MuonSize z = muon_size(m.rows, m.cols);
  char* at = static_cast<char*>(scratch);
  auto take = [&](size_t bytes) {
    void* p = at;
    at += up256(bytes);
    return p;
  };
  double* const partial = static_cast<double*>(take((size_t)m.batch * NORM_MOST * sizeof(double)));
  auto planes = [&](int rows, int ld) {
    Planes p;
    p.stride = (size_t)rows * ld;
    p.ld = ld;
    p.hi = static_cast<_Float16*>(take(m.batch * p.stride * 2));
    p.lo = static_cast<_Float16*>(take(m.batch * p.stride * 2));
    return p;
  };
  Planes x[2] = {planes(z.mp, z.np), planes(z.mp, z.np)}, xt[2] = {planes(z.np, z.mp), planes(z.np, z.mp)};
  const Planes g = planes(z.mp, z.mp), q = planes(z.mp, z.mp);
  if (m.grad_dtype == LF_F32) LF_TRY(start<DT_F32>(ctx, m, z, partial, plan.x[0], x[0], xt[0]));
  else if (m.grad_dtype == LF_F16) LF_TRY(start<DT_F16>(ctx, m, z, partial, plan.x[0], x[0], xt[0]));
  else LF_TRY(start<DT_BF16>(ctx, m, z, partial, plan.x[0], x[0], xt[0]));
  for (int k = 0; k < m.steps; ++k) {
    const float* c = m.coefficients + 3 * k;
    const int ex = plan.x[k], eg = plan.g[k], ep = plan.p[k], now = k & 1;
    Product gram{x[now], x[now], z.np, g, g, std::ldexp(1.f, eg - 2 * ex), 0.f, 0.f};
    LF_TRY(product<GRAM>(ctx, gram, m, z, "muon.gram"));
    Product square{g, g, z.mp, q, q, std::ldexp(c[2], ep - 2 * eg), std::ldexp(c[1], ep - eg), std::ldexp(c[0], ep)};
    LF_TRY(product<SQUARE>(ctx, square, m, z, "muon.square"));
    const bool last = k + 1 == m.steps;
    Product apply{q, xt[now], z.mp, x[!now], xt[!now], std::ldexp(1.f, (last ? 0 : plan.x[k + 1]) - ep - ex), 0.f, 0.f};
    if (!last) LF_TRY(product<APPLY>(ctx, apply, m, z, "muon.apply"));
    else if (m.out_dtype == LF_F32) LF_TRY((product<LAST, DT_F32>(ctx, apply, m, z, "muon.last")));
    else if (m.out_dtype == LF_F16) LF_TRY((product<LAST, DT_F16>(ctx, apply, m, z, "muon.last")));
    else LF_TRY((product<LAST, DT_BF16>(ctx, apply, m, z, "muon.last")));
  }
  return LF_OK;
}

}  // namespace lf
