// The transition's training step, fused for 64 or 128 channels and hidden widths whose weights stay in LDS
// (other widths run as single operators, lf_train.cpp).
//
// A wave takes 32 rows through the whole pass.  A product's output, kept in 8 bits, is the next product's
// operand in the very registers (keep_tile), so nothing between the two products leaves the wave but what
// the backward pass needs.
//
//   forward:  x -> x8, y8 = q(LN(x)); per 128 hidden units h8 = q(relu(y8 W1 + b1)), acc += h8 W2;
//             out = acc + b2 (+ x)
//   backward: d8 = q(dout); per 128 hidden units e8 = q(d8 W2^T where h8 > 0), acc += e8 W1^T = dy;
//             dx = LN's gradient of dy (+ dout), ds and do summed over the block's rows
//
// The forward pass moves 2 b c + 2 c + h bytes a row, the backward 2 b c + 2 c + 2 h: at 5.1 TB/s 37 us and 52 us for
// 147456 rows of 128 x 512 in bf16, which take 70 us and 80 us.  The vector instructions (decoding the weights
// of both products, rounding to codes, the norm) are more than half of the time, the matrix instructions a quarter.
// Run as single operators the two calls take 97 us for 69 and 196 us for 144.  Tiles of 16 rows for the last, partly
// filled turn gained 4 % for this shape, lost 3 % for 207872 rows of 64 x 256, and are not there.
#include <algorithm>

#include "lf_fp8.h"

namespace lf {

constexpr int TW = 8, TM = 2, TROWS = 16 * TM;   // waves of a block, tiles of 16 rows and rows of a wave

struct TrainParams {
  const void* in;               // x, or the gradient of out
  void* out;                    // out, or the gradient of x
  int rows, hidden, accumulate;
  const float *scale, *offset, *b1, *b2;
  float eps;
  int fast_var;
  const uint8_t *w1, *s1, *w2, *s2;   // first and second product's weights, packed [outputs][inputs]
  Kept k1, k2, kh;              // forward: x8, y8, h8 (written); backward: d8, e8 (written), h8 (read)
  Kept kx;                      // backward: x8 (read)
  float *mean, *rstd;
  float* partial;               // backward: [blocks][2][C]
};

// A lane's columns of its rows as storage words: 16 at 16 g, then (C = 128) 16 at 64 + 16 g.
template <int ACT, int C>
struct RowWords {
  static constexpr int NH = C / 64, W = (int)sizeof(typename Act<ACT>::T);
  u32x4 w[TM][NH][W];
  __device__ __forceinline__ float get(int q, int a, int e) const {
    constexpr int per = 16 / W;
    return run_get<ACT>(w[q][a][e / per], e % per);
  }
};

// No condition on the loads: rows past the end repeat the last one.
template <int ACT, int C>
__device__ __forceinline__ void rows_load(RowWords<ACT, C>& x, const void* src, long long m0, int left, int r, int g) {
  typedef RowWords<ACT, C> R;
  const char* base = static_cast<const char*>(src) + (size_t)m0 * C * R::W;
#pragma unroll
  for (int q = 0; q < TM; ++q)
#pragma unroll
    for (int a = 0; a < R::NH; ++a)
#pragma unroll
      for (int v = 0; v < R::W; ++v)
        x.w[q][a][v] = *reinterpret_cast<const u32x4*>(
            base + (uint32_t)(min(TM * r + q, left - 1) * C * R::W + (64 * a + 16 * g) * R::W + 16 * v));
}

// One row's values as codes, the missing half as zeros.
template <int NH>
__device__ __forceinline__ void keep_row(XFrag<TM>& k, int q, const float (&v)[NH][16]) {
  float top = 0.f;
#pragma unroll
  for (int a = 0; a < NH; ++a)
#pragma unroll
    for (int e = 0; e < 16; ++e) top = fmaxf(top, fabsf(v[a][e]));
  const int byte = row_byte(top, [&] {
    float f = 0.f;
#pragma unroll
    for (int a = 0; a < NH; ++a)
#pragma unroll
      for (int e = 0; e < 16; ++e) f = fmaxf(f, fabsf(v[a][e]) < __builtin_inff() ? fabsf(v[a][e]) : 0.f);
    return f;
  });
  const float f = scale_value(byte);
  k.scale |= (uint32_t)byte << (8 * q);
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      if (a < NH) k.v[q][a][b] = encode4(v[a % NH][4 * b], v[a % NH][4 * b + 1], v[a % NH][4 * b + 2], v[a % NH][4 * b + 3], f);
      else k.v[q][a][b] = 0;
    }
}

// Weights of both products and the vectors to LDS.  The first product has `groups` tiles of outputs, the
// second as many of columns.
template <int OUT2, int C>
__device__ __forceinline__ void stage_all(uint8_t* smem, const TrainParams& p, int groups, int wave, int lane) {
  for (int i = wave; i < groups * 32; i += TW) {
    const int tile = i >> 4;
    if (tile < groups) w_stage<OUT_KEPT>(smem + tile * WTILE, p.w1, C, p.hidden, tile, 0, i & 15, lane);
    else w_stage<OUT2>(smem + tile * WTILE, p.w2, p.hidden, C, 0, tile - groups, i & 15, lane);
  }
}

// The weights' scale bytes of up to 4 groups, one byte each.  Loaded once: a load in the loop would have to
// wait for the stores before it.
__device__ __forceinline__ uint32_t scale_word(const uint8_t* s, int groups) {
  uint32_t w = 0;
  for (int i = 0; i < groups; ++i) w |= (uint32_t)s[i] << (8 * i);
  return __builtin_amdgcn_readfirstlane(w);
}

// Tiles of 32 rows of this block, dealt out to its waves in turn.
struct Tiles {
  int first, end;
};
__device__ __forceinline__ Tiles block_tiles(int rows, int wave) {
  const long long tiles = ((long long)rows + TROWS - 1) / TROWS;
  return {(int)(tiles * blockIdx.x / gridDim.x) + wave, (int)(tiles * (blockIdx.x + 1) / gridDim.x)};
}

template <int ACT, int C>
__global__ __launch_bounds__(TW * 64, 2) void train_forward_kernel(TrainParams p) {
  constexpr int NH = C / 64, NT2 = C / 16;
  extern __shared__ __attribute__((aligned(16))) uint8_t train_smem[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int groups = p.hidden / GROUP;
  float* const vec = reinterpret_cast<float*>(train_smem + (size_t)2 * groups * WTILE);   // scale, offset, b2, b1
  stage_all<ACT, C>(train_smem, p, groups, wave, lane);
  for (int i = threadIdx.x; i < C; i += TW * 64) {
    vec[i] = p.scale[i];
    vec[C + i] = p.offset[i];
    vec[2 * C + i] = p.b2 ? p.b2[i] : 0.f;
  }
  for (int i = threadIdx.x; i < p.hidden; i += TW * 64) vec[3 * C + i] = p.b1 ? p.b1[i] : 0.f;
  const uint32_t s1 = scale_word(p.s1, groups), s2 = scale_word(p.s2, groups);
  const Tiles tiles = block_tiles(p.rows, wave);
  RowWords<ACT, C> x;
  auto load = [&](int tile) __attribute__((always_inline)) {
    const long long m0 = (long long)tile * TROWS;
    rows_load<ACT, C>(x, p.in, m0, (int)min((long long)TROWS, p.rows - m0), r, g);
  };
  load(min(tiles.first, tiles.end - 1));
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();

  const int i1 = n_of<OUT_KEPT>(0, r), i2 = n_of<ACT>(0, r);
  const uint8_t* const wa = train_smem + i1 * GROUP + ((g ^ key_of<OUT_KEPT>(i1)) << 4);
  const uint8_t* const wax = train_smem + i1 * GROUP + ((g ^ key_of<OUT_KEPT>(i1) ^ 4) << 4);
  const uint8_t* const wb = train_smem + groups * WTILE + i2 * GROUP + ((g ^ key_of<ACT>(i2)) << 4);
  const uint8_t* const wbx = train_smem + groups * WTILE + i2 * GROUP + ((g ^ key_of<ACT>(i2) ^ 4) << 4);
  LinearParams fin{};           // what finish() reads
  fin.rows = p.rows;
  fin.outputs = C;
  fin.residual = p.accumulate ? p.in : nullptr;
  fin.out = p.out;

  for (int tile = tiles.first; tile < tiles.end; tile += TW) {
    const long long m0 = (long long)tile * TROWS;
    const int left = (int)min((long long)TROWS, p.rows - m0);
    XFrag<TM> x8, y8;
    x8.scale = y8.scale = 0;
    float mean[TM], rstd[TM];
#pragma unroll
    for (int q = 0; q < TM; ++q) {
      __builtin_amdgcn_sched_barrier(0);   // one row of a lane at a time
      float v[NH][16], s = 0.f;
#pragma unroll
      for (int a = 0; a < NH; ++a)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          v[a][e] = x.get(q, a, e);
          s += v[a][e];
        }
      keep_row<NH>(x8, q, v);
      mean[q] = lanes4_sum(s) / C;
      float var = 0.f;
      if (p.fast_var) {
#pragma unroll
        for (int a = 0; a < NH; ++a)
#pragma unroll
          for (int e = 0; e < 16; ++e) var += v[a][e] * v[a][e];
      }
#pragma unroll
      for (int a = 0; a < NH; ++a)
#pragma unroll
        for (int e = 0; e < 16; ++e) v[a][e] -= mean[q];
      if (p.fast_var) {
        var = lanes4_sum(var) / C - mean[q] * mean[q];
        var = var < 0.f ? 0.f : var;
      } else {
#pragma unroll
        for (int a = 0; a < NH; ++a)
#pragma unroll
          for (int e = 0; e < 16; ++e) var += v[a][e] * v[a][e];
        var = lanes4_sum(var) / C;
      }
      rstd[q] = 1.0f / sqrtf(var + p.eps);
#pragma unroll
      for (int a = 0; a < NH; ++a)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const f4 sc = *reinterpret_cast<const f4*>(vec + 64 * a + 16 * g + 4 * b);
          const f4 of = *reinterpret_cast<const f4*>(vec + C + 64 * a + 16 * g + 4 * b);
#pragma unroll
          for (int j = 0; j < 4; ++j) v[a][4 * b + j] = v[a][4 * b + j] * rstd[q] * sc[j] + of[j];
        }
      keep_row<NH>(y8, q, v);
    }
    // the next rows are under way from here on; past the last ones these again, which nothing uses
    if constexpr (ACT != DT_F32) load(min(tile + TW, tiles.end - 1));
    store_kept(x8, p.k1.codes + (size_t)m0 * C, p.k1.scales + m0, C, left, C, r, g);
    store_kept(y8, p.k2.codes + (size_t)m0 * C, p.k2.scales + m0, C, left, C, r, g);
    if (g == 0)
#pragma unroll
      for (int q = 0; q < TM; ++q)
        if (TM * r + q < left) {
          p.mean[m0 + TM * r + q] = mean[q];
          p.rstd[m0 + TM * r + q] = rstd[q];
        }

    f4 acc[NT2][TM];
#pragma unroll
    for (int t = 0; t < NT2; ++t)
#pragma unroll
      for (int q = 0; q < TM; ++q) acc[t][q] = *reinterpret_cast<const f4*>(vec + 2 * C + n_of<ACT>(t, 4 * g));
    for (int hb = 0; hb < groups; ++hb) {
      f4 hid[8][TM];
      mma<OUT_KEPT, true, C == 64>(hid, wa + hb * WTILE, wax + hb * WTILE, y8, s1 >> (8 * hb) & 255, vec + 3 * C + hb * GROUP, g,
                                          [] {});
#pragma unroll
      for (int t = 0; t < 8; ++t)
#pragma unroll
        for (int q = 0; q < TM; ++q)
#pragma unroll
          for (int j = 0; j < 4; ++j) hid[t][q][j] = __builtin_elementwise_maximum(hid[t][q][j], 0.f);   // keeps NaN
      XFrag<TM> h8;
      keep_tile(hid, h8);
      store_kept(h8, p.kh.codes + (size_t)m0 * p.hidden + hb * GROUP, p.kh.scales + (size_t)hb * p.kh.sp + m0, p.hidden,
                 left, GROUP, r, g);
      mma<ACT, false, false>(acc, wb + hb * WTILE, wbx + hb * WTILE, h8, s2 >> (8 * hb) & 255, vec, g, [] {});
    }
    finish<ACT>(acc, fin, m0, 0, r, g);
    if constexpr (ACT == DT_F32) load(min(tile + TW, tiles.end - 1));
  }
}

// v[k] of the first N / 2 plus v[k + N / 2] of the rest: lanes whose bit is clear keep the sums of the first
// half over them and the lane that the permute pairs them with, the others those of the second half.
template <int CTRL, int N, int M>
__device__ __forceinline__ void halve(float (&v)[M], bool upper) {
#pragma unroll
  for (int k = 0; k < N / 2; ++k) {
    const float a = v[k] + dpp_f<CTRL>(v[k]), b = v[k + N / 2] + dpp_f<CTRL>(v[k + N / 2]);
    v[k] = upper ? b : a;
  }
}

template <int ACT, int C>
__global__ __launch_bounds__(TW * 64, 2) void train_backward_kernel(TrainParams p) {
  constexpr int NH = C / 64, NT2 = C / 16;
  extern __shared__ __attribute__((aligned(16))) uint8_t train_smem[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int groups = p.hidden / GROUP;
  float* const vec = reinterpret_cast<float*>(train_smem + (size_t)2 * groups * WTILE);   // scale, zeros, [TW][2][C] sums
  stage_all<OUT_KEPT, C>(train_smem, p, groups, wave, lane);
  for (int i = threadIdx.x; i < C; i += TW * 64) vec[i] = p.scale[i];
  for (int i = threadIdx.x; i < GROUP; i += TW * 64) vec[C + i] = 0.f;
  float* const sums = vec + C + GROUP;
  const uint32_t s1 = scale_word(p.s1, groups), s2 = scale_word(p.s2, groups);
  const Tiles tiles = block_tiles(p.rows, wave);
  RowWords<ACT, C> x;
  auto load = [&](int tile) __attribute__((always_inline)) {
    const long long m0 = (long long)tile * TROWS;
    rows_load<ACT, C>(x, p.in, m0, (int)min((long long)TROWS, p.rows - m0), r, g);
  };
  load(min(tiles.first, tiles.end - 1));
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();

  const int i1 = n_of<OUT_KEPT>(0, r);
  const uint8_t* const wa = train_smem + i1 * GROUP + ((g ^ key_of<OUT_KEPT>(i1)) << 4);
  const uint8_t* const wax = train_smem + i1 * GROUP + ((g ^ key_of<OUT_KEPT>(i1) ^ 4) << 4);
  f4 total = {0.f, 0.f, 0.f, 0.f};

  for (int tile = tiles.first; tile < tiles.end; tile += TW) {
    const long long m0 = (long long)tile * TROWS;
    const int left = (int)min((long long)TROWS, p.rows - m0);
    XFrag<TM> d8;
    d8.scale = 0;
#pragma unroll
    for (int q = 0; q < TM; ++q) {
      __builtin_amdgcn_sched_barrier(0);   // one row of a lane at a time
      float v[NH][16];
#pragma unroll
      for (int a = 0; a < NH; ++a)
#pragma unroll
        for (int e = 0; e < 16; ++e) v[a][e] = x.get(q, a, e);
      keep_row<NH>(d8, q, v);
    }
    store_kept(d8, p.k1.codes + (size_t)m0 * C, p.k1.scales + m0, C, left, C, r, g);

    f4 dy[NT2][TM];
#pragma unroll
    for (int t = 0; t < NT2; ++t)
#pragma unroll
      for (int q = 0; q < TM; ++q) dy[t][q] = f4{0.f, 0.f, 0.f, 0.f};
    u32x4 gate[TM][2];
    auto load_gate = [&](int hb) __attribute__((always_inline)) {
#pragma unroll
      for (int q = 0; q < TM; ++q)
#pragma unroll
        for (int a = 0; a < 2; ++a)
          gate[q][a] = *reinterpret_cast<const u32x4*>(
              p.kh.codes + (size_t)m0 * p.hidden + hb * GROUP +
              (uint32_t)(__umul24(min(TM * r + q, left - 1), p.hidden) + 64 * a + 16 * g));
    };
    load_gate(0);
    for (int hb = 0; hb < groups; ++hb) {
      f4 e[8][TM];
      mma<OUT_KEPT, true, C == 64>(e, wa + hb * WTILE, wax + hb * WTILE, d8, s1 >> (8 * hb) & 255, vec + C, g, [] {});
#pragma unroll
      for (int t = 0; t < 8; ++t)
#pragma unroll
        for (int q = 0; q < TM; ++q) gate4(e[t][q], gate[q][t >> 2][t & 3]);
      load_gate(min(hb + 1, groups - 1));     // before the stores, which its wait would be for too
      XFrag<TM> e8;
      keep_tile(e, e8);
      store_kept(e8, p.k2.codes + (size_t)m0 * p.hidden + hb * GROUP, p.k2.scales + (size_t)hb * p.k2.sp + m0, p.hidden,
                 left, GROUP, r, g);
      const int at = (groups + hb) * WTILE;
      mma<OUT_KEPT, false, false>(dy, wa + at, wax + at, e8, s2 >> (8 * hb) & 255, vec, g, [] {});
    }

    // LayerNorm's gradient: a lane has columns 64 a + 16 g + 4 b + j of its rows in dy[4 a + b][q][j]
    float sv[2 * C / 4];        // its columns' ds, then do
#pragma unroll
    for (int k = 0; k < C / 2; ++k) sv[k] = 0.f;
    load(tile);                 // the gradient again, for the residual
#pragma unroll
    for (int q = 0; q < TM; ++q) {
      __builtin_amdgcn_sched_barrier(0);
      const int row = min(TM * r + q, left - 1);
      const float mean = p.mean[m0 + row], rstd = p.rstd[m0 + row];
      const float xs = scale_value(p.kx.scales[m0 + row]);
      u32x4 xc[NH];
#pragma unroll
      for (int a = 0; a < NH; ++a)
        xc[a] = *reinterpret_cast<const u32x4*>(p.kx.codes + (size_t)m0 * C + (uint32_t)(row * C + 64 * a + 16 * g));
      if (TM * r + q >= left) {
#pragma unroll
        for (int t = 0; t < NT2; ++t) dy[t][q] = f4{0.f, 0.f, 0.f, 0.f};
      }
      float h[NH][16], sa = 0.f, sb = 0.f;
#pragma unroll
      for (int a = 0; a < NH; ++a)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          decode4(xc[a][b], xs, h[a] + 4 * b);
          const f4 sc = *reinterpret_cast<const f4*>(vec + 64 * a + 16 * g + 4 * b);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float d = dy[4 * a + b][q][j], hh = (h[a][4 * b + j] - mean) * rstd;
            h[a][4 * b + j] = hh;
            sv[16 * a + 4 * b + j] += d * hh;
            sv[C / 4 + 16 * a + 4 * b + j] += d;
            const float gd = d * sc[j];
            dy[4 * a + b][q][j] = gd;
            sa += gd;
            sb += gd * hh;
          }
        }
      sa = lanes4_sum(sa) / C;
      sb = lanes4_sum(sb) / C;
#pragma unroll
      for (int a = 0; a < NH; ++a)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          float o = rstd * (dy[4 * a + e / 4][q][e % 4] - sa - h[a][e] * sb);
          if (p.accumulate) o += x.get(q, a, e);
          h[a][e] = o;
        }
      if (TM * r + q < left) {
        typedef RowWords<ACT, C> R;
        char* dst = static_cast<char*>(p.out) + (size_t)m0 * C * R::W + (uint32_t)((TM * r + q) * C * R::W + 16 * g * R::W);
        constexpr int E = 4 / R::W;
#pragma unroll
        for (int a = 0; a < NH; ++a)
#pragma unroll
          for (int v = 0; v < R::W; ++v) {
            u32x4 w;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int e = (4 * v + k) * E;
              w[k] = run_word<ACT>(h[a][e], h[a][e + E - 1]);
            }
            *reinterpret_cast<u32x4*>(dst + 64 * a * R::W + 16 * v) = w;
          }
      }
    }
    load(min(tile + TW, tiles.end - 1));     // past the last rows these again, which nothing uses

    // the columns' sums over the 16 lanes that share them, which end with four of them each
    halve<0x140, C / 2>(sv, r & 8);          // row mirror: ds or do
    halve<0x141, C / 4>(sv, r & 4);          // half mirror
    halve<0x1B, C / 8>(sv, r & 2);           // quad [3,2,1,0]
    if constexpr (C == 128) {
      halve<0xB1, C / 16>(sv, r & 1);        // quad [1,0,3,2]
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) sv[k] += dpp_f<0xB1>(sv[k]);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) total[k] += sv[k];
  }

  // C = 128: bit 3 of r says ds or do, bit 2 the half a, bits 1 and 0 b; C = 64: bit 3, then b in bits 2 and 1
  const int col = C == 128 ? 64 * ((r >> 2) & 1) + 16 * g + 4 * (r & 3) : 16 * g + 4 * ((r >> 1) & 3);
  if (C == 128 || (r & 1) == 0) *reinterpret_cast<f4*>(sums + (wave * 2 + (r >> 3)) * C + col) = total;
  __syncthreads();
  for (int c = threadIdx.x; c < 2 * C; c += TW * 64) {
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < TW; ++w) t += sums[w * 2 * C + c];
    p.partial[(size_t)blockIdx.x * 2 * C + c] = t;
  }
}

namespace {

int train_blocks(const lf_context* ctx, int rows) {
  // a tile for every SIMD before a second one
  return (int)std::min<long long>(((long long)rows + TROWS * 4 - 1) / (TROWS * 4), ctx->num_cus);
}

template <int ACT, int C>
int go(lf_context* ctx, const TrainParams& p, bool backward) {
  static const bool lds = [] {
    bool ok = true;
    for (auto k : {&train_forward_kernel<ACT, C>, &train_backward_kernel<ACT, C>})
      ok = ok && hipFuncSetAttribute(reinterpret_cast<const void*>(k), hipFuncAttributeMaxDynamicSharedMemorySize,
                                     160 * 1024) == hipSuccess;
    return ok;
  }();
  if (!lds) return set_error(LF_ERR_DEVICE, "transition training: the device refuses the LDS it needs");
  const size_t smem = (size_t)2 * (p.hidden / GROUP) * WTILE +
                      sizeof(float) * (backward ? C + GROUP + TW * 2 * C : 3 * C + p.hidden);
  hipLaunchKernelGGL((backward ? &train_backward_kernel<ACT, C> : &train_forward_kernel<ACT, C>),
                     dim3(train_blocks(ctx, p.rows)), dim3(TW * 64), smem, ctx->stream, p);
  return check_hip(hipGetLastError(), "transition training launch");
}
int go(lf_context* ctx, const TrainParams& p, int dt, int c, bool backward) {
  if (c == 64)
    return dt == LF_F32   ? go<DT_F32, 64>(ctx, p, backward)
           : dt == LF_F16 ? go<DT_F16, 64>(ctx, p, backward)
                          : go<DT_BF16, 64>(ctx, p, backward);
  return dt == LF_F32   ? go<DT_F32, 128>(ctx, p, backward)
         : dt == LF_F16 ? go<DT_F16, 128>(ctx, p, backward)
                        : go<DT_BF16, 128>(ctx, p, backward);
}

}  // namespace

// 128 KB of weight tiles, and whole groups of hidden units; rows of 16-byte pieces.
bool train_fused(int channels, int hidden, const void* in, const void* out) {
  return (channels == 64 || channels == 128) && hidden % GROUP == 0 && hidden <= 4 * GROUP &&
         ((reinterpret_cast<uintptr_t>(in) | reinterpret_cast<uintptr_t>(out)) & 15) == 0;
}

int run_train_forward(lf_context* ctx, const lf_transition_train_args& a, const lf_fp8_weight& w1, const lf_fp8_weight& w2) {
  TrainParams p{};
  p.in = a.act;
  p.out = a.out;
  p.rows = a.rows;
  p.hidden = a.hidden;
  p.accumulate = a.accumulate;
  p.scale = a.w->norm_scale;
  p.offset = a.w->norm_offset;
  p.b1 = a.w->b1;
  p.b2 = a.w->b2;
  p.eps = a.epsilon;
  p.fast_var = a.fast_variance;
  p.w1 = static_cast<const uint8_t*>(w1.codes);
  p.s1 = static_cast<const uint8_t*>(w1.scales);
  p.w2 = static_cast<const uint8_t*>(w2.codes);
  p.s2 = static_cast<const uint8_t*>(w2.scales);
  p.k1 = kept_view(a.saved->act);
  p.k2 = kept_view(a.saved->normed);
  p.kh = kept_view(a.saved->hidden);
  p.mean = a.saved->mean;
  p.rstd = a.saved->rstd;
  LaunchScope ls(ctx, "forward");
  return go(ctx, p, a.act_dtype, a.channels, false);
}

size_t train_partials(int channels) { return (size_t)512 * 2 * channels * sizeof(float); }   // a block a CU at most

int run_train_backward(lf_context* ctx, const lf_transition_backward_args& a, const lf_fp8_weight& w2,
                       const lf_fp8_weight& w1, const Kept& d, const Kept& e, float* partial) {
  TrainParams p{};
  p.in = a.grad;
  p.out = a.out;
  p.rows = a.rows;
  p.hidden = a.hidden;
  p.accumulate = a.accumulate;
  p.scale = a.w->norm_scale;
  p.w1 = static_cast<const uint8_t*>(w2.codes);      // the first product of the backward pass is W2's
  p.s1 = static_cast<const uint8_t*>(w2.scales);
  p.w2 = static_cast<const uint8_t*>(w1.codes);
  p.s2 = static_cast<const uint8_t*>(w1.scales);
  p.k1 = d;
  p.k2 = e;
  p.kh = kept_view(a.saved->hidden);
  p.kx = kept_view(a.saved->act);
  p.mean = a.saved->mean;
  p.rstd = a.saved->rstd;
  p.partial = partial;
  LF_REQUIRE(train_blocks(ctx, a.rows) <= 512, "transition training: more than 512 compute units");
  {
    LaunchScope ls(ctx, "backward");
    LF_TRY(go(ctx, p, a.act_dtype, a.channels, true));
  }
  return run_norm_join(ctx, partial, train_blocks(ctx, a.rows), a.channels, a.grad_norm_scale, a.grad_norm_offset, a.grad_dtype);
}

}  // namespace lf
