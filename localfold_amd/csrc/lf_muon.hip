// Newton-Schulz products (lf_orthogonalize, lf_muon_step): X <- (a I + b G + c G^2) X with G = X X^T, X scaled
// to a Frobenius norm of one at first, on the orientation that makes G small (m x m, X m x n).
//
// Operands are pairs of f16, v = hi + lo: products hi hi + hi lo + lo hi keep 22 bits of each factor and are summed
// in f32.  A power of two per step and matrix, known from the coefficients alone (muon_plan), keeps hi
// within 2^14 and lo's last bit at 2^-38 of the largest value that the matrix can have, so nothing leaves
// f16's range.  Rounding X to bf16, as is usual, would leave 2^-9 of the largest singular values on the
// small ones, which a run of five steps makes a few hundred times larger.
//
// Fragments.  An operand is kept as fragments of 16 rows by 32 of the contraction, as the instruction takes
// them: lane (r, g) = (lane % 16, lane / 16) has row r and eight k.  Which eight is free, as long as both
// operands agree: k = 16 (e / 4) + 4 g + e % 4 for e < 8.  A product's result has, in lane (r, g), rows 4 g + e of
// column r of a tile of 16 x 16, so two tiles one above the other are, as they lie in registers, a fragment
// of the result's transpose; for a symmetric result, of the result itself.  The other order, where it is needed,
// comes from a product with the identity, which is exact.
#include <algorithm>
#include <cmath>

#include "lf_step.h"

namespace lf {

namespace {

struct MuonSize {
  int m, n;                    // the smaller side, the larger
};

__device__ __forceinline__ f4 mfma_pair(h8 ah, h8 al, h8 bh, h8 bl, f4 c) {
  c = mfma16(al, bh, c);
  c = mfma16(ah, bl, c);
  return mfma16(ah, bh, c);
}

// Four values into half `part` of a pair of fragments.  The empty assembly makes the compiler pack pairs at once: kept
// apart until they are used, they would take twice the registers.
__device__ __forceinline__ void split4(f4 v, h8& hi, h8& lo, int part) {
  u32x4 h = __builtin_bit_cast(u32x4, hi), l = __builtin_bit_cast(u32x4, lo);
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const h2 p = h2{(_Float16)v[2 * e], (_Float16)v[2 * e + 1]};
    const h2 q = h2{(_Float16)(v[2 * e] - (float)p[0]), (_Float16)(v[2 * e + 1] - (float)p[1])};
    uint32_t a = __builtin_bit_cast(uint32_t, p), b = __builtin_bit_cast(uint32_t, q);
    asm volatile("" : "+v"(a), "+v"(b));
    h[2 * part + e] = a;
    l[2 * part + e] = b;
  }
  hi = __builtin_bit_cast(h8, h);
  lo = __builtin_bit_cast(h8, l);
}

// The fragment of the identity that takes half `part` of a fragment's k to columns.
__device__ __forceinline__ h8 identity(int part, int r, int g) {
  h8 v;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = (_Float16)((e >> 2) == part && r == 4 * g + (e & 3) ? 1.f : 0.f);
  return v;
}
// Fragment f (16 rows, 32 k) transposed: half `part` of its k, 16 of them, by its 16 rows, as half of a fragment.
__device__ __forceinline__ h4 turn(h8 f, h8 eye) {
  const f4 d = mfma16(f, eye, f4{0.f, 0.f, 0.f, 0.f});
  return h4{(_Float16)d[0], (_Float16)d[1], (_Float16)d[2], (_Float16)d[3]};
}

// u of an element, from the momentum that is already the new one.
template <int DT>
__device__ __forceinline__ float muon_u(const Muon& a, size_t i) {
  const float g = Act<DT>::ld(static_cast<const typename Act<DT>::T*>(a.grad) + i);
  if (!a.momentum) return g;
  return a.nesterov ? g + a.momentum_factor * a.momentum_out[i] : a.momentum_out[i];
}

// The place of X's element (i, j) in the stored matrix.
__device__ __forceinline__ size_t place(const Muon& a, int i, int j) {
  return a.rows > a.cols ? (size_t)j * a.cols + i : (size_t)i * a.cols + j;
}

// Rows i to i + 3 of column j of X, in one access where they lie side by side.
template <int DT>
__device__ __forceinline__ f4 muon_u4(const Muon& a, const MuonSize& z, size_t base, int i, int j) {
  typedef typename Act<DT>::T T;
  f4 v = {0.f, 0.f, 0.f, 0.f};
  if (j >= z.n) return v;
  if (a.rows > a.cols && i + 4 <= z.m) {
    struct Vec { T v[4]; } gv;
    f4 mv = v;
    const size_t at = base + place(a, i, j);
    __builtin_memcpy(&gv, static_cast<const T*>(a.grad) + at, sizeof(gv));
    if (a.momentum) __builtin_memcpy(&mv, a.momentum_out + at, 16);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float g = Act<DT>::ld(gv.v + e);
      v[e] = !a.momentum ? g : a.nesterov ? g + a.momentum_factor * mv[e] : mv[e];
    }
    return v;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (i + e < z.m) v[e] = muon_u<DT>(a, base + place(a, i + e, j));
  return v;
}

template <int OUT>
__device__ __forceinline__ void muon_store4(const Muon& m, const MuonSize& z, size_t base, int i, int j, f4 o) {
  typedef typename Act<OUT>::T T;
  if (j >= z.n) return;
  struct Vec { T v[4]; } w;
  const size_t at = base + place(m, i, j), step = m.rows > m.cols ? 1 : m.cols;
  const T* const weight = static_cast<const T*>(m.weight) + at;
  T* const out = static_cast<T*>(m.out) + at;
  const bool whole = m.rows > m.cols && i + 4 <= z.m;
  if (m.weight && whole) __builtin_memcpy(&w, weight, sizeof(w));
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (i + e >= z.m) continue;
    float v = -m.rate * o[e];
    if (m.weight) v = m.keep * Act<OUT>::ld(whole ? w.v + e : weight + e * step) + v;
    Act<OUT>::st(whole ? w.v + e : out + e * step, v);
  }
  if (whole) __builtin_memcpy(out, &w, sizeof(w));
}

// ---- one block a matrix --------------------------------------------------------------------------

// m to 128 and n to 512: a block runs all steps.  Each of its 8 waves keeps J tiles of 16 columns of X, all rows, in
// registers, as fragments of X^T: the operand of P X, whose result is the next X^T in place.  G takes X by rows: J
// times the waves turn a tile each, 128 columns together, and put it into LDS, and all add to their tiles of G.  G
// and then P are in LDS.  MB: m in 32s.
// Bound by a step's chain of products, LDS and barriers on one CU: 3.8 us a step for 64 x 256 and 12 once, 18.6 and 45 for
// 128 x 512.
template <int MB>
struct MuonTiles {               // a wave's tiles of G: A by B of MT by MT
  static constexpr int MT = 2 * MB, A = MB == 4 ? 2 : 1, B = MB == 4 ? 4 : MB == 2 ? 2 : 1, ACROSS = MT / B;
};

struct MuonSteps {
  float gram[MUON_STEPS], square[MUON_STEPS], gb[MUON_STEPS], diagonal[MUON_STEPS], apply[MUON_STEPS];
  int count, start, end;       // X's first and last exponent
};

// The stored matrix passes through LDS, JW tiles a wave at a time, so that memory is read and written in whole lines.
// Rows of LDS are 4 columns longer than the matrix's: lanes g then start 16 banks apart.
template <int MB, int J>
struct MuonRegion {
  static constexpr int JW = J < 2 ? J : 2, W = 128 * JW;         // columns of X at a time
  static constexpr int BYTES = 4 * (32 * MB * (W + 4) > W * (32 * MB + 4) ? 32 * MB * (W + 4) : W * (32 * MB + 4));
  bool tall;
  int pitch, m, n, ld;
  int width;                   // columns of X that exist, from the first of these on
  int rows, cols;              // of the stored matrix
  uint32_t first;
  __device__ __forceinline__ MuonRegion(const Muon& a, const MuonSize& z)
      : tall(a.rows > a.cols), pitch(tall ? 32 * MB + 4 : W + 4), m(z.m), n(z.n), ld(a.cols) {}
  __device__ __forceinline__ void at(int j0) {
    width = max(0, min(W, n - 128 * j0));
    rows = tall ? width : m;
    cols = tall ? m : width;
    first = 128 * j0 * (tall ? ld : 1);
  }
};

// A thread's items of rows of `per`, 512 apart.
struct MuonWalk {
  int per, row, col, rows, cols;
  __device__ __forceinline__ explicit MuonWalk(int n) : per(max(n, 1)), rows(512 / per), cols(512 % per) {
    row = threadIdx.x / per;
    col = threadIdx.x % per;
  }
  __device__ __forceinline__ void next() {
    row += rows;
    col += cols;
    if (col >= per) {
      col -= per;
      ++row;
    }
  }
};

// Reads u, V elements a lane side by side, stores the momentum (AGAIN: it is the new one already) and puts u into LDS; the
// sum of squares.
template <int DT, int V, bool AGAIN, class R>
__device__ __forceinline__ double muon_take(const Muon& a, const R& in, size_t base, float* tile) {
  typedef typename Act<DT>::T T;
  struct Vec { T v[V]; };
  struct VecF { float v[V]; };
  constexpr int BATCH = 8;     // loads under way
  const int items = in.rows * (in.cols / V);
  MuonWalk walk(in.cols / V);
  const T* const grad = static_cast<const T*>(a.grad) + base + in.first;
  const float* const old = (AGAIN ? a.momentum_out : a.momentum) + base + in.first;
  float* const now = a.momentum_out + base + in.first;
  double t = 0;
  for (int i0 = 0; i0 < items; i0 += 512 * BATCH) {
    Vec gv[BATCH];
    VecF mv[BATCH];
    int row[BATCH], col[BATCH];
    bool there[BATCH];
#pragma unroll
    for (int k = 0; k < BATCH; ++k) {
      there[k] = walk.row < in.rows;
      row[k] = there[k] ? walk.row : 0;
      col[k] = walk.col * V;
      walk.next();
      const uint32_t at = row[k] * in.ld + col[k];
      __builtin_memcpy(&gv[k], grad + at, sizeof(Vec));
      if (a.momentum) __builtin_memcpy(&mv[k], old + at, sizeof(VecF));
    }
#pragma unroll
    for (int k = 0; k < BATCH; ++k) {
      if (!there[k]) continue;
      VecF u;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        u.v[e] = Act<DT>::ld(gv[k].v + e);
        if (a.momentum) {
          if (!AGAIN) mv[k].v[e] = a.momentum_factor * mv[k].v[e] + u.v[e];
          u.v[e] = a.nesterov ? u.v[e] + a.momentum_factor * mv[k].v[e] : mv[k].v[e];
        }
        t += (double)u.v[e] * u.v[e];
      }
      if (!AGAIN && a.momentum) __builtin_memcpy(now + (row[k] * in.ld + col[k]), &mv[k], sizeof(VecF));
      __builtin_memcpy(tile + row[k] * in.pitch + col[k], &u, sizeof(VecF));
    }
  }
  return t;
}

// The output of what LDS holds.
template <int OUT, int V, class R>
__device__ __forceinline__ void muon_give(const Muon& a, const R& in, size_t base, const float* tile) {
  typedef typename Act<OUT>::T T;
  struct Vec { T v[V]; };
  struct VecF { float v[V]; };
  constexpr int BATCH = 8;
  const int items = in.rows * (in.cols / V);
  MuonWalk walk(in.cols / V);
  const T* const weight = static_cast<const T*>(a.weight) + base + in.first;
  T* const out = static_cast<T*>(a.out) + base + in.first;
  for (int i0 = 0; i0 < items; i0 += 512 * BATCH) {
    Vec w[BATCH];
    int row[BATCH], col[BATCH];
    bool there[BATCH];
#pragma unroll
    for (int k = 0; k < BATCH; ++k) {
      there[k] = walk.row < in.rows;
      row[k] = there[k] ? walk.row : 0;
      col[k] = walk.col * V;
      walk.next();
      if (a.weight) __builtin_memcpy(&w[k], weight + (row[k] * in.ld + col[k]), sizeof(Vec));
    }
#pragma unroll
    for (int k = 0; k < BATCH; ++k) {
      if (!there[k]) continue;
      VecF o;
      __builtin_memcpy(&o, tile + row[k] * in.pitch + col[k], sizeof(VecF));
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float v = -a.rate * o.v[e];
        Act<OUT>::st(w[k].v + e, a.weight ? a.keep * Act<OUT>::ld(w[k].v + e) + v : v);
      }
      __builtin_memcpy(out + (row[k] * in.ld + col[k]), &w[k], sizeof(Vec));
    }
  }
}

// What a wave of a block does in a step; its tiles of G begin at (ta, tb).
template <int MB>
struct MuonCore {
  typedef MuonTiles<MB> Q;
  typedef f4 Tiles[Q::A][Q::B];
  uint8_t *xs, *gs;            // X by rows, 128 columns: [tile][32 columns][hi, lo]; G or P: [tile][32 rows][hi, lo]
  int wave, lane, ta, tb;
  bool mine;
  __device__ __forceinline__ MuonCore(uint8_t* smem, int wave_, int lane_)
      : xs(smem), gs(smem + Q::MT * 4 * 2048), wave(wave_), lane(lane_), ta(wave_ / Q::ACROSS * Q::A), tb(wave_ % Q::ACROSS * Q::B),
        mine(wave_ / Q::ACROSS * Q::A < Q::MT) {}

  static __device__ __forceinline__ void clear(Tiles& v) {
#pragma unroll
    for (int i = 0; i < Q::A; ++i)
#pragma unroll
      for (int k = 0; k < Q::B; ++k) v[i][k] = f4{0.f, 0.f, 0.f, 0.f};
  }
  // The wave's 16 columns by rows into LDS.
  __device__ __forceinline__ void turn_columns(const h8 (&xh)[MB], const h8 (&xl)[MB], const h8 (&eye)[2]) const {
#pragma unroll
    for (int kb = 0; kb < MB; ++kb)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        __builtin_amdgcn_sched_barrier(0);
        uint8_t* const at = xs + ((2 * kb + h) * 4 + (wave >> 1)) * 2048 + lane * 16 + 8 * (wave & 1);
        *reinterpret_cast<h4*>(at) = turn(xh[kb], eye[h]);
        *reinterpret_cast<h4*>(at + 1024) = turn(xl[kb], eye[h]);
      }
  }
  // v += the product of `from`, KBS fragments a row, with its own transpose.
  template <int KBS>
  __device__ __forceinline__ void times_itself(Tiles& v, const uint8_t* from) const {
#pragma unroll
    for (int kb = 0; kb < KBS; ++kb) {
      __builtin_amdgcn_sched_barrier(0);     // or all fragments would be read at once, and spill
      h8 ah[Q::A], al[Q::A];
#pragma unroll
      for (int i = 0; i < Q::A; ++i) {
        const uint8_t* const at = from + ((ta + i) * KBS + kb) * 2048 + lane * 16;
        ah[i] = *reinterpret_cast<const h8*>(at);
        al[i] = *reinterpret_cast<const h8*>(at + 1024);
      }
#pragma unroll
      for (int k = 0; k < Q::B; ++k) {
        const uint8_t* const at = from + ((tb + k) * KBS + kb) * 2048 + lane * 16;
        const h8 bh = *reinterpret_cast<const h8*>(at), bl = *reinterpret_cast<const h8*>(at + 1024);
#pragma unroll
        for (int i = 0; i < Q::A; ++i) v[i][k] = mfma_pair(ah[i], al[i], bh, bl, v[i][k]);
      }
    }
  }
  // A symmetric tile (ta + i, tb + k) in its place: rows of tile tb + k, k of tile ta + i.
  __device__ __forceinline__ void put(const Tiles& v) const {
#pragma unroll
    for (int k = 0; k < Q::B; ++k)
#pragma unroll
      for (int i = 0; i < Q::A; ++i) {
        __builtin_amdgcn_sched_barrier(0);
        h8 hi, lo;
        split4(v[i][k], hi, lo, 0);
        uint8_t* const at = gs + ((tb + k) * MB + (ta + i) / 2) * 2048 + lane * 16 + 8 * ((ta + i) & 1);
        *reinterpret_cast<h4*>(at) = h4{hi[0], hi[1], hi[2], hi[3]};
        *reinterpret_cast<h4*>(at + 1024) = h4{lo[0], lo[1], lo[2], lo[3]};
      }
  }
  // From G's tiles, as summed, to P in LDS; every wave has read what was in gs.
  __device__ __forceinline__ void to_p(Tiles& gram, const MuonSteps& steps, int s) const {
    if (mine) {
#pragma unroll
      for (int i = 0; i < Q::A; ++i)
#pragma unroll
        for (int k = 0; k < Q::B; ++k) gram[i][k] *= steps.gram[s];
      put(gram);
    }
    __syncthreads();
    Tiles p;
    clear(p);
    if (mine) {
      times_itself<MB>(p, gs);
      const int r = lane & 15, g = lane >> 4;
#pragma unroll
      for (int i = 0; i < Q::A; ++i)
#pragma unroll
        for (int k = 0; k < Q::B; ++k) {
          p[i][k] = p[i][k] * steps.square[s] + gram[i][k] * steps.gb[s];
          if (ta + i == tb + k)
#pragma unroll
            for (int e = 0; e < 4; ++e) p[i][k][e] += r == 4 * g + e ? steps.diagonal[s] : 0.f;
        }
    }
    __syncthreads();          // G is read
    if (mine) put(p);
    __syncthreads();
  }
  // J of the wave's column tiles times P, in place; they share the reads of P.
  template <int J>
  __device__ __forceinline__ void apply(h8 (*xh)[MB], h8 (*xl)[MB], float factor) const {
    f4 y[J][Q::MT];
#pragma unroll
    for (int t = 0; t < Q::MT; ++t) {
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int q = 0; q < J; ++q) y[q][t] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kb = 0; kb < MB; ++kb) {
        const uint8_t* const at = gs + (t * MB + kb) * 2048 + lane * 16;
        const h8 ph = *reinterpret_cast<const h8*>(at), pl = *reinterpret_cast<const h8*>(at + 1024);
#pragma unroll
        for (int q = 0; q < J; ++q) y[q][t] = mfma_pair(ph, pl, xh[q][kb], xl[q][kb], y[q][t]);
      }
    }
#pragma unroll
    for (int q = 0; q < J; ++q)
#pragma unroll
      for (int t = 0; t < Q::MT; ++t) {
        __builtin_amdgcn_sched_barrier(0);
        split4(y[q][t] * factor, xh[q][t / 2], xl[q][t / 2], t & 1);
      }
  }
};

template <int MB, int J, int DT, int OUT>
__global__ __launch_bounds__(512, 2) void muon_block_kernel(Muon a, MuonSize z, MuonSteps steps) {
  extern __shared__ __attribute__((aligned(16))) uint8_t muon_smem[];
  __shared__ double norm[8];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  int r = lane & 15, g = lane >> 4;
  const size_t base = (size_t)blockIdx.x * a.rows * a.cols;
  h8 xh[J][MB], xl[J][MB];
  MuonRegion<MB, J> in(a, z);
  {
    float u[J][MB][8];
    double t = 0;
#pragma unroll
    for (int j0 = 0; j0 < J; j0 += in.JW) {
      if (j0 > 0) __syncthreads();         // the last columns are read
      in.at(j0);
      float* const tile = reinterpret_cast<float*>(muon_smem);
      if (a.cols % 4 == 0) t += muon_take<DT, 4, false>(a, in, base, tile);
      else t += muon_take<DT, 1, false>(a, in, base, tile);
      __syncthreads();
#pragma unroll
      for (int j = 0; j < in.JW; ++j) {
        const int c = 16 * (8 * j + wave) + r;
#pragma unroll
        for (int kb = 0; kb < MB; ++kb)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int i = 32 * kb + 16 * (e >> 2) + 4 * g + (e & 3);
            const float v = tile[in.tall ? c * in.pitch + i : i * in.pitch + c];
            u[j0 + j][kb][e] = i < z.m && c < in.width ? v : 0.f;
          }
      }
    }
    for (int o = 32; o > 0; o >>= 1) t += __shfl_xor(t, o, 64);
    if (lane == 0) norm[wave] = t;
    __syncthreads();
    t = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) t += norm[i];
    const double f = 1.0 / (sqrt(t) + a.epsilon);
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int kb = 0; kb < MB; ++kb)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          __builtin_amdgcn_sched_barrier(0);
          f4 v;
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = ldexpf((float)(u[j][kb][4 * h + e] * f), steps.start);
          split4(v, xh[j][kb], xl[j][kb], h);
        }
  }
  const h8 eye[2] = {identity(0, r, g), identity(1, r, g)};
  const MuonCore<MB> core(muon_smem, wave, lane);
  for (int s = 0; s < steps.count; ++s) {
    typename MuonCore<MB>::Tiles gram;
    core.clear(gram);
#pragma unroll
    for (int j = 0; j < J; ++j) {
      __syncthreads();        // what was there is read
      core.turn_columns(xh[j], xl[j], eye);
      __syncthreads();
      if (core.mine) core.template times_itself<4>(gram, core.xs);
    }
    core.to_p(gram, steps, s);
    constexpr int JP = J > 1 ? 2 : 1;     // column tiles at a time
#pragma unroll
    for (int j = 0; j < J; j += JP) core.template apply<JP>(xh + j, xl + j, steps.apply[s]);
  }
  // What is stored is hi + lo, 22 bits at least of the largest values: the products before keep no more.
  asm volatile("" : "+v"(r), "+v"(g));     // or the places of all elements would be kept in registers throughout
  const float back = ldexpf(1.f, -steps.end);
#pragma unroll
  for (int j0 = 0; j0 < J; j0 += in.JW) {
    __syncthreads();                       // LDS is read
    in.at(j0);
    float* const tile = reinterpret_cast<float*>(muon_smem);
#pragma unroll
    for (int j = 0; j < in.JW; ++j) {
      const int c = 16 * (8 * j + wave) + r;
#pragma unroll
      for (int kb = 0; kb < MB; ++kb)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int i = 32 * kb + 16 * (e >> 2) + 4 * g + (e & 3);
          tile[in.tall ? c * in.pitch + i : i * in.pitch + c] = ((float)xh[j0 + j][kb][e] + (float)xl[j0 + j][kb][e]) * back;
        }
    }
    __syncthreads();
    if (a.cols % 4 == 0) muon_give<OUT, 4>(a, in, base, tile);
    else muon_give<OUT, 1>(a, in, base, tile);
  }
}

constexpr int NORM_MOST = 1024;   // blocks that share a matrix's norm

// ---- a block 128 columns, a launch a step ------------------------------------------------------------

// Few matrices of 65 to 128 rows: a block each 128 columns of them, whose parts of G go through memory: a launch adds up
// the parts, makes P (every block of a matrix its own), multiplies its columns and leaves them and their part of the next G.
struct MuonPanels {
  int panels, parts;           // blocks of a matrix, of its norm
  const double* norms;
  uint8_t* x;                  // [matrix][panel][wave][32 rows][hi, lo][lane]: fragments of X^T
  const float* in;             // parts of G: [matrix][panel][tile][lane][4]
  float* out;
};
enum { PANEL_FIRST = 0, PANEL_STEP = 1, PANEL_LAST = 2 };

template <int KIND, int DT, int OUT>
__global__ __launch_bounds__(512, 2) void muon_panel_kernel(Muon a, MuonSize z, MuonSteps steps, int s, MuonPanels q) {
  constexpr int MB = 4, TILES = 64;
  extern __shared__ __attribute__((aligned(16))) uint8_t muon_smem[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  // a matrix's blocks on one XCD, whose L2 holds what they leave for each other (blocks are dealt out to 8 in turn)
  const int slot = blockIdx.x >> 3, panel = slot % q.panels, matrix = slot / q.panels * 8 + (blockIdx.x & 7);
  if (matrix >= a.batch) return;
  const size_t place0 = (size_t)matrix * q.panels + panel;
  const size_t base = (size_t)matrix * a.rows * a.cols;
  const MuonCore<MB> core(muon_smem, wave, lane);
  float* const tile = reinterpret_cast<float*>(muon_smem);
  uint8_t* const saved = q.x + (place0 * 8 + wave) * MB * 2048 + lane * 16;
  MuonRegion<MB, 1> in(a, z);
  in.at(panel);
  const int c = 16 * wave + r;
  h8 xh[1][MB], xl[1][MB];
  if constexpr (KIND == PANEL_FIRST) {
    double t = 0;
    for (int i = lane; i < q.parts; i += 64) t += q.norms[matrix * NORM_MOST + i];
    if (a.cols % 4 == 0) muon_take<DT, 4, true>(a, in, base, tile);
    else muon_take<DT, 1, true>(a, in, base, tile);
    for (int o = 32; o > 0; o >>= 1) t += __shfl_xor(t, o, 64);
    const double f = 1.0 / (sqrt(t) + a.epsilon);
    __syncthreads();
#pragma unroll
    for (int kb = 0; kb < MB; ++kb)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        f4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = 32 * kb + 16 * h + 4 * g + e;
          const float u = tile[in.tall ? c * in.pitch + i : i * in.pitch + c];
          v[e] = i < z.m && c < in.width ? ldexpf((float)(u * f), steps.start) : 0.f;
        }
        split4(v, xh[0][kb], xl[0][kb], h);
      }
    __syncthreads();          // u is read
  } else {
    typename MuonCore<MB>::Tiles gram;
    core.clear(gram);
#pragma unroll
    for (int kb = 0; kb < MB; ++kb) {
      xh[0][kb] = *reinterpret_cast<const h8*>(saved + kb * 2048);
      xl[0][kb] = *reinterpret_cast<const h8*>(saved + kb * 2048 + 1024);
    }
    constexpr int A = MuonTiles<MB>::A, B = MuonTiles<MB>::B;
    for (int k0 = 0; k0 < q.panels; k0 += 4) {       // the loads of four parts under way together
      f4 v[4][A][B];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const f4* const at = reinterpret_cast<const f4*>(q.in) + ((size_t)matrix * q.panels + min(k0 + k, q.panels - 1)) * TILES * 64 + lane;
#pragma unroll
        for (int i = 0; i < A; ++i)
#pragma unroll
          for (int j = 0; j < B; ++j) v[k][i][j] = at[((core.ta + i) * 8 + core.tb + j) * 64];
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (k0 + k < q.panels)
#pragma unroll
          for (int i = 0; i < A; ++i)
#pragma unroll
            for (int j = 0; j < B; ++j) gram[i][j] += v[k][i][j];
    }
    core.to_p(gram, steps, s);
    core.template apply<1>(xh, xl, steps.apply[s]);
  }
  if constexpr (KIND == PANEL_LAST) {
    const float back = ldexpf(1.f, -steps.end);
    __syncthreads();          // P is read
#pragma unroll
    for (int kb = 0; kb < MB; ++kb)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int i = 32 * kb + 16 * (e >> 2) + 4 * g + (e & 3);
        tile[in.tall ? c * in.pitch + i : i * in.pitch + c] = ((float)xh[0][kb][e] + (float)xl[0][kb][e]) * back;
      }
    __syncthreads();
    if (a.cols % 4 == 0) muon_give<OUT, 4>(a, in, base, tile);
    else muon_give<OUT, 1>(a, in, base, tile);
  } else {
    const h8 eye[2] = {identity(0, r, g), identity(1, r, g)};
#pragma unroll
    for (int kb = 0; kb < MB; ++kb) {
      *reinterpret_cast<h8*>(saved + kb * 2048) = xh[0][kb];
      *reinterpret_cast<h8*>(saved + kb * 2048 + 1024) = xl[0][kb];
    }
    core.turn_columns(xh[0], xl[0], eye);
    __syncthreads();
    typename MuonCore<MB>::Tiles gram;
    core.clear(gram);
    core.template times_itself<4>(gram, core.xs);
    f4* const at = reinterpret_cast<f4*>(q.out) + place0 * TILES * 64 + lane;
#pragma unroll
    for (int i = 0; i < MuonTiles<MB>::A; ++i)
#pragma unroll
      for (int j = 0; j < MuonTiles<MB>::B; ++j) at[((core.ta + i) * 8 + core.tb + j) * 64] = gram[i][j];
  }
}

// ---- larger matrices: a product a launch ---------------------------------------------------------

// A matrix in scratch, as fragments: [rows / 16][k / 32][hi, lo], 1 KB each; rows and k are multiples of 128, zeros
// behind the matrix.
struct Frags {
  uint8_t* at;
  int kbs;
  size_t stride;               // bytes between matrices of the batch
};
__device__ __forceinline__ uint8_t* frag(const Frags& f, int tile, int kb) {
  return f.at + blockIdx.z * f.stride + ((size_t)tile * f.kbs + kb) * 2048;
}

// Sums of squares, in double: f32's largest values do not overflow it.
template <int DT>
__global__ __launch_bounds__(256) void muon_norm_kernel(Muon a, double* partial) {
  __shared__ double sm[4];
  const long long count = (long long)a.rows * a.cols;
  const size_t base = (size_t)blockIdx.y * count;
  double t = 0;
  constexpr int V = 4;           // elements under way
  for (long long i0 = (long long)blockIdx.x * 256 * V + threadIdx.x; i0 < count; i0 += (long long)gridDim.x * 256 * V) {
    float gv[V], mv[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const size_t i = base + min(i0 + k * 256, count - 1);
      gv[k] = Act<DT>::ld(static_cast<const typename Act<DT>::T*>(a.grad) + i);
      mv[k] = a.momentum ? a.momentum[i] : 0.f;
    }
#pragma unroll
    for (int k = 0; k < V; ++k) {
      if (i0 + k * 256 >= count) continue;
      float u = gv[k];
      if (a.momentum) {
        const float m = a.momentum_factor * mv[k] + u;
        a.momentum_out[base + i0 + k * 256] = m;
        u = a.nesterov ? u + a.momentum_factor * m : m;
      }
      t += (double)u * u;
    }
  }
  for (int o = 32; o > 0; o >>= 1) t += __shfl_xor(t, o, 64);
  if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = t;
  __syncthreads();
  if (threadIdx.x == 0) partial[blockIdx.y * NORM_MOST + blockIdx.x] = sm[0] + sm[1] + sm[2] + sm[3];
}

// Stores a wave's two tiles of 16 columns, 32 rows, of X: fragments of X^T (j tiles jt, jt + 1) and of X (i tiles).
__device__ __forceinline__ void store_x(const h8 (&hi)[2], const h8 (&lo)[2], const Frags& x, const Frags& xt, int jt, int kb,
                                        int lane) {
  const int r = lane & 15, g = lane >> 4;
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    uint8_t* const at = frag(xt, jt + q, kb) + lane * 16;
    *reinterpret_cast<h8*>(at) = hi[q];
    *reinterpret_cast<h8*>(at + 1024) = lo[q];
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const h8 eye = identity(h, r, g);
    const h4 a = turn(hi[0], eye), b = turn(hi[1], eye), c = turn(lo[0], eye), d = turn(lo[1], eye);
    uint8_t* const at = frag(x, 2 * kb + h, jt / 2) + lane * 16;
    *reinterpret_cast<h8*>(at) = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    *reinterpret_cast<h8*>(at + 1024) = __builtin_shufflevector(c, d, 0, 1, 2, 3, 4, 5, 6, 7);
  }
}

// X = u / (|u| + epsilon) times 2^e; a wave takes 32 rows by 32 columns.
template <int DT>
__global__ __launch_bounds__(256) void muon_start_kernel(Muon a, MuonSize z, const double* partial, int parts, int e, Frags x,
                                                         Frags xt) {
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  double t = 0;
  for (int i = lane; i < parts; i += 64) t += partial[blockIdx.z * NORM_MOST + i];
  for (int o = 32; o > 0; o >>= 1) t += __shfl_xor(t, o, 64);
  const double f = 1.0 / (sqrt(t) + a.epsilon);
  const size_t base = (size_t)blockIdx.z * a.rows * a.cols;
  const int kb = blockIdx.y, jt = (blockIdx.x * 4 + (threadIdx.x >> 6)) * 2;
  h8 hi[2], lo[2];
#pragma unroll
  for (int q = 0; q < 2; ++q)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      f4 v = muon_u4<DT>(a, z, base, 32 * kb + 16 * h + 4 * g, 16 * (jt + q) + r);
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = ldexpf((float)(v[k] * f), e);
      split4(v, hi[q], lo[q], h);
    }
  store_x(hi, lo, x, xt, jt, kb, lane);
}

enum { GRAM = 0, GRAM_PART = 1, SQUARE = 2, APPLY = 3, LAST = 4 };

struct Product {
  Frags a, b;                  // out[i][j] = sum over k of a[i][k] b[j][k]
  int steps, parts;            // of 32 k; GRAM_PART: blocks that share a tile's steps
  Frags out, out_t;            // APPLY: X and its transpose; GRAM, SQUARE: a symmetric matrix
  float* partial;              // GRAM_PART: [part][tile of the block][tile][lane][4]
  float f;                     // factor of the sum
  float fb, fa;                // SQUARE: of a's own element, and the diagonal's
};

// The t-th of the tiles on and above the diagonal of n x n.
__device__ __forceinline__ void upper(int t, int n, int& i, int& j) {
  i = 0;
  while (t >= n - i) {
    t -= n - i;
    ++i;
  }
  j = i + t;
}

// Symmetric results: two tiles one above the other in their place, and, off the diagonal, turned in the other.
__device__ __forceinline__ void store_symmetric(const f4 (&v)[2][2], const Frags& out, int ti, int tj, bool both, int lane) {
  const int r = lane & 15, g = lane >> 4;
  h8 hi[2], lo[2];
#pragma unroll
  for (int q = 0; q < 2; ++q) {
#pragma unroll
    for (int h = 0; h < 2; ++h) split4(v[h][q], hi[q], lo[q], h);
    uint8_t* const at = frag(out, tj + q, ti / 2) + lane * 16;
    *reinterpret_cast<h8*>(at) = hi[q];
    *reinterpret_cast<h8*>(at + 1024) = lo[q];
  }
  if (!both) return;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const h8 eye = identity(h, r, g);
    const h4 a = turn(hi[0], eye), b = turn(hi[1], eye), c = turn(lo[0], eye), d = turn(lo[1], eye);
    uint8_t* const at = frag(out, ti + h, tj / 2) + lane * 16;
    *reinterpret_cast<h8*>(at) = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    *reinterpret_cast<h8*>(at + 1024) = __builtin_shufflevector(c, d, 0, 1, 2, 3, 4, 5, 6, 7);
  }
}

// A block of four waves computes 32 W by 32 W, a wave 16 W by 16 W (W 2 or 4), 32 k a step, both operands through one of
// DEPTH LDS buffers, DEPTH - 1 steps ahead; fragments are read a step ahead too, so that the products do not wait for LDS.
// Four buffers where a CU has one block anyway, two, which leave room for two blocks, where there are more: 1024 x 1024
// times 1024 x 4096 (256 blocks) takes 34 us and 40, five steps of 96 matrices of 256 x 1024 995 and 854.
template <int W>
struct MuonFrags {
  h8 ah[W], al[W], bh[W], bl[W];
};

template <int KIND, int W, int DEPTH, int OUT>
__global__ __launch_bounds__(256, DEPTH == 4 && W == 4 ? 1 : 2) void muon_product_kernel(Product p, Muon m, MuonSize z, int across) {
  constexpr int STAGE = 4 * W * 2048, EACH = STAGE / 4096;      // copies of 1 KB a wave
  // Separate objects: reads of one are then known not to wait for copies into another.
  __shared__ __attribute__((aligned(16))) uint8_t S0[STAGE], S1[STAGE], S2[DEPTH == 4 ? STAGE : 16], S3[DEPTH == 4 ? STAGE : 16];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  int bi, bj, part = 0;
  if constexpr (KIND == APPLY || KIND == LAST) {
    // an XCD takes a run of blocks, 4 along m, then all along n: five steps of 4096 x 1024 take 389 us, 395 without
    const int each = gridDim.x >> 3, id = gridDim.x & 7 ? blockIdx.x : (blockIdx.x & 7) * each + (blockIdx.x >> 3);
    const int down = gridDim.x / across, turn = id / (4 * down), in = id - turn * 4 * down, tall = min(4, across - turn * 4);
    bi = turn * 4 + in % tall;
    bj = in / tall;
  } else {
    const int tile = KIND == GRAM_PART ? blockIdx.x / p.parts : blockIdx.x;
    part = KIND == GRAM_PART ? blockIdx.x % p.parts : 0;
    upper(tile, across, bi, bj);
  }
  const int s0 = KIND == GRAM_PART ? (int)((long long)p.steps * part / p.parts) : 0;
  const int s1 = KIND == GRAM_PART ? (int)((long long)p.steps * (part + 1) / p.parts) : p.steps;
  // [2 W tiles of a][2 W tiles of b], hi and lo of each side by side
  const uint8_t* const src = wave < 2 ? frag(p.a, bi * 2 * W + (wave & 1) * W, 0) : frag(p.b, bj * 2 * W + (wave & 1) * W, 0);
  const uint32_t row = (uint32_t)(wave < 2 ? p.a.kbs : p.b.kbs) * 2048;
  auto stage = [&](uint8_t* dst, int s) __attribute__((always_inline)) {
#if __HIP_DEVICE_COMPILE__
    const uint64_t v = reinterpret_cast<uint64_t>(src);
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
    const __amdgpu_buffer_rsrc_t rs =
        __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>((uint64_t)hi << 32 | lo), 0, 0xffffffffu, 0x27000);
#pragma unroll
    for (int i = 0; i < EACH; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, dst + (wave * EACH + i) * 1024, 16, lane * 16, (i >> 1) * row + s * 2048 + (i & 1) * 1024,
                                               0, 0);
#else
    (void)src, (void)row, (void)dst, (void)s;
#endif
  };
  const int wi = wave >> 1, wj = wave & 1;
  f4 acc[W][W];
#pragma unroll
  for (int i = 0; i < W; ++i)
#pragma unroll
    for (int j = 0; j < W; ++j) acc[i][j] = f4{0.f, 0.f, 0.f, 0.f};
  typedef MuonFrags<W> F;
  auto read = [&](F& f, const uint8_t* buf) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < W; ++t) {
      const uint8_t* const a = buf + (wi * W + t) * 2048 + lane * 16;
      const uint8_t* const b = buf + (2 * W + wj * W + t) * 2048 + lane * 16;
      f.ah[t] = *reinterpret_cast<const h8*>(a);
      f.al[t] = *reinterpret_cast<const h8*>(a + 1024);
      f.bh[t] = *reinterpret_cast<const h8*>(b);
      f.bl[t] = *reinterpret_cast<const h8*>(b + 1024);
    }
  };
  // past the end the last step again, which nothing uses
  stage(S0, s0);
  stage(S1, min(s0 + 1, s1 - 1));
  if constexpr (DEPTH == 4) {
    stage(S2, min(s0 + 2, s1 - 1));
    stage(S3, min(s0 + 3, s1 - 1));
  }
  F f0, f1;
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"((DEPTH - 1) * EACH) : "memory");
  __builtin_amdgcn_s_barrier();
  read(f0, S0);
  // Step s: its fragments are in `now`, step s + 1 is in `buf`, and `freed` held step s.
  auto step = [&](int s, const F& now, F& next, const uint8_t* buf, uint8_t* freed) __attribute__((always_inline)) {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((DEPTH - 2) * EACH) : "memory");
    __builtin_amdgcn_s_barrier();       // every wave's copies of s + 1 are there, every wave has read s
    __builtin_amdgcn_sched_barrier(0);
    read(next, buf);
    stage(freed, min(s + DEPTH, s1 - 1));
#pragma unroll
    for (int i = 0; i < W; ++i)
#pragma unroll
      for (int j = 0; j < W; ++j) acc[i][j] = mfma_pair(now.ah[i], now.al[i], now.bh[j], now.bl[j], acc[i][j]);
    __builtin_amdgcn_sched_barrier(0);   // products touch no memory: they would be moved past the next barrier
  };
  int s = s0;
  if constexpr (DEPTH == 4) {
    for (; s + 3 < s1; s += 4) {
      step(s, f0, f1, S1, S0);
      step(s + 1, f1, f0, S2, S1);
      step(s + 2, f0, f1, S3, S2);
      step(s + 3, f1, f0, S0, S3);
    }
    if (s < s1) step(s, f0, f1, S1, S0);
    if (s + 1 < s1) step(s + 1, f1, f0, S2, S1);
    if (s + 2 < s1) step(s + 2, f0, f1, S3, S2);
  } else {
    for (; s + 1 < s1; s += 2) {
      step(s, f0, f1, S1, S0);
      step(s + 1, f1, f0, S0, S1);
    }
    if (s < s1) step(s, f0, f1, S1, S0);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the last copies, which nothing reads
  const int ti = (bi * 2 + wi) * W, tj = (bj * 2 + wj) * W;
  if constexpr (KIND == GRAM_PART) {
    f4* const at = reinterpret_cast<f4*>(p.partial) +
                   ((((size_t)blockIdx.z * p.parts + part) * (across * (across + 1) / 2) + blockIdx.x / p.parts) * 4 + wave) * W * W * 64 + lane;
#pragma unroll
    for (int i = 0; i < W; ++i)
#pragma unroll
      for (int j = 0; j < W; ++j) at[(i * W + j) * 64] = acc[i][j];
    return;
  }
#pragma unroll
  for (int i = 0; i < W; i += 2)
#pragma unroll
    for (int j = 0; j < W; j += 2) {
      f4 v[2][2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int q = 0; q < 2; ++q) v[h][q] = acc[i + h][j + q] * p.f;
      if constexpr (KIND == SQUARE) {      // + fb of a's element: symmetric, so rows tj, k ti
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const uint8_t* const at = frag(p.a, tj + j + q, (ti + i) / 2) + lane * 16;
          const h8 hi = *reinterpret_cast<const h8*>(at), lo = *reinterpret_cast<const h8*>(at + 1024);
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              v[h][q][e] += p.fb * ((float)hi[4 * h + e] + (float)lo[4 * h + e]);
              if (ti + i + h == tj + j + q && r == 4 * g + e) v[h][q][e] += p.fa;
            }
        }
      }
      if constexpr (KIND == GRAM || KIND == SQUARE) {
        store_symmetric(v, p.out, ti + i, tj + j, bi != bj, lane);
      } else if constexpr (KIND == APPLY) {
        h8 hi[2], lo[2];
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
          for (int h = 0; h < 2; ++h) split4(v[h][q], hi[q], lo[q], h);
        store_x(hi, lo, p.out, p.out_t, tj + j, (ti + i) / 2, lane);
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int q = 0; q < 2; ++q)
            muon_store4<OUT>(m, z, (size_t)blockIdx.z * m.rows * m.cols, (ti + i + h) * 16 + 4 * g, (tj + j + q) * 16 + r, v[h][q]);
      }
    }
}

// The parts of G's tiles added up; a wave a pair of tiles by two.
template <int W>
__global__ __launch_bounds__(256) void muon_join_kernel(Product p, int across) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, tiles = across * (across + 1) / 2;
  constexpr int EACH = W * W / 4;          // pairs by two of a wave's tiles
  const int tile = blockIdx.x / EACH, k = blockIdx.x % EACH, i = k / (W / 2) * 2, j = k % (W / 2) * 2;
  int bi, bj;
  upper(tile, across, bi, bj);
  f4 v[2][2];
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int q = 0; q < 2; ++q) v[h][q] = f4{0.f, 0.f, 0.f, 0.f};
  for (int part = 0; part < p.parts; ++part) {
    const f4* const at = reinterpret_cast<const f4*>(p.partial) +
                         ((((size_t)blockIdx.z * p.parts + part) * tiles + tile) * 4 + wave) * W * W * 64 + lane;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int q = 0; q < 2; ++q) v[h][q] += at[((i + h) * W + j + q) * 64];
  }
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int q = 0; q < 2; ++q) v[h][q] *= p.f;
  store_symmetric(v, p.out, (bi * 2 + (wave >> 1)) * W + i, (bj * 2 + (wave & 1)) * W + j, bi != bj, lane);
}

MuonSize muon_size(long long rows, long long cols) { return MuonSize{(int)std::min(rows, cols), (int)std::max(rows, cols)}; }

// ---- which kernels -------------------------------------------------------------------------------

constexpr int CUS = 256;

enum MuonKind { BLOCK, PANELS, PRODUCTS };
// Panels where a matrix has three or more and the chip holds all of them at once: 64 matrices of 128 x 512 take 112 us, and
// 137 in blocks of their own, 65 175 and 137; 64 of 128 x 384 97 and 134, 86 176 and 139; 16 of 128 x 256, two panels, 78 and
// 75, 64 91 and 77.  Beyond 512 columns the others are products: 32 of 128 x 1024 124 and 187, 33 197 and 191.
MuonKind muon_kind(long long batch, const MuonSize& z) {
  const long long panels = (z.n + 127) / 128;
  if (z.m > 64 && z.m <= 128 && panels > 2 && panels <= 8 && batch * panels <= CUS) return PANELS;
  return z.m <= 128 && z.n <= 512 ? BLOCK : PRODUCTS;
}
int norm_parts(long long count) { return (int)std::min<long long>(NORM_MOST, (count + 4095) / 4096); }

struct MuonGrid {
  int mp, np, w, across, gram_parts;   // padded sides, W, blocks along m
};
MuonGrid muon_grid(long long batch, const MuonSize& z) {
  MuonGrid q;
  q.mp = (z.m + 127) / 128 * 128;
  q.np = (z.n + 127) / 128 * 128;
  q.w = batch * (q.mp / 128) * (q.np / 128) >= CUS ? 4 : 2;
  q.across = q.mp / (32 * q.w);
  // G's tiles are few: parts of 8 steps at least until they fill the chip
  const long long tiles = batch * q.across * (q.across + 1) / 2;
  q.gram_parts = (int)std::max<long long>(1, std::min<long long>(2 * CUS / tiles, q.np / 256));
  return q;
}

size_t up256(size_t n) { return (n + 255) & ~size_t(255); }

int norms(lf_context* ctx, const Muon& a, double* partial) {
  const dim3 grid(norm_parts((long long)a.rows * a.cols), a.batch), block(256);
  LaunchScope ls(ctx, "muon.norm");
  if (a.grad_dtype == LF_F32) hipLaunchKernelGGL((muon_norm_kernel<DT_F32>), grid, block, 0, ctx->stream, a, partial);
  else if (a.grad_dtype == LF_F16) hipLaunchKernelGGL((muon_norm_kernel<DT_F16>), grid, block, 0, ctx->stream, a, partial);
  else hipLaunchKernelGGL((muon_norm_kernel<DT_BF16>), grid, block, 0, ctx->stream, a, partial);
  return check_hip(hipGetLastError(), "muon norm launch");
}

template <int DT>
int start(lf_context* ctx, const Muon& a, const MuonSize& z, const MuonGrid& q, const double* partial, int e, const Frags& x,
          const Frags& xt) {
  LaunchScope ls(ctx, "muon.start");
  hipLaunchKernelGGL((muon_start_kernel<DT>), dim3(q.np / 128, q.mp / 32, a.batch), dim3(256), 0, ctx->stream, a, z, partial,
                     norm_parts((long long)a.rows * a.cols), e, x, xt);
  return check_hip(hipGetLastError(), "muon start launch");
}

constexpr int PANEL_LDS = std::max(2 * 4 * 4 * 2048 + 2 * 4 * 4 * 2048, MuonRegion<4, 1>::BYTES);
template <int KIND, int DT = DT_F32, int OUT = DT_F32>
int panel(lf_context* ctx, const Muon& m, const MuonSize& z, const MuonSteps& f, int s, const MuonPanels& q, const char* label) {
  const auto kernel = muon_panel_kernel<KIND, DT, OUT>;
  static const hipError_t lds = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, PANEL_LDS);
  LF_TRY(check_hip(lds, "muon LDS"));
  LaunchScope ls(ctx, label);
  hipLaunchKernelGGL(kernel, dim3((m.batch + 7) / 8 * 8 * q.panels), dim3(512), PANEL_LDS, ctx->stream, m, z, f, s, q);
  return check_hip(hipGetLastError(), "muon panel launch");
}

template <int KIND, int W, int OUT = DT_F32>
void go_product(lf_context* ctx, const Product& p, const Muon& m, const MuonSize& z, const MuonGrid& q) {
  const int tiles = q.across * (q.across + 1) / 2;
  const int blocks = KIND == GRAM_PART ? tiles * p.parts : KIND == APPLY || KIND == LAST ? q.across * (q.np / (32 * W)) : tiles;
  const dim3 grid(blocks, 1, m.batch);
  if ((long long)blocks * m.batch <= CUS)
    hipLaunchKernelGGL((muon_product_kernel<KIND, W, 4, OUT>), grid, dim3(256), 0, ctx->stream, p, m, z, q.across);
  else
    hipLaunchKernelGGL((muon_product_kernel<KIND, W, 2, OUT>), grid, dim3(256), 0, ctx->stream, p, m, z, q.across);
}
template <int KIND, int OUT = DT_F32>
int product(lf_context* ctx, const Product& p, const Muon& m, const MuonSize& z, const MuonGrid& q, const char* label) {
  LaunchScope ls(ctx, label);
  MuonGrid g = q;
  // G^2's tiles are few too, and its sums short: smaller tiles rather than parts
  if (KIND == SQUARE && q.w == 4 && (long long)m.batch * q.across * (q.across + 1) / 2 < CUS) g.w = 2, g.across = 2 * q.across;
  if (g.w == 4) go_product<KIND, 4, OUT>(ctx, p, m, z, g);
  else go_product<KIND, 2, OUT>(ctx, p, m, z, g);
  return check_hip(hipGetLastError(), "muon product launch");
}

template <int MB, int J, int DT, int OUT>
int go_block(lf_context* ctx, const Muon& m, const MuonSize& z, const MuonSteps& s) {
  constexpr int LDS = std::max(2 * MB * 4 * 2048 + 2 * MB * MB * 2048, MuonRegion<MB, J>::BYTES);
  const auto kernel = muon_block_kernel<MB, J, DT, OUT>;
  static const hipError_t lds = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
  LF_TRY(check_hip(lds, "muon LDS"));
  LaunchScope ls(ctx, "muon.block");
  hipLaunchKernelGGL(kernel, dim3(m.batch), dim3(512), LDS, ctx->stream, m, z, s);
  return check_hip(hipGetLastError(), "muon launch");
}
template <int MB, int DT, int OUT>
int go_block(lf_context* ctx, const Muon& m, const MuonSize& z, const MuonSteps& s) {
  if (z.n <= 128) return go_block<MB, 1, DT, OUT>(ctx, m, z, s);
  if (z.n <= 256) return go_block<MB, 2, DT, OUT>(ctx, m, z, s);
  return go_block<MB, 4, DT, OUT>(ctx, m, z, s);
}
template <int DT, int OUT>
int go_block(lf_context* ctx, const Muon& m, const MuonSize& z, const MuonSteps& s) {
  if (z.m <= 32) return go_block<1, DT, OUT>(ctx, m, z, s);
  if (z.m <= 64) return go_block<2, DT, OUT>(ctx, m, z, s);
  return go_block<4, DT, OUT>(ctx, m, z, s);
}
template <int DT>
int go_block(lf_context* ctx, const Muon& m, const MuonSize& z, const MuonSteps& s) {
  if (m.out_dtype == LF_F32) return go_block<DT, DT_F32>(ctx, m, z, s);
  if (m.out_dtype == LF_F16) return go_block<DT, DT_F16>(ctx, m, z, s);
  return go_block<DT, DT_BF16>(ctx, m, z, s);
}

}  // namespace

size_t muon_bytes(long long batch, long long rows, long long cols) {
  const MuonSize z = muon_size(rows, cols);
  const MuonKind kind = muon_kind(batch, z);
  if (kind == BLOCK) return 0;
  if (kind == PANELS) return up256(batch * NORM_MOST * sizeof(double)) + batch * ((z.n + 127) / 128) * (size_t)(3 * 65536);
  const MuonGrid q = muon_grid(batch, z);
  const size_t x = up256(batch * (size_t)q.mp * q.np * 4), g = up256(batch * (size_t)q.mp * q.mp * 4);
  const size_t parts = q.gram_parts > 1 ? batch * (size_t)q.gram_parts * (q.across * (q.across + 1) / 2) * (32 * q.w) * (32 * q.w) * 4 : 0;
  return up256(batch * NORM_MOST * sizeof(double)) + 4 * x + 2 * g + up256(parts);
}

int run_muon(lf_context* ctx, const Muon& m, const MuonPlan& plan, void* scratch) {
  const MuonSize z = muon_size(m.rows, m.cols);
  MuonSteps f{};
  f.count = m.steps;
  f.start = plan.x[0];
  f.end = plan.x[m.steps];
  for (int k = 0; k < m.steps; ++k) {
    const float* c = m.coefficients + 3 * k;
    const int ex = plan.x[k], eg = plan.g[k], ep = plan.p[k];
    f.gram[k] = std::ldexp(1.f, eg - 2 * ex);
    f.square[k] = std::ldexp(c[2], ep - 2 * eg);
    f.gb[k] = std::ldexp(c[1], ep - eg);
    f.diagonal[k] = std::ldexp(c[0], ep);
    f.apply[k] = std::ldexp(1.f, plan.x[k + 1] - ep - ex);
  }
  const MuonKind kind = muon_kind(m.batch, z);
  if (kind == BLOCK) {
    if (m.grad_dtype == LF_F32) return go_block<DT_F32>(ctx, m, z, f);
    if (m.grad_dtype == LF_F16) return go_block<DT_F16>(ctx, m, z, f);
    return go_block<DT_BF16>(ctx, m, z, f);
  }
  if (kind == PANELS) {
    char* const at = static_cast<char*>(scratch);
    double* const sums = reinterpret_cast<double*>(at);
    MuonPanels q{};
    q.panels = (z.n + 127) / 128;
    q.parts = norm_parts((long long)m.rows * m.cols);
    q.norms = sums;
    const size_t each = (size_t)m.batch * q.panels * 65536;
    q.x = reinterpret_cast<uint8_t*>(at + up256((size_t)m.batch * NORM_MOST * sizeof(double)));
    float* const parts[2] = {reinterpret_cast<float*>(q.x + each), reinterpret_cast<float*>(q.x + 2 * each)};
    LF_TRY(norms(ctx, m, sums));
    q.out = parts[0];
    if (m.grad_dtype == LF_F32) LF_TRY((panel<PANEL_FIRST, DT_F32>(ctx, m, z, f, 0, q, "muon.first")));
    else if (m.grad_dtype == LF_F16) LF_TRY((panel<PANEL_FIRST, DT_F16>(ctx, m, z, f, 0, q, "muon.first")));
    else LF_TRY((panel<PANEL_FIRST, DT_BF16>(ctx, m, z, f, 0, q, "muon.first")));
    for (int k = 0; k < m.steps; ++k) {
      q.in = parts[k & 1];
      q.out = parts[!(k & 1)];
      if (k + 1 < m.steps) LF_TRY((panel<PANEL_STEP>(ctx, m, z, f, k, q, "muon.step")));
      else if (m.out_dtype == LF_F32) LF_TRY((panel<PANEL_LAST, DT_F32, DT_F32>(ctx, m, z, f, k, q, "muon.last")));
      else if (m.out_dtype == LF_F16) LF_TRY((panel<PANEL_LAST, DT_F32, DT_F16>(ctx, m, z, f, k, q, "muon.last")));
      else LF_TRY((panel<PANEL_LAST, DT_F32, DT_BF16>(ctx, m, z, f, k, q, "muon.last")));
    }
    return LF_OK;
  }
  const MuonGrid q = muon_grid(m.batch, z);
  char* at = static_cast<char*>(scratch);
  auto take = [&](size_t bytes) {
    char* p = at;
    at += up256(bytes);
    return p;
  };
  double* const sums = reinterpret_cast<double*>(take((size_t)m.batch * NORM_MOST * sizeof(double)));
  auto frags = [&](int rows, int k) {
    Frags p;
    p.kbs = k / 32;
    p.stride = (size_t)rows * k * 4;
    p.at = reinterpret_cast<uint8_t*>(take(m.batch * p.stride));
    return p;
  };
  const Frags x[2] = {frags(q.mp, q.np), frags(q.mp, q.np)}, xt[2] = {frags(q.np, q.mp), frags(q.np, q.mp)};
  const Frags g = frags(q.mp, q.mp), pm = frags(q.mp, q.mp);
  float* const partial = reinterpret_cast<float*>(at);
  LF_TRY(norms(ctx, m, sums));
  if (m.grad_dtype == LF_F32) LF_TRY(start<DT_F32>(ctx, m, z, q, sums, f.start, x[0], xt[0]));
  else if (m.grad_dtype == LF_F16) LF_TRY(start<DT_F16>(ctx, m, z, q, sums, f.start, x[0], xt[0]));
  else LF_TRY(start<DT_BF16>(ctx, m, z, q, sums, f.start, x[0], xt[0]));
  for (int k = 0; k < m.steps; ++k) {
    const int now = k & 1;
    const Product gram{x[now], x[now], q.np / 32, q.gram_parts, g, g, partial, f.gram[k], 0.f, 0.f};
    if (q.gram_parts > 1) {
      LF_TRY(product<GRAM_PART>(ctx, gram, m, z, q, "muon.gram"));
      LaunchScope ls(ctx, "muon.join");
      const int pairs = q.across * (q.across + 1) / 2 * q.w * q.w / 4;
      if (q.w == 4) hipLaunchKernelGGL((muon_join_kernel<4>), dim3(pairs, 1, m.batch), dim3(256), 0, ctx->stream, gram, q.across);
      else hipLaunchKernelGGL((muon_join_kernel<2>), dim3(pairs, 1, m.batch), dim3(256), 0, ctx->stream, gram, q.across);
      LF_TRY(check_hip(hipGetLastError(), "muon join launch"));
    } else {
      LF_TRY(product<GRAM>(ctx, gram, m, z, q, "muon.gram"));
    }
    const Product square{g, g, q.mp / 32, 1, pm, pm, nullptr, f.square[k], f.gb[k], f.diagonal[k]};
    LF_TRY(product<SQUARE>(ctx, square, m, z, q, "muon.square"));
    const bool last = k + 1 == m.steps;
    const Product apply{pm, xt[now], q.mp / 32, 1, x[!now], xt[!now], nullptr, last ? std::ldexp(f.apply[k], -f.end) : f.apply[k], 0.f, 0.f};
    if (!last) LF_TRY(product<APPLY>(ctx, apply, m, z, q, "muon.apply"));
    else if (m.out_dtype == LF_F32) LF_TRY((product<LAST, DT_F32>(ctx, apply, m, z, q, "muon.last")));
    else if (m.out_dtype == LF_F16) LF_TRY((product<LAST, DT_F16>(ctx, apply, m, z, q, "muon.last")));
    else LF_TRY((product<LAST, DT_BF16>(ctx, apply, m, z, q, "muon.last")));
  }
  return LF_OK;
}

}  // namespace lf
