// Training operators: what their host side and their kernels share.  The 8-bit format (e4m3 codes
// with a power of two per group of 128) is described in include/localfold.h.
#pragma once
#include "lf_common.h"
#include "lf_ops.h"

namespace lf {

constexpr int GROUP = 128;

// Device views of the format: plain pointers and pitches.
struct Kept {
  uint8_t* codes;
  uint8_t* scales;
  int rows, cols, pitch, sp;   // sp: pitch of the scale rows
};
inline Kept kept_view(const lf_checkpoint& c) {
  return Kept{static_cast<uint8_t*>(c.codes), static_cast<uint8_t*>(c.scales), c.rows, c.cols,
              (int)LF_CHECKPOINT_PITCH(c.cols), (int)LF_CHECKPOINT_SCALE_PITCH(c.rows)};
}

struct LinearParams {
  Kept x;                       // [rows, inputs]
  const uint8_t *w, *ws;        // weight codes [outputs][x.pitch], scales [groups of outputs][groups of inputs]
  int rows, inputs, outputs;
  const float* bias;
  int relu;
  const uint8_t* relu_of;       // codes of a checkpoint of [rows, outputs], or null
  const void* residual;
  void* out;                    // null: q
  Kept q;
};

// Launchers over validated arguments (lf_train.cpp validates).
int run_checkpoint_pack(lf_context* ctx, const void* act, int dt, const Kept& k);
int run_checkpoint_unpack(lf_context* ctx, void* act, int dt, const Kept& k);
struct PackWeight {
  const void* data;
  int dtype, rows, cols;        // stored matrix
  int transpose;                // 1: the packed matrix is [cols, rows]
  uint8_t *codes, *scales;
};
int run_pack_weights(lf_context* ctx, const PackWeight* w, int count);
int run_layer_norm(lf_context* ctx, const lf_layer_norm_args& a);
size_t layer_norm_partials(int rows, int channels);
// wide: a.grad is f32, whatever act_dtype is.
int run_layer_norm_backward(lf_context* ctx, const lf_layer_norm_backward_args& a, void* scratch, bool wide = false);
int run_fp8_linear(lf_context* ctx, const LinearParams& p, int out_dtype, const char* label);
// One of up to two products of the same rows in a launch: out = [a.cols, b.cols] = sum over rows of a^T b;
// bias = sum of a's rows, or of b's when bias_of_b.
struct WeightGrad {
  Kept a, b;
  void *out, *bias;
  bool bias_of_b;
};
size_t weight_grad_partials(int rows, int outputs, int inputs, int products = 1);   // of products of one size; 0: not split
size_t weight_grad_scratch(int rows, int outputs, int inputs);   // what a caller's buffer has: one split's sums at least
int run_weight_grads(lf_context* ctx, const WeightGrad* w, int count, int dt, void* scratch, const char* label);

// Adds [blocks][2 channels] partial sums of scale and offset gradients.
int run_norm_join(lf_context* ctx, const float* partial, int blocks, int channels, void* grad_scale, void* grad_offset,
                  int dt);
// The transition's training step in one kernel each way, where train_fused says that there is one: packed
// weights of the forward pass w1, w2, of the backward w2, w1; d, e: the kept gradients of out and hidden.
bool train_fused(int channels, int hidden, const void* in, const void* out);
int run_train_forward(lf_context* ctx, const lf_transition_train_args& a, const lf_fp8_weight& w1, const lf_fp8_weight& w2);
size_t train_partials(int channels);
int run_train_backward(lf_context* ctx, const lf_transition_backward_args& a, const lf_fp8_weight& w2,
                       const lf_fp8_weight& w1, const Kept& d, const Kept& e, float* partial);

// ---- device helpers ---------------------------------------------------------------------------

template <int CTRL>
__device__ __forceinline__ float dpp_f(float v) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xF, 0xF, true));
}
struct OpSum {
  static __device__ __forceinline__ float f(float a, float b) { return a + b; }
};
struct OpMax {
  static __device__ __forceinline__ float f(float a, float b) { return fmaxf(a, b); }
};
// Reduction over aligned teams of L lanes (8, 16, 32 or 64), every lane gets it: permutes within
// quads, mirrors within 8 and 16 lanes (what a mirror swaps already holds equal values), then
// swaps of 16- and 32-lane rows.  Vector instructions only.
template <int L, class OP>
__device__ __forceinline__ float team_reduce(float v) {
  v = OP::f(v, dpp_f<0xB1>(v));    // quad [1,0,3,2]
  v = OP::f(v, dpp_f<0x4E>(v));    // quad [2,3,0,1]
  v = OP::f(v, dpp_f<0x141>(v));   // half-row mirror
  if constexpr (L >= 16) v = OP::f(v, dpp_f<0x140>(v));   // row mirror
  if constexpr (L >= 32) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = OP::f(__uint_as_float(a[0]), __uint_as_float(a[1]));
  }
  if constexpr (L >= 64) {
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = OP::f(__uint_as_float(b[0]), __uint_as_float(b[1]));
  }
  return v;
}

// Eight consecutive activations p[0..8), of which the first n exist (the others read as zero).  Whole
// eights take 16-byte loads whatever the element alignment (global loads may be unaligned on gfx950).
template <int ACT>
__device__ __forceinline__ void load8(const typename Act<ACT>::T* p, int n, float (&v)[8]) {
  typedef typename Act<ACT>::T T;
  if (n >= 8) {
    uint32_t w[2 * sizeof(T)];
    __builtin_memcpy(w, p, sizeof(w));
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if constexpr (ACT == DT_F32) v[k] = __uint_as_float(w[k]);
      else if constexpr (ACT == DT_BF16) v[k] = __uint_as_float((k & 1) ? (w[k >> 1] & 0xffff0000u) : (w[k >> 1] << 16));
      else v[k] = h2f((uint16_t)((k & 1) ? (w[k >> 1] >> 16) : (w[k >> 1] & 0xffffu)));
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = k < n ? Act<ACT>::ld(p + k) : 0.f;
  }
}

template <int ACT>
__device__ __forceinline__ void store8(typename Act<ACT>::T* p, int n, const float (&v)[8]) {
  typedef typename Act<ACT>::T T;
  if (n >= 8) {
    uint4 o[sizeof(T) / 2];
    pack8<ACT>(v, o);
    __builtin_memcpy(p, o, 8 * sizeof(T));
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < n) Act<ACT>::st(p + k, v[k]);
  }
}

// Largest magnitude of eight values, 0 where all are NaN; NaN is passed over, an infinity is not.
__device__ __forceinline__ float amax8(const float (&v)[8]) {
  float m = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) m = fmaxf(m, fabsf(v[k]));
  return m;
}
__device__ __forceinline__ float amax8_finite(const float (&v)[8]) {
  float m = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) m = fmaxf(m, fabsf(v[k]) < __builtin_inff() ? fabsf(v[k]) : 0.f);
  return m;
}

// The stored byte of the smallest power of two that puts m within 448 = 1.75 * 2^8: m = f * 2^p with
// f in [1, 2) needs 2^(p - 8), or 2^(p - 7) when f > 1.75.  At least 1, so that the power is a normal
// number.
__device__ __forceinline__ int scale_byte(float m) {
  const uint32_t u = __float_as_uint(m);
  const int b = (int)(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return b < 1 ? 1 : b;
}
__device__ __forceinline__ float scale_value(int b) { return __uint_as_float((uint32_t)b << 23); }

// Four values over a power of two as codes.  Within 448 by the choice of the scale; the instruction divides
// exactly, rounds to nearest even and makes infinities and NaN the NaN code.
__device__ __forceinline__ uint32_t encode4(float v0, float v1, float v2, float v3, float scale) {
  typedef short s2v __attribute__((ext_vector_type(2)));
  s2v c = {0, 0};
  c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(c, v0, v1, scale, false);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(c, v2, v3, scale, true);
  return __builtin_bit_cast(uint32_t, c);
}
__device__ __forceinline__ uint2 encode8(const float (&v)[8], float scale) {
  return make_uint2(encode4(v[0], v[1], v[2], v[3], scale), encode4(v[4], v[5], v[6], v[7], scale));
}

__device__ __forceinline__ void decode4(uint32_t w, float s, float* v) {
  v[0] = __builtin_amdgcn_cvt_f32_fp8((int)w, 0) * s;
  v[1] = __builtin_amdgcn_cvt_f32_fp8((int)w, 1) * s;
  v[2] = __builtin_amdgcn_cvt_f32_fp8((int)w, 2) * s;
  v[3] = __builtin_amdgcn_cvt_f32_fp8((int)w, 3) * s;
}

// Encodes the eight values of each lane of a team (16 lanes, or the 8 of an 8-lane row) that holds one
// row's group of 128 and writes codes and scale.  c0: the lane's first column.  `write`: the row exists.
template <int TEAM>
__device__ __forceinline__ void keep8(const Kept& k, size_t row, int c0, const float (&v)[8], bool write) {
  float m = team_reduce<TEAM, OpMax>(amax8(v));
  if (__builtin_expect(m == __builtin_inff(), 0)) m = -1.f;
  if (__builtin_expect(__any(m < 0.f), 0)) {
    const float f = team_reduce<TEAM, OpMax>(amax8_finite(v));
    m = m < 0.f ? f : m;
  }
  const int b = scale_byte(m);
  const uint2 q = encode8(v, scale_value(b));
  if (write && c0 < k.pitch) {
    *reinterpret_cast<uint2*>(k.codes + row * (size_t)k.pitch + c0) = q;
    if ((c0 & (GROUP - 1)) == 0) k.scales[(size_t)(c0 / GROUP) * k.sp + row] = (uint8_t)b;
  }
}

}  // namespace lf
