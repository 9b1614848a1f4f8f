// The training step's operators beside the transition: what lf_step.cpp, which validates, and the kernels'
// files share.  The 4-bit format (e2m1 codes with a power of two per group of 32) is described in
// include/localfold.h.
#pragma once
#include "lf_train.h"

namespace lf {

// ---- relative positions ----
int run_relative_position(lf_context* ctx, const lf_relative_position_args& a);
size_t relative_partials(int queries, int keys, int channels, int rows);
int run_relative_position_backward(lf_context* ctx, const lf_relative_position_backward_args& a, void* scratch);

// out[e] = sum over p < count of partial[p][e], e < width, in a fixed order; from `split` on into out2 (or nowhere).
int run_join(lf_context* ctx, const float* partial, int count, long long width, long long split, void* out, void* out2, int dt,
             const char* label);

// ---- 4-bit products ----
constexpr int MX_GROUP = 32;
struct Mx {                      // device view: bytes of a row of codes and of a row of scales
  uint8_t* codes;
  uint8_t* scales;
  int rows, cols;
  size_t pitch, sp;
};
inline Mx mx_view(const lf_mx4& m) {
  return Mx{static_cast<uint8_t*>(m.codes), static_cast<uint8_t*>(m.scales), m.rows, m.cols, LF_MX4_PITCH(m.cols) / 2,
            LF_MX4_SCALE_PITCH(m.rows)};
}
size_t mx4_sum_partials(int rows, int cols);
int run_mx4_pack(lf_context* ctx, const lf_mx4_pack_args& a, void* scratch);
int run_mx4_unpack(lf_context* ctx, const lf_mx4_unpack_args& a);
size_t mx4_linear_bytes(int rows, int inputs, int outputs, bool from_act);
int run_mx4_linear(lf_context* ctx, const lf_mx4_linear_args& a, void* scratch);

// ---- orthogonalised updates ----
struct Muon {
  int batch, rows, cols;
  int grad_dtype;
  const void* grad;
  const float* momentum;       // null: u = grad
  float* momentum_out;
  float momentum_factor;
  bool nesterov;
  int out_dtype;
  const void* weight;          // null: out = O(u)
  void* out;
  float keep, rate;            // out = keep weight - rate O(u)
  int steps;
  const float* coefficients;
  float epsilon;
};
// Exponents that keep every product of a run in the range of f16: what is stored of step k's X, G and P is the
// value times 2^x, 2^g, 2^p.
constexpr int MUON_STEPS = 32;
struct MuonPlan {
  int x[MUON_STEPS + 1], g[MUON_STEPS], p[MUON_STEPS];
};
bool muon_plan(int steps, const float* coefficients, MuonPlan* plan);   // false: the polynomials leave the range
size_t muon_bytes(long long batch, long long rows, long long cols);
int run_muon(lf_context* ctx, const Muon& m, const MuonPlan& plan, void* scratch);

// ---- device helpers ----
// What is written or read once and not soon again passes by the caches (whole words, any alignment of the elements):
// outputs of 147456 rows of 128 x 512 in bf16 took 59 us, and take 46 past them.
template <class T>
__device__ __forceinline__ void stream_out(void* p, const T& v) {
  typedef uint32_t W __attribute__((ext_vector_type(sizeof(T) / 4), aligned(2)));
  __builtin_nontemporal_store(__builtin_bit_cast(W, v), static_cast<W*>(p));
}
template <class T>
__device__ __forceinline__ void stream_in(T& v, const void* p) {
  typedef uint32_t W __attribute__((ext_vector_type(sizeof(T) / 4), aligned(2)));
  v = __builtin_bit_cast(T, __builtin_nontemporal_load(static_cast<const W*>(p)));
}

}  // namespace lf
