// Entry points of the training step's operators beside the transition (include/localfold.h): relative
// positions, 4-bit products, orthogonalised updates.  Validation and scratch.
#include "lf_checks.h"
#include "lf_step.h"

namespace lf {

namespace {

constexpr int MOST_BOUNDARIES = 4095;
constexpr int MOST_MX_COLS = 1 << 26;     // offsets of 64 rows of codes are 32 bits
constexpr int MOST_SIDE = 16384;         // of a matrix that is made orthogonal
constexpr int MOST_BATCH = 65535;        // a grid's third dimension

int check_pairs(const char* fn, const lf_relative_pairs* p, int channels) {
  const Name f{fn, nullptr};
  LF_REQUIRE(p, f + ": pairs is NULL");
  LF_REQUIRE(p->queries > 0 && p->keys > 0, f + ": dimensions must be positive");
  LF_REQUIRE(channels > 0 && channels <= MOST_CHANNELS, f + ": channels must be in 1..4096");
  LF_REQUIRE((long long)p->queries * p->keys <= MOST_ELEMENTS / channels, f + ": more than 2^34 elements");
  LF_REQUIRE(p->boundary_count >= 0 && p->boundary_count <= MOST_BOUNDARIES, f + ": boundaries must be 0..4095");
  LF_TRY(check_vec(fn, "boundaries", p->boundaries, p->boundary_count == 0));
  LF_TRY(check_vec(fn, "query_positions", p->query_positions));
  LF_TRY(check_vec(fn, "key_positions", p->key_positions));
  LF_REQUIRE((p->query_segments == nullptr) == (p->key_segments == nullptr), f + ": both sides have segments, or neither");
  LF_TRY(check_vec(fn, "query_segments", p->query_segments, true));
  return check_vec(fn, "key_segments", p->key_segments, true);
}

int relative_position(lf_context* ctx, const lf_relative_position_args& a) {
  static const char fn[] = "lf_relative_position";
  LF_TRY(check_pairs(fn, a.pairs, a.channels));
  LF_REQUIRE(a.table && a.out, "lf_relative_position: table or out is NULL");
  LF_TRY(check_act(fn, "table", a.table, a.table_dtype));
  LF_TRY(check_vec(fn, "bias", a.bias, true));
  LF_TRY(check_act(fn, "act", a.act, a.act_dtype));
  LF_TRY(check_act(fn, "out", a.out, a.act_dtype));
  return run_relative_position(ctx, a);
}

int relative_position_backward(lf_context* ctx, const lf_relative_position_backward_args& a) {
  static const char fn[] = "lf_relative_position_backward";
  LF_TRY(check_pairs(fn, a.pairs, a.channels));
  LF_REQUIRE(a.grad && a.grad_table, "lf_relative_position_backward: grad or grad_table is NULL");
  LF_TRY(check_act(fn, "grad", a.grad, a.act_dtype));
  LF_TRY(check_act(fn, "grad_table", a.grad_table, a.grad_dtype));
  LF_TRY(check_act(fn, "grad_bias", a.grad_bias, a.grad_dtype));
  void* scratch = nullptr;
  LF_TRY(take_scratch(ctx, fn, a.scratch, a.scratch_bytes,
                      relative_partials(a.pairs->queries, a.pairs->keys, a.channels, LF_RELATIVE_ROWS(a.pairs)), &scratch));
  return run_relative_position_backward(ctx, a, scratch);
}

// Rows and columns whose packed form, either way round, stays within the limit.
int check_size(const char* fn, long long rows, long long cols) {
  const Name f{fn, nullptr};
  LF_REQUIRE(rows > 0 && cols > 0, f + ": dimensions must be positive");
  LF_REQUIRE(cols <= MOST_MX_COLS, f + ": 4-bit matrices are at most 2^26 wide");
  LF_REQUIRE((long long)LF_MX4_SCALE_PITCH(rows) <= MOST_ELEMENTS / (long long)LF_MX4_PITCH(cols), f + ": more than 2^34 elements");
  return LF_OK;
}

int check_mx(const char* fn, const char* name, const lf_mx4& m, long long rows, long long cols) {
  const Name f{fn, name};
  LF_REQUIRE(m.codes && m.scales, f + " has NULL codes or scales");
  LF_REQUIRE(aligned(m.codes, 16) && aligned(m.scales, 16), f + " is not 16-byte aligned");
  LF_REQUIRE(m.rows == rows && m.cols == cols, f + " is " + std::to_string(m.rows) + " x " + std::to_string(m.cols) +
                                                   "; expected " + std::to_string(rows) + " x " + std::to_string(cols));
  return LF_OK;
}

int mx4_pack(lf_context* ctx, const lf_mx4_pack_args& a) {
  static const char fn[] = "lf_mx4_pack";
  LF_TRY(check_size(fn, a.rows, a.cols));
  LF_REQUIRE(a.act, "lf_mx4_pack: act is NULL");
  LF_TRY(check_act(fn, "act", a.act, a.act_dtype));
  LF_REQUIRE(a.out || a.transposed || a.sums, "lf_mx4_pack: no output is given");
  if (a.out) LF_TRY(check_mx(fn, "out", *a.out, a.rows, a.cols));
  if (a.transposed) {
    LF_TRY(check_size(fn, a.cols, a.rows));
    LF_TRY(check_mx(fn, "transposed", *a.transposed, a.cols, a.rows));
  }
  void* scratch = nullptr;
  if (a.sums) {
    LF_TRY(check_act(fn, "sums", a.sums, a.sums_dtype));
    LF_TRY(take_scratch(ctx, fn, a.scratch, a.scratch_bytes, mx4_sum_partials(a.rows, a.cols), &scratch));
  }
  return run_mx4_pack(ctx, a, scratch);
}

int mx4_unpack(lf_context* ctx, const lf_mx4_unpack_args& a) {
  static const char fn[] = "lf_mx4_unpack";
  LF_REQUIRE(a.kept && a.act, "lf_mx4_unpack: act or kept is NULL");
  LF_TRY(check_size(fn, a.kept->rows, a.kept->cols));
  LF_TRY(check_mx(fn, "kept", *a.kept, a.kept->rows, a.kept->cols));
  LF_TRY(check_act(fn, "act", a.act, a.act_dtype));
  return run_mx4_unpack(ctx, a);
}

int mx4_linear(lf_context* ctx, const lf_mx4_linear_args& a) {
  static const char fn[] = "lf_mx4_linear";
  LF_REQUIRE(a.w && a.out, "lf_mx4_linear: w or out is NULL");
  LF_REQUIRE((a.kept == nullptr) != (a.act == nullptr), "lf_mx4_linear: either kept or act is given");
  const long long inputs = a.w->cols, outputs = a.w->rows;
  LF_TRY(check_size(fn, outputs, inputs));
  LF_TRY(check_size(fn, a.rows, inputs));
  LF_REQUIRE((long long)a.rows * outputs <= MOST_ELEMENTS, "lf_mx4_linear: more than 2^34 elements");
  LF_TRY(check_mx(fn, "w", *a.w, outputs, inputs));
  if (a.kept) LF_TRY(check_mx(fn, "kept", *a.kept, a.rows, inputs));
  else LF_TRY(check_act(fn, "act", a.act, a.act_dtype));
  LF_TRY(check_vec(fn, "bias", a.bias, true));
  LF_TRY(check_act(fn, "residual", a.residual, a.out_dtype));
  LF_TRY(check_act(fn, "out", a.out, a.out_dtype));
  void* scratch = nullptr;
  const size_t need = mx4_linear_bytes(a.rows, (int)inputs, (int)outputs, a.act != nullptr);
  if (need) LF_TRY(take_scratch(ctx, fn, a.scratch, a.scratch_bytes, need, &scratch));
  return run_mx4_linear(ctx, a, scratch);
}

int check_muon(const char* fn, const Muon& m, MuonPlan* plan) {
  const Name f{fn, nullptr};
  LF_REQUIRE(m.batch > 0 && m.rows > 0 && m.cols > 0, f + ": dimensions must be positive");
  LF_REQUIRE(m.rows <= MOST_SIDE && m.cols <= MOST_SIDE, f + ": matrices are at most 16384 x 16384");
  LF_REQUIRE(m.batch <= MOST_BATCH, f + ": at most 65535 matrices");
  LF_REQUIRE((long long)m.batch * ((m.rows + 127) / 128 * 128) * ((m.cols + 127) / 128 * 128) <= MOST_ELEMENTS,
             f + ": more than 2^34 elements");
  LF_REQUIRE(m.grad && m.out, f + ": an input or output is NULL");
  LF_TRY(check_act(fn, "the input", m.grad, m.grad_dtype));
  LF_TRY(check_act(fn, "the output", m.out, m.out_dtype));
  LF_REQUIRE(m.steps >= 1 && m.steps <= MUON_STEPS, f + ": steps must be in 1..32");
  LF_REQUIRE(m.coefficients, f + ": coefficients are NULL");
  LF_REQUIRE(m.epsilon >= 0.f && std::isfinite(m.epsilon), f + ": epsilon must be finite and not negative");
  for (int i = 0; i < 3 * m.steps; ++i) LF_REQUIRE(std::isfinite(m.coefficients[i]), f + ": coefficients must be finite");
  LF_REQUIRE(muon_plan(m.steps, m.coefficients, plan), f + ": the coefficients' polynomials leave the range of the products");
  return LF_OK;
}

int orthogonalize(lf_context* ctx, const lf_orthogonalize_args& a) {
  static const char fn[] = "lf_orthogonalize";
  Muon m{};
  m.batch = a.batch;
  m.rows = a.rows;
  m.cols = a.cols;
  m.grad_dtype = m.out_dtype = a.act_dtype;
  m.grad = a.act;
  m.out = a.out;
  m.rate = -1.f;
  m.steps = a.steps;
  m.coefficients = a.coefficients;
  m.epsilon = a.epsilon;
  MuonPlan plan;
  LF_TRY(check_muon(fn, m, &plan));
  void* scratch = nullptr;
  const size_t need = muon_bytes(a.batch, a.rows, a.cols);
  if (need) LF_TRY(take_scratch(ctx, fn, a.scratch, a.scratch_bytes, need, &scratch));
  return run_muon(ctx, m, plan, scratch);
}

int muon_step(lf_context* ctx, const lf_muon_step_args& a) {
  static const char fn[] = "lf_muon_step";
  LF_REQUIRE(a.weight, "lf_muon_step: weight is NULL");
  LF_TRY(check_act(fn, "weight", a.weight, a.weight_dtype));
  LF_REQUIRE((a.momentum == nullptr) == (a.momentum_out == nullptr), "lf_muon_step: momentum and momentum_out are given together");
  LF_TRY(check_vec(fn, "momentum", a.momentum, true));
  LF_TRY(check_vec(fn, "momentum_out", a.momentum_out, true));
  for (float v : {a.momentum_factor, a.rate, a.decay, a.scale})
    LF_REQUIRE(std::isfinite(v), "lf_muon_step: momentum_factor, rate, decay and scale must be finite");
  Muon m{};
  m.batch = a.batch;
  m.rows = a.rows;
  m.cols = a.cols;
  m.grad_dtype = a.grad_dtype;
  m.grad = a.grad;
  m.momentum = a.momentum;
  m.momentum_out = a.momentum_out;
  m.momentum_factor = a.momentum_factor;
  m.nesterov = a.nesterov != 0;
  m.out_dtype = a.weight_dtype;
  m.weight = a.weight;
  m.out = a.weight_out;
  m.keep = (float)(1.0 - (double)a.rate * a.decay);
  m.rate = (float)((double)a.rate * a.scale);
  LF_REQUIRE(std::isfinite(m.keep) && std::isfinite(m.rate), "lf_muon_step: 1 - rate decay and rate scale must be finite in f32");
  m.steps = a.steps;
  m.coefficients = a.coefficients;
  m.epsilon = a.epsilon;
  MuonPlan plan;
  LF_TRY(check_muon(fn, m, &plan));
  void* scratch = nullptr;
  const size_t need = muon_bytes(a.batch, a.rows, a.cols);
  if (need) LF_TRY(take_scratch(ctx, fn, a.scratch, a.scratch_bytes, need, &scratch));
  return run_muon(ctx, m, plan, scratch);
}

}  // namespace

// The largest |value| that [0, s] can become under a s + b s^3 + c s^5, and the same for the factor a + b s^2 +
// c s^4 alone: their values at the ends and where the derivative is zero.  In double, a 2^-10 above.
namespace {
double most_factor(double s, double a, double b, double c) {
  const double u = s * s;
  double m = std::max(std::fabs(a), std::fabs(a + b * u + c * u * u));
  if (c != 0) {
    const double v = -b / (2 * c);
    if (v > 0 && v < u) m = std::max(m, std::fabs(a + b * v + c * v * v));
  }
  return m * (1 + 1.0 / 1024);
}
double most_value(double s, double a, double b, double c) {
  auto at = [&](double x) { return std::fabs(x * (a + x * x * (b + x * x * c))); };
  double m = at(s);
  double roots[2];
  int count = 0;
  if (c != 0) {                 // 5 c v^2 + 3 b v + a = 0, v = s^2
    const double d = 9 * b * b - 20 * a * c;
    if (d >= 0) {
      roots[count++] = (-3 * b + std::sqrt(d)) / (10 * c);
      roots[count++] = (-3 * b - std::sqrt(d)) / (10 * c);
    }
  } else if (b != 0) {
    roots[count++] = -a / (3 * b);
  }
  for (int i = 0; i < count; ++i)
    if (roots[i] > 0 && roots[i] < s * s) m = std::max(m, at(std::sqrt(roots[i])));
  return m * (1 + 1.0 / 1024);
}
// 2^e m is within 2^14, an eighth of f16's largest value.
int exponent_for(double m) {
  int e;
  std::frexp(std::max(m, std::ldexp(1.0, -40)), &e);   // m < 2^e
  return 14 - e;
}
}  // namespace

bool muon_plan(int steps, const float* coefficients, MuonPlan* plan) {
  double s = 1 + 1.0 / 1024;    // |X| = 1 at most, in the Frobenius norm, which no singular value exceeds
  for (int k = 0; k < steps; ++k) {
    const double a = coefficients[3 * k], b = coefficients[3 * k + 1], c = coefficients[3 * k + 2];
    const double p = most_factor(s, a, b, c), next = most_value(s, a, b, c);
    if (!(p < std::ldexp(1.0, 24)) || !(next < std::ldexp(1.0, 24))) return false;
    plan->x[k] = exponent_for(s);
    plan->g[k] = exponent_for(s * s);
    plan->p[k] = exponent_for(p);
    s = next;
  }
  plan->x[steps] = exponent_for(s);
  return true;
}

}  // namespace lf

extern "C" {
LF_TRAIN_ENTRY(lf_relative_position, lf_relative_position_args, relative_position)
LF_TRAIN_ENTRY(lf_relative_position_backward, lf_relative_position_backward_args, relative_position_backward)
LF_TRAIN_ENTRY(lf_mx4_pack, lf_mx4_pack_args, mx4_pack)
LF_TRAIN_ENTRY(lf_mx4_unpack, lf_mx4_unpack_args, mx4_unpack)
LF_TRAIN_ENTRY(lf_mx4_linear, lf_mx4_linear_args, mx4_linear)
LF_TRAIN_ENTRY(lf_orthogonalize, lf_orthogonalize_args, orthogonalize)
LF_TRAIN_ENTRY(lf_muon_step, lf_muon_step_args, muon_step)

size_t lf_relative_position_backward_scratch(const lf_relative_pairs* pairs, int channels) {
  if (!pairs || pairs->queries <= 0 || pairs->keys <= 0 || channels <= 0 || pairs->boundary_count < 0) return 0;
  return lf::relative_partials(pairs->queries, pairs->keys, channels, LF_RELATIVE_ROWS(pairs));
}
size_t lf_mx4_pack_scratch(int rows, int cols) { return rows > 0 && cols > 0 ? lf::mx4_sum_partials(rows, cols) : 0; }
size_t lf_mx4_linear_scratch(int rows, int inputs, int outputs, int from_act) {
  return rows > 0 && inputs > 0 && outputs > 0 ? lf::mx4_linear_bytes(rows, inputs, outputs, from_act != 0) : 0;
}
size_t lf_muon_scratch(int batch, int rows, int cols) {
  return batch > 0 && rows > 0 && cols > 0 ? lf::muon_bytes(batch, rows, cols) : 0;
}
}
