// Entry points of the training operators (include/localfold.h): validation, scratch, and the
// transition's training step as an ordered run of them.
#include <cmath>
#include <new>
#include <string>

#include "lf_train.h"

namespace lf {

namespace {

constexpr int MOST_CHANNELS = 4096;      // of a LayerNorm row (16 registers of it a lane)
constexpr int MOST_COLS = 65536;
constexpr long long MOST_ELEMENTS = 1LL << 34;   // of one matrix: launches count threads in 32 bits

bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// What an error names, put together only where there is one.
struct Name {
  const char *fn, *argument;
  std::string operator+(const std::string& rest) const {
    return argument ? std::string(fn) + ": " + argument + rest : fn + rest;
  }
};

int check_shape(const char* fn, long long rows, long long cols, long long most_cols) {
  const Name f{fn, nullptr};
  LF_REQUIRE(rows > 0 && cols > 0, f + ": dimensions must be positive");
  LF_REQUIRE(cols <= most_cols, f + ": rows are at most " + std::to_string(most_cols) + " wide");
  LF_REQUIRE(rows * (long long)LF_CHECKPOINT_PITCH(cols) <= MOST_ELEMENTS, f + ": more than 2^34 elements");
  return LF_OK;
}

int check_act(const char* fn, const char* name, const void* p, int dt) {
  const Name f{fn, nullptr};
  LF_REQUIRE(act_dtype_ok(dt), f + ": dtypes are f32, f16 or bf16");
  LF_REQUIRE(aligned(p, act_bytes(dt)), f + ": " + name + " is not aligned to its type");
  return LF_OK;
}

int check_kept(const char* fn, const char* name, const lf_checkpoint& c, long long rows, long long cols) {
  const Name f{fn, name};
  LF_REQUIRE(c.codes && c.scales, f + " has NULL codes or scales");
  LF_REQUIRE(aligned(c.codes, 16) && aligned(c.scales, 16), f + " is not 16-byte aligned");
  LF_REQUIRE(c.rows == rows && c.cols == cols, f + " is " + std::to_string(c.rows) + " x " + std::to_string(c.cols) +
                                                   "; expected " + std::to_string(rows) + " x " + std::to_string(cols));
  return LF_OK;
}

int check_vec(const char* fn, const char* name, const void* p, bool optional = false) {
  const Name f{fn, nullptr};
  LF_REQUIRE(p || optional, f + ": " + name + " is NULL");
  LF_REQUIRE(aligned(p, 4), f + ": " + name + " is not aligned to its type");
  return LF_OK;
}

int check_weight(const char* fn, const char* name, const lf_weight& w) {
  const Name f{fn, name};
  LF_REQUIRE(w.data, f + " is NULL");
  LF_REQUIRE(w.layout == LF_IN_OUT || w.layout == LF_OUT_IN, f + ": bad layout");
  if (w.dtype == LF_INT8 || w.dtype == LF_INT5)
    return set_error(LF_ERR_UNSUPPORTED, f + ": int8 and int5 weights are not trained");
  LF_REQUIRE(act_dtype_ok(w.dtype), f + ": unknown dtype " + std::to_string(w.dtype));
  LF_REQUIRE(aligned(w.data, act_bytes(w.dtype)), f + " is not aligned to its type");
  LF_REQUIRE(w.rows > 0 && w.cols > 0 && w.rows <= MOST_COLS && w.cols <= MOST_COLS, f + ": dimensions must be in 1..65536");
  return LF_OK;
}

// Scratch of a call: the caller's, or the context's workspace.  The workspace moves when a later call
// grows it, which a captured graph would not see.
int take_scratch(lf_context* ctx, const char* fn, void* given, size_t given_bytes, size_t need, void** out) {
  const Name f{fn, nullptr};
  if (given) {
    LF_REQUIRE(given_bytes >= need, f + ": scratch has " + std::to_string(given_bytes) + " bytes; needs " + std::to_string(need));
    LF_REQUIRE(aligned(given, 16), f + ": scratch is not 16-byte aligned");
    *out = given;
    return LF_OK;
  }
  hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
  LF_TRY(check_hip(hipStreamIsCapturing(ctx->stream, &st), "stream capture status"));
  LF_REQUIRE(st == hipStreamCaptureStatusNone, f + ": a captured call needs scratch of its own");
  return workspace(ctx, &need, out, 1);
}

// ---- single operators ------------------------------------------------------------------------

int checkpoint_args(const char* fn, const lf_checkpoint_args& a) {
  const Name f{fn, nullptr};
  LF_REQUIRE(a.kept && a.act, f + ": NULL activations or checkpoint");
  LF_TRY(check_shape(fn, a.kept->rows, a.kept->cols, MOST_COLS));
  LF_TRY(check_kept(fn, "kept", *a.kept, a.kept->rows, a.kept->cols));
  return check_act(fn, "act", a.act, a.act_dtype);
}
int checkpoint_pack(lf_context* ctx, const lf_checkpoint_args& a) {
  LF_TRY(checkpoint_args("lf_checkpoint_pack", a));
  return run_checkpoint_pack(ctx, a.act, a.act_dtype, kept_view(*a.kept));
}
int checkpoint_unpack(lf_context* ctx, const lf_checkpoint_args& a) {
  LF_TRY(checkpoint_args("lf_checkpoint_unpack", a));
  return run_checkpoint_unpack(ctx, a.act, a.act_dtype, kept_view(*a.kept));
}

int layer_norm(lf_context* ctx, const lf_layer_norm_args& a) {
  static const char fn[] = "lf_layer_norm";
  LF_TRY(check_shape(fn, a.rows, a.channels, MOST_CHANNELS));
  LF_REQUIRE(a.act, "lf_layer_norm: act is NULL");
  LF_TRY(check_act(fn, "act", a.act, a.act_dtype));
  LF_TRY(check_act(fn, "out", a.out, a.act_dtype));
  LF_TRY(check_vec(fn, "scale", a.scale));
  LF_TRY(check_vec(fn, "offset", a.offset));
  LF_REQUIRE((a.mean == nullptr) == (a.rstd == nullptr), "lf_layer_norm: mean and rstd are given together");
  LF_TRY(check_vec(fn, "mean", a.mean, true));
  LF_TRY(check_vec(fn, "rstd", a.rstd, true));
  LF_REQUIRE(a.epsilon > 0.f && std::isfinite(a.epsilon), "lf_layer_norm: epsilon must be finite and positive");
  if (a.act_kept) LF_TRY(check_kept(fn, "act_kept", *a.act_kept, a.rows, a.channels));
  if (a.out_kept) LF_TRY(check_kept(fn, "out_kept", *a.out_kept, a.rows, a.channels));
  LF_REQUIRE(a.out || a.out_kept || a.act_kept || a.mean, "lf_layer_norm: no output is given");
  return run_layer_norm(ctx, a);
}

int layer_norm_backward(lf_context* ctx, const lf_layer_norm_backward_args& a) {
  static const char fn[] = "lf_layer_norm_backward";
  LF_TRY(check_shape(fn, a.rows, a.channels, MOST_CHANNELS));
  LF_REQUIRE(a.grad, "lf_layer_norm_backward: grad is NULL");
  LF_REQUIRE((a.act == nullptr) != (a.act_kept == nullptr), "lf_layer_norm_backward: either act or act_kept is given");
  LF_TRY(check_act(fn, "grad", a.grad, a.act_dtype));
  LF_TRY(check_act(fn, "act", a.act, a.act_dtype));
  LF_TRY(check_act(fn, "residual", a.residual, a.act_dtype));
  LF_TRY(check_act(fn, "out", a.out, a.act_dtype));
  if (a.act_kept) LF_TRY(check_kept(fn, "act_kept", *a.act_kept, a.rows, a.channels));
  LF_TRY(check_vec(fn, "mean", a.mean));
  LF_TRY(check_vec(fn, "rstd", a.rstd));
  LF_TRY(check_vec(fn, "scale", a.scale));
  LF_REQUIRE((a.grad_scale == nullptr) == (a.grad_offset == nullptr),
             "lf_layer_norm_backward: grad_scale and grad_offset are given together");
  LF_REQUIRE(a.out || a.grad_scale, "lf_layer_norm_backward: no output is given");
  LF_REQUIRE(a.out || !a.residual, "lf_layer_norm_backward: a residual without out");
  void* scratch = nullptr;
  if (a.grad_scale) {
    LF_TRY(check_act(fn, "grad_scale", a.grad_scale, a.grad_dtype));
    LF_TRY(check_act(fn, "grad_offset", a.grad_offset, a.grad_dtype));
    LF_TRY(take_scratch(ctx, fn, a.scratch, a.scratch_bytes, layer_norm_partials(a.rows, a.channels), &scratch));
  }
  return run_layer_norm_backward(ctx, a, scratch);
}

PackWeight pack_of(const lf_weight& w, bool backward, void* codes, void* scales) {
  // packed [outputs][inputs]: a stored [in][out] matrix is transposed for the forward product, a stored
  // [out][in] one for the backward
  return PackWeight{w.data, w.dtype, w.rows, w.cols, (w.layout == LF_IN_OUT) != backward,
                    static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales)};
}

int fp8_pack_weight(lf_context* ctx, const lf_fp8_weight_args& a) {
  static const char fn[] = "lf_fp8_pack_weight";
  LF_TRY(check_weight(fn, "w", a.w));
  LF_REQUIRE(a.out && a.out->codes && a.out->scales, "lf_fp8_pack_weight: out is NULL");
  LF_REQUIRE(aligned(a.out->codes, 16) && aligned(a.out->scales, 16), "lf_fp8_pack_weight: out is not 16-byte aligned");
  const PackWeight p = pack_of(a.w, a.backward != 0, a.out->codes, a.out->scales);
  const int n = p.transpose ? p.cols : p.rows, k = p.transpose ? p.rows : p.cols;
  LF_REQUIRE(a.out->outputs == n && a.out->inputs == k,
             "lf_fp8_pack_weight: out is " + std::to_string(a.out->outputs) + " x " + std::to_string(a.out->inputs) +
                 "; expected " + std::to_string(n) + " x " + std::to_string(k));
  return run_pack_weights(ctx, &p, 1);
}

int fp8_linear(lf_context* ctx, const lf_fp8_linear_args& a) {
  static const char fn[] = "lf_fp8_linear";
  LF_REQUIRE(a.act && a.w, "lf_fp8_linear: act or w is NULL");
  const lf_fp8_weight& w = *a.w;
  LF_REQUIRE(w.codes && w.scales, "lf_fp8_linear: w has NULL codes or scales");
  LF_REQUIRE(aligned(w.codes, 16) && aligned(w.scales, 16), "lf_fp8_linear: w is not 16-byte aligned");
  LF_TRY(check_shape(fn, a.act->rows, w.inputs, MOST_COLS));
  LF_TRY(check_shape(fn, a.act->rows, w.outputs, MOST_COLS));
  LF_TRY(check_kept(fn, "act", *a.act, a.act->rows, w.inputs));
  LF_TRY(check_vec(fn, "bias", a.bias, true));
  if (a.relu_of) LF_TRY(check_kept(fn, "relu_of", *a.relu_of, a.act->rows, w.outputs));
  LF_REQUIRE((a.out == nullptr) != (a.out_kept == nullptr), "lf_fp8_linear: either out or out_kept is given");
  if (a.out) {
    LF_TRY(check_act(fn, "out", a.out, a.out_dtype));
    LF_TRY(check_act(fn, "residual", a.residual, a.out_dtype));
  } else {
    LF_REQUIRE(!a.residual, "lf_fp8_linear: a residual needs out");
    LF_TRY(check_kept(fn, "out_kept", *a.out_kept, a.act->rows, w.outputs));
  }
  LinearParams p{};
  p.x = kept_view(*a.act);
  p.w = static_cast<const uint8_t*>(w.codes);
  p.ws = static_cast<const uint8_t*>(w.scales);
  p.rows = a.act->rows;
  p.inputs = w.inputs;
  p.outputs = w.outputs;
  p.bias = a.bias;
  p.relu = a.relu;
  p.relu_of = a.relu_of ? static_cast<const uint8_t*>(a.relu_of->codes) : nullptr;
  p.residual = a.residual;
  p.out = a.out;
  if (a.out_kept) p.q = kept_view(*a.out_kept);
  p.q.pitch = (int)LF_CHECKPOINT_PITCH(w.outputs);
  return run_fp8_linear(ctx, p, a.out ? a.out_dtype : LF_BF16, "fp8.linear");
}

int fp8_weight_grad(lf_context* ctx, const lf_fp8_weight_grad_args& a) {
  static const char fn[] = "lf_fp8_weight_grad";
  LF_REQUIRE(a.grad && a.act && a.out, "lf_fp8_weight_grad: grad, act or out is NULL");
  LF_TRY(check_shape(fn, a.grad->rows, a.grad->cols, MOST_COLS));
  LF_TRY(check_shape(fn, a.grad->rows, a.act->cols, MOST_COLS));
  LF_TRY(check_kept(fn, "grad", *a.grad, a.grad->rows, a.grad->cols));
  LF_TRY(check_kept(fn, "act", *a.act, a.grad->rows, a.act->cols));
  LF_REQUIRE(a.layout == LF_IN_OUT || a.layout == LF_OUT_IN, "lf_fp8_weight_grad: bad layout");
  LF_TRY(check_act(fn, "out", a.out, a.grad_dtype));
  LF_TRY(check_act(fn, "bias", a.bias, a.grad_dtype));
  void* scratch = nullptr;
  const size_t need = weight_grad_partials(a.grad->rows, a.grad->cols, a.act->cols);
  if (a.scratch || need)     // rows that are not split leave no partial sums
    LF_TRY(take_scratch(ctx, fn, a.scratch, a.scratch_bytes,
                        a.scratch ? weight_grad_scratch(a.grad->rows, a.grad->cols, a.act->cols) : need, &scratch));
  const bool in_out = a.layout == LF_IN_OUT;
  const WeightGrad w{kept_view(in_out ? *a.act : *a.grad), kept_view(in_out ? *a.grad : *a.act), a.out, a.bias, in_out};
  return run_weight_grads(ctx, &w, 1, a.grad_dtype, scratch, "fp8.weight_grad");
}

// ---- the transition's training step ------------------------------------------------------------

size_t up(size_t n) { return (n + 255) & ~size_t(255); }
size_t kept_bytes(long long rows, long long cols) {
  return up(rows * LF_CHECKPOINT_PITCH(cols)) + up(LF_CHECKPOINT_GROUPS(cols) * LF_CHECKPOINT_SCALE_PITCH(rows));
}
size_t packed_bytes(long long n, long long k) {
  return up(n * LF_CHECKPOINT_PITCH(k)) + up(LF_CHECKPOINT_GROUPS(n) * LF_CHECKPOINT_GROUPS(k));
}

// Carves a call's scratch.
struct Carve {
  char* at;
  void* take(size_t bytes) {
    void* p = at;
    at += up(bytes);
    return p;
  }
  lf_checkpoint kept(int rows, int cols) {
    lf_checkpoint c{rows, cols, nullptr, nullptr};
    c.codes = take(rows * LF_CHECKPOINT_PITCH(cols));
    c.scales = take(LF_CHECKPOINT_GROUPS(cols) * LF_CHECKPOINT_SCALE_PITCH(rows));
    return c;
  }
  lf_fp8_weight weight(int n, int k) {
    lf_fp8_weight w{n, k, nullptr, nullptr};
    w.codes = take(n * LF_CHECKPOINT_PITCH(k));
    w.scales = take(LF_CHECKPOINT_GROUPS(n) * LF_CHECKPOINT_GROUPS(k));
    return w;
  }
};

size_t train_bytes(int, int c, int h) { return packed_bytes(h, c) + packed_bytes(c, h); }
size_t backward_bytes(int rows, int c, int h) {
  const size_t partials = std::max(weight_grad_partials(rows, h, c, 2), std::max(layer_norm_partials(rows, c), train_partials(c)));
  return packed_bytes(h, c) + packed_bytes(c, h) + kept_bytes(rows, c) + kept_bytes(rows, h) +
         up((size_t)rows * c * 4) + up(partials);
}

int check_transition(const char* fn, int rows, int c, int h, const lf_transition_weights* w, const lf_transition_saved* s) {
  const Name f{fn, nullptr};
  LF_TRY(check_shape(fn, rows, c, MOST_CHANNELS));
  LF_TRY(check_shape(fn, rows, h, MOST_COLS));
  LF_REQUIRE(w, f + ": weights are NULL");
  LF_REQUIRE(s, f + ": saved is NULL");
  LF_TRY(check_vec(fn, "norm_scale", w->norm_scale));
  LF_TRY(check_vec(fn, "norm_offset", w->norm_offset));
  LF_TRY(check_vec(fn, "b1", w->b1, true));
  LF_TRY(check_vec(fn, "b2", w->b2, true));
  LF_TRY(check_weight(fn, "w1", w->w1));
  LF_TRY(check_weight(fn, "w2", w->w2));
  const bool t1 = w->w1.layout == LF_IN_OUT, t2 = w->w2.layout == LF_IN_OUT;
  LF_REQUIRE((t1 ? w->w1.rows : w->w1.cols) == c && (t1 ? w->w1.cols : w->w1.rows) == h, f + ": w1 does not lead from channels to hidden");
  LF_REQUIRE((t2 ? w->w2.rows : w->w2.cols) == h && (t2 ? w->w2.cols : w->w2.rows) == c, f + ": w2 does not lead from hidden to channels");
  LF_TRY(check_kept(fn, "saved act", s->act, rows, c));
  LF_TRY(check_kept(fn, "saved normed", s->normed, rows, c));
  LF_TRY(check_kept(fn, "saved hidden", s->hidden, rows, h));
  LF_TRY(check_vec(fn, "saved mean", s->mean));
  return check_vec(fn, "saved rstd", s->rstd);
}

int transition_train(lf_context* ctx, const lf_transition_train_args& a) {
  static const char fn[] = "lf_transition_train";
  LF_TRY(check_transition(fn, a.rows, a.channels, a.hidden, a.w, a.saved));
  LF_REQUIRE(a.act && a.out, "lf_transition_train: act and out must be device pointers");
  LF_TRY(check_act(fn, "act", a.act, a.act_dtype));
  LF_TRY(check_act(fn, "out", a.out, a.act_dtype));
  LF_REQUIRE(a.epsilon > 0.f && std::isfinite(a.epsilon), "lf_transition_train: epsilon must be finite and positive");
  const lf_transition_weights& w = *a.w;
  const lf_transition_saved& s = *a.saved;
  const int c = a.channels, h = a.hidden;
  void* scratch = nullptr;
  LF_TRY(take_scratch(ctx, fn, a.scratch, a.scratch_bytes, train_bytes(a.rows, c, h), &scratch));
  Carve carve{static_cast<char*>(scratch)};
  const lf_fp8_weight w1 = carve.weight(h, c), w2 = carve.weight(c, h);
  StageScope stage(ctx, "transition.train");
  const PackWeight packs[2] = {pack_of(w.w1, false, w1.codes, w1.scales), pack_of(w.w2, false, w2.codes, w2.scales)};
  LF_TRY(run_pack_weights(ctx, packs, 2));
  if (train_fused(c, h, a.act, a.out)) return run_train_forward(ctx, a, w1, w2);

  lf_layer_norm_args n{};
  n.rows = a.rows;
  n.channels = c;
  n.act_dtype = a.act_dtype;
  n.act = a.act;
  n.scale = w.norm_scale;
  n.offset = w.norm_offset;
  n.epsilon = a.epsilon;
  n.fast_variance = a.fast_variance;
  n.mean = s.mean;
  n.rstd = s.rstd;
  n.act_kept = &s.act;
  n.out_kept = &s.normed;
  LF_TRY(layer_norm(ctx, n));

  lf_fp8_linear_args l{};
  l.act = &s.normed;
  l.w = &w1;
  l.bias = w.b1;
  l.relu = 1;
  l.out_kept = &s.hidden;
  LF_TRY(fp8_linear(ctx, l));

  lf_fp8_linear_args o{};
  o.act = &s.hidden;
  o.w = &w2;
  o.bias = w.b2;
  o.out_dtype = a.act_dtype;
  o.residual = a.accumulate ? a.act : nullptr;
  o.out = a.out;
  return fp8_linear(ctx, o);
}

int transition_backward(lf_context* ctx, const lf_transition_backward_args& a) {
  static const char fn[] = "lf_transition_backward";
  LF_TRY(check_transition(fn, a.rows, a.channels, a.hidden, a.w, a.saved));
  LF_REQUIRE(a.grad && a.out, "lf_transition_backward: grad and out must be device pointers");
  LF_TRY(check_act(fn, "grad", a.grad, a.act_dtype));
  LF_TRY(check_act(fn, "out", a.out, a.act_dtype));
  LF_REQUIRE(a.grad_norm_scale && a.grad_norm_offset && a.grad_w1 && a.grad_w2, "lf_transition_backward: a gradient is NULL");
  for (const void* p : {a.grad_norm_scale, a.grad_norm_offset, a.grad_w1, a.grad_b1, a.grad_w2, a.grad_b2})
    LF_TRY(check_act(fn, "a gradient", p, a.grad_dtype));
  const lf_transition_weights& w = *a.w;
  const lf_transition_saved& s = *a.saved;
  const int c = a.channels, h = a.hidden;
  void* scratch = nullptr;
  LF_TRY(take_scratch(ctx, fn, a.scratch, a.scratch_bytes, backward_bytes(a.rows, c, h), &scratch));
  Carve carve{static_cast<char*>(scratch)};
  // the input gradients' operands: w2 transposed leads from channels to hidden, w1 back to channels
  const lf_fp8_weight w2 = carve.weight(h, c), w1 = carve.weight(c, h);
  const lf_checkpoint d = carve.kept(a.rows, c), e = carve.kept(a.rows, h);
  void* dy = carve.take((size_t)a.rows * c * 4);
  void* partials = carve.at;
  StageScope stage(ctx, "transition.backward");
  const PackWeight packs[2] = {pack_of(w.w2, true, w2.codes, w2.scales), pack_of(w.w1, true, w1.codes, w1.scales)};
  LF_TRY(run_pack_weights(ctx, packs, 2));
  const bool t2 = w.w2.layout == LF_IN_OUT, t1 = w.w1.layout == LF_IN_OUT;
  // half the blocks each: half the partial sums of two launches, and one start and end
  const WeightGrad grads[2] = {
      {kept_view(t2 ? s.hidden : d), kept_view(t2 ? d : s.hidden), a.grad_w2, a.grad_b2, t2},
      {kept_view(t1 ? s.normed : e), kept_view(t1 ? e : s.normed), a.grad_w1, a.grad_b1, t1}};
  if (train_fused(c, h, a.grad, a.out)) {
    LF_TRY(run_train_backward(ctx, a, w2, w1, kept_view(d), kept_view(e), static_cast<float*>(partials)));
    return run_weight_grads(ctx, grads, 2, a.grad_dtype, partials, "fp8.weight_grads");
  }
  LF_TRY(run_checkpoint_pack(ctx, a.grad, a.act_dtype, kept_view(d)));
  lf_fp8_linear_args l{};
  l.act = &d;
  l.w = &w2;
  l.relu_of = &s.hidden;
  l.out_kept = &e;
  LF_TRY(fp8_linear(ctx, l));
  LF_TRY(run_weight_grads(ctx, grads, 2, a.grad_dtype, partials, "fp8.weight_grads"));
  lf_fp8_linear_args o{};
  o.act = &e;
  o.w = &w1;
  o.out_dtype = LF_F32;      // as the fused pass has it: rounded to 16 bits, the norm's gradients were twice as far off
  o.out = dy;
  LF_TRY(fp8_linear(ctx, o));

  lf_layer_norm_backward_args n{};
  n.rows = a.rows;
  n.channels = c;
  n.act_dtype = a.act_dtype;
  n.grad = dy;
  n.act_kept = &s.act;
  n.mean = s.mean;
  n.rstd = s.rstd;
  n.scale = w.norm_scale;
  n.residual = a.accumulate ? a.grad : nullptr;
  n.out = a.out;
  n.grad_dtype = a.grad_dtype;
  n.grad_scale = a.grad_norm_scale;
  n.grad_offset = a.grad_norm_offset;
  return run_layer_norm_backward(ctx, n, partials, true);
}

// The caller's current device stays what it was, and no exception leaves a C entry point.
struct DeviceScope {
  int before = -1;
  explicit DeviceScope(int device) {
    if (hipGetDevice(&before) != hipSuccess) before = -1;
    if (before != device) (void)hipSetDevice(device);
    else before = -1;
  }
  ~DeviceScope() {
    if (before >= 0) (void)hipSetDevice(before);
  }
};

template <class F>
int guarded(F f) noexcept {
  try {
    return f();
  } catch (const std::bad_alloc&) {
    return LF_ERR_MEMORY;
  } catch (...) {
    return LF_ERR_DEVICE;
  }
}

}  // namespace
}  // namespace lf

#define LF_TRAIN_ENTRY(fn, argtype, impl)                                                    \
  int fn(lf_context* ctx, const argtype* args) {                                             \
    return lf::guarded([&]() -> int {                                                        \
      if (!ctx || !args) return lf::set_error(LF_ERR_INVALID, #fn ": NULL context or args"); \
      lf::DeviceScope device(ctx->device);                                                   \
      return lf::impl(ctx, *args);                                                           \
    });                                                                                      \
  }

extern "C" {
LF_TRAIN_ENTRY(lf_checkpoint_pack, lf_checkpoint_args, checkpoint_pack)
LF_TRAIN_ENTRY(lf_checkpoint_unpack, lf_checkpoint_args, checkpoint_unpack)
LF_TRAIN_ENTRY(lf_layer_norm, lf_layer_norm_args, layer_norm)
LF_TRAIN_ENTRY(lf_layer_norm_backward, lf_layer_norm_backward_args, layer_norm_backward)
LF_TRAIN_ENTRY(lf_fp8_pack_weight, lf_fp8_weight_args, fp8_pack_weight)
LF_TRAIN_ENTRY(lf_fp8_linear, lf_fp8_linear_args, fp8_linear)
LF_TRAIN_ENTRY(lf_fp8_weight_grad, lf_fp8_weight_grad_args, fp8_weight_grad)
LF_TRAIN_ENTRY(lf_transition_train, lf_transition_train_args, transition_train)
LF_TRAIN_ENTRY(lf_transition_backward, lf_transition_backward_args, transition_backward)

static bool positive(int a, int b, int c = 1) { return a > 0 && b > 0 && c > 0; }
size_t lf_layer_norm_backward_scratch(int rows, int channels) {
  return positive(rows, channels) ? lf::layer_norm_partials(rows, channels) : 0;
}
size_t lf_fp8_weight_grad_scratch(int rows, int outputs, int inputs) {
  return positive(rows, outputs, inputs) ? lf::weight_grad_scratch(rows, outputs, inputs) : 0;
}
size_t lf_transition_train_scratch(int rows, int channels, int hidden) {
  return positive(rows, channels, hidden) ? lf::train_bytes(rows, channels, hidden) : 0;
}
size_t lf_transition_backward_scratch(int rows, int channels, int hidden) {
  return positive(rows, channels, hidden) ? lf::backward_bytes(rows, channels, hidden) : 0;
}
}
