// What the entry points of the training operators share (include/localfold.h): checks of arguments,
// scratch, the current device and the exceptions.
#pragma once
#include <cmath>
#include <new>
#include <string>

#include "lf_train.h"

namespace lf {

constexpr int MOST_CHANNELS = 4096;      // of a LayerNorm row (16 registers of it a lane)
constexpr int MOST_COLS = 65536;
constexpr long long MOST_ELEMENTS = 1LL << 34;   // of one matrix: launches count threads in 32 bits

inline bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// What an error names, put together only where there is one.
struct Name {
  const char *fn, *argument;
  std::string operator+(const std::string& rest) const {
    return argument ? std::string(fn) + ": " + argument + rest : fn + rest;
  }
};

inline int check_shape(const char* fn, long long rows, long long cols, long long most_cols) {
  const Name f{fn, nullptr};
  LF_REQUIRE(rows > 0 && cols > 0, f + ": dimensions must be positive");
  LF_REQUIRE(cols <= most_cols, f + ": rows are at most " + std::to_string(most_cols) + " wide");
  LF_REQUIRE(rows * (long long)LF_CHECKPOINT_PITCH(cols) <= MOST_ELEMENTS, f + ": more than 2^34 elements");
  return LF_OK;
}

inline int check_act(const char* fn, const char* name, const void* p, int dt) {
  const Name f{fn, nullptr};
  LF_REQUIRE(act_dtype_ok(dt), f + ": dtypes are f32, f16 or bf16");
  LF_REQUIRE(aligned(p, act_bytes(dt)), f + ": " + name + " is not aligned to its type");
  return LF_OK;
}

inline int check_vec(const char* fn, const char* name, const void* p, bool optional = false) {
  const Name f{fn, nullptr};
  LF_REQUIRE(p || optional, f + ": " + name + " is NULL");
  LF_REQUIRE(aligned(p, 4), f + ": " + name + " is not aligned to its type");
  return LF_OK;
}

// Scratch of a call: the caller's, or the context's workspace.  The workspace moves when a later call
// grows it, which a captured graph would not see.
inline int take_scratch(lf_context* ctx, const char* fn, void* given, size_t given_bytes, size_t need, void** out) {
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

inline size_t up(size_t n) { return (n + 255) & ~size_t(255); }

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

}  // namespace lf

#define LF_TRAIN_ENTRY(fn, argtype, impl)                                                    \
  int fn(lf_context* ctx, const argtype* args) {                                             \
    return lf::guarded([&]() -> int {                                                        \
      if (!ctx || !args) return lf::set_error(LF_ERR_INVALID, #fn ": NULL context or args"); \
      lf::DeviceScope device(ctx->device);                                                   \
      return lf::impl(ctx, *args);                                                           \
    });                                                                                      \
  }

