// Shared host-side helpers of the hipattn library: error convention, tensor
// descriptor checks, stream lookup.  Device code lives in the .hip files.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <stdexcept>
#include <string>

#include "../../include/hipattn.h"

namespace hipattn {

// Thrown inside the library, turned into the C ABI's `char*` by HA_PROTECT,
// the counterpart of the reference's PROTECT macro
// (rllm/tch-cuda/kernels/vllm_bindings.cpp:7-13).
struct Error : std::runtime_error {
  using std::runtime_error::runtime_error;
};

[[noreturn]] inline void fail(const char *fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  throw Error(buf);
}

// Throws what another entry point of the library has returned, if that is an error.
inline void raise(char *err) {
  if (err == nullptr) return;
  const std::string msg(err);
  free(err);
  fail("%s", msg.c_str());
}

#define HA_CHECK(cond, ...)                 \
  do {                                      \
    if (!(cond)) ::hipattn::fail(__VA_ARGS__); \
  } while (0)

#define HA_HIP(call)                                                      \
  do {                                                                    \
    hipError_t ha_err_ = (call);                                          \
    if (ha_err_ != hipSuccess)                                            \
      ::hipattn::fail("%s failed: %s", #call, hipGetErrorString(ha_err_)); \
  } while (0)

#define HA_PROTECT(...)                  \
  try {                                  \
    __VA_ARGS__;                         \
    return nullptr;                      \
  } catch (const std::exception &e) {    \
    return strdup(e.what());             \
  } catch (...) {                        \
    return strdup("hipattn: unknown error"); \
  }

inline int dtype_size(int dtype) {
  switch (dtype) {
    case HIPATTN_F32: return 4;
    case HIPATTN_F16: return 2;
    case HIPATTN_BF16: return 2;
    case HIPATTN_I32: return 4;
    case HIPATTN_I64: return 8;
    case HIPATTN_U8: return 1;
  }
  fail("unknown dtype %d", dtype);
}

inline const char *dtype_name(int dtype) {
  switch (dtype) {
    case HIPATTN_F32: return "f32";
    case HIPATTN_F16: return "f16";
    case HIPATTN_BF16: return "bf16";
    case HIPATTN_I32: return "i32";
    case HIPATTN_I64: return "i64";
    case HIPATTN_U8: return "u8";
  }
  return "?";
}

inline bool is_float_dtype(int dtype) {
  return dtype == HIPATTN_F32 || dtype == HIPATTN_F16 || dtype == HIPATTN_BF16;
}

inline void check_tensor(const hipattn_tensor *t, const char *name, int ndim) {
  HA_CHECK(t != nullptr, "%s: tensor is NULL", name);
  HA_CHECK(t->ndim == ndim, "%s: expected %d dims, got %d", name, ndim, t->ndim);
  HA_CHECK(t->ndim <= HIPATTN_MAX_DIMS, "%s: too many dims", name);
  (void)dtype_size(t->dtype);
  for (int i = 0; i < t->ndim; i++)
    HA_CHECK(t->sizes[i] >= 0, "%s: negative size in dim %d", name, i);
}

inline int64_t numel(const hipattn_tensor *t) {
  int64_t n = 1;
  for (int i = 0; i < t->ndim; i++) n *= t->sizes[i];
  return n;
}

inline bool is_contiguous(const hipattn_tensor *t) {
  int64_t expect = 1;
  for (int i = t->ndim - 1; i >= 0; i--) {
    if (t->sizes[i] != 1 && t->strides[i] != expect) return false;
    expect *= t->sizes[i];
  }
  return true;
}

// Whether no byte between the first and the last element of one lies there of the other (strides not negative).
inline bool apart(const hipattn_tensor *a, const hipattn_tensor *b) {
  auto end = [](const hipattn_tensor *t) {
    int64_t last = 0;
    for (int i = 0; i < t->ndim; i++) last += (t->sizes[i] - 1) * t->strides[i];
    return static_cast<const char *>(t->data) + (last + 1) * dtype_size(t->dtype);
  };
  return numel(a) == 0 || numel(b) == 0 || end(a) <= static_cast<const char *>(b->data) || end(b) <= static_cast<const char *>(a->data);
}

inline void check_contiguous(const hipattn_tensor *t, const char *name) {
  HA_CHECK(numel(t) == 0 || is_contiguous(t), "%s must be contiguous", name);
}

inline void check_data(const hipattn_tensor *t, const char *name) {
  HA_CHECK(numel(t) == 0 || t->data != nullptr, "%s: data pointer is NULL", name);
}

inline void check_index_tensor(const hipattn_tensor *t, const char *name, int ndim) {
  check_tensor(t, name, ndim);
  HA_CHECK(t->dtype == HIPATTN_I32 || t->dtype == HIPATTN_I64,
           "%s must be int32 or int64, got %s", name, dtype_name(t->dtype));
  check_contiguous(t, name);
  check_data(t, name);
}

// The stream an op enqueues on: the argument if given, else the calling
// thread's current stream (hipattn_stream_set_current), else the default.
hipStream_t resolve_stream(void *stream);

inline void check_launch(const char *what) {
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) fail("%s: launch failed: %s", what, hipGetErrorString(e));
}

}  // namespace hipattn
