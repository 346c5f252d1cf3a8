// Host-side pieces that every file behind the C ABI shares: failure classes,
// the exception fence, device buffers and the streams that handles run on.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <memory>
#include <stdexcept>
#include <string>

#include "../../include/mixmoe.h"

// The message of the calling thread's last failure (mxm_last_error).
extern thread_local std::string g_last_error;

// Failure classes of the bridge's status codes (gpu/mlx_bridge.cpp:814-823):
// an argument the call cannot accept (MXM_ERR_ARGS), a runtime that is not
// initialised (MXM_ERR_INIT); every other failure -- a HIP error, a call out
// of sequence -- is MXM_ERR.
struct ArgError : std::runtime_error {
  using std::runtime_error::runtime_error;
};
struct InitError : std::runtime_error {
  using std::runtime_error::runtime_error;
};

template <class Ex>
[[noreturn]] void vthrow(const char* fmt, va_list ap) {
  char buf[512];
  vsnprintf(buf, sizeof buf, fmt, ap);
  throw Ex(buf);
}

// An argument error (shape, dtype, index, size limit, NULL pointer).
[[noreturn]] inline void fail(const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vthrow<ArgError>(fmt, ap);
}
// A runtime failure or a call out of sequence.
[[noreturn]] inline void fail_rt(const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vthrow<std::runtime_error>(fmt, ap);
}
// The HIP runtime or the device is not (or cannot be) initialised.
[[noreturn]] inline void fail_init(const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vthrow<InitError>(fmt, ap);
}

#define HIPCK(expr)                                                                       \
  do {                                                                                    \
    hipError_t _e = (expr);                                                               \
    if (_e != hipSuccess)                                                                 \
      fail_rt("HIP error %s at %s:%d", hipGetErrorString(_e), __FILE__, __LINE__);       \
  } while (0)

template <typename F>
int fenced(F&& f) {
  try {
    return f();
  } catch (const ArgError& e) {
    g_last_error = e.what();
    return MXM_ERR_ARGS;
  } catch (const InitError& e) {
    g_last_error = e.what();
    return MXM_ERR_INIT;
  } catch (const std::exception& e) {
    g_last_error = e.what();
    return MXM_ERR;
  } catch (...) {
    g_last_error = "unknown exception";
    return MXM_ERR;
  }
}

struct DevBuf {
  void* p = nullptr;
  size_t bytes = 0;
  DevBuf() = default;
  DevBuf(const DevBuf&) = delete;
  DevBuf& operator=(const DevBuf&) = delete;
  ~DevBuf() { reset(); }
  void alloc(size_t n) {
    reset();
    if (n == 0) n = 256;
    HIPCK(hipMalloc(&p, n));
    bytes = n;
  }
  void reset() {
    if (p) (void)hipFree(p);
    p = nullptr;
    bytes = 0;
  }
  template <typename T>
  T* as() const { return static_cast<T*>(p); }
};

// A stream on `dev`, which has to be the current device; it lives as long as
// the last handle that runs on it.
struct StreamRef {
  hipStream_t stream = nullptr;
  int device = 0;
  explicit StreamRef(int dev) : device(dev) {
    HIPCK(hipStreamCreateWithFlags(&stream, hipStreamNonBlocking));
  }
  StreamRef(const StreamRef&) = delete;
  StreamRef& operator=(const StreamRef&) = delete;
  ~StreamRef() {
    (void)hipStreamSynchronize(stream);
    (void)hipStreamDestroy(stream);
  }
};

// The stream of a live op handle, or null.
std::shared_ptr<StreamRef> mxm_op_stream(int64_t h);
// A handle number that no other handle of the process has had.
int64_t mxm_new_handle();
