// Registry and helpers of the handles around the MoE op (residual norms, gradient
// sets, token embeddings, token losses): each has a stream of its own or shares
// another handle's.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <map>
#include <memory>
#include <mutex>

#include "mxm_host.h"

struct TrainHandle {
  std::shared_ptr<StreamRef> stream_ref;
  int n_cu = 256;
  virtual ~TrainHandle() = default;
  hipStream_t stream() const { return stream_ref->stream; }
};

inline std::mutex g_train_mu;
inline std::map<int64_t, std::shared_ptr<TrainHandle>> g_train;

inline std::shared_ptr<TrainHandle> find(int64_t h) {
  std::lock_guard<std::mutex> lk(g_train_mu);
  const auto it = g_train.find(h);
  return it == g_train.end() ? nullptr : it->second;
}
template <class T>
std::shared_ptr<T> get(int64_t h) {
  return std::dynamic_pointer_cast<T>(find(h));
}

inline std::shared_ptr<StreamRef> stream_of_handle(int64_t h) {
  if (auto s = mxm_op_stream(h)) return s;
  const auto t = find(h);
  return t ? t->stream_ref : nullptr;
}

// Makes `dev` current for a call and puts the caller's device back.
struct DeviceGuard {
  int prev = -1;
  bool moved = false;
  explicit DeviceGuard(int dev) {
    HIPCK(hipGetDevice(&prev));
    if (prev != dev) {
      HIPCK(hipSetDevice(dev));
      moved = true;
    }
  }
  ~DeviceGuard() {
    if (moved) (void)hipSetDevice(prev);
  }
};

inline int64_t keep(std::shared_ptr<TrainHandle> t) {
  const int64_t h = mxm_new_handle();
  std::lock_guard<std::mutex> lk(g_train_mu);
  g_train[h] = std::move(t);
  return h;
}

template <class T>
int destroy(int64_t h, const char* what) {
  return fenced([&] {
    std::shared_ptr<TrainHandle> victim;
    {
      std::lock_guard<std::mutex> lk(g_train_mu);
      const auto it = g_train.find(h);
      if (it == g_train.end() || !dynamic_cast<T*>(it->second.get())) {
        g_last_error = std::string(what) + " invalid handle";
        return MXM_ERR_OP;
      }
      victim = std::move(it->second);
      g_train.erase(it);
    }
    return MXM_OK;
  });
}

#define HANDLE_OR_RETURN(T, var, h, what)          \
  const std::shared_ptr<T> var = get<T>(h);        \
  if (!var) {                                      \
    g_last_error = what " invalid handle";         \
    return MXM_ERR_OP;                             \
  }

inline bool float_dtype(int64_t t) { return t == MXM_DTYPE_F32 || t == MXM_DTYPE_BF16; }

inline void check_pointer(const char* what, const char* name, const void* p, bool bf16, bool required) {
  if (!p && required) fail("%s %s must be non-NULL", what, name);
  if (reinterpret_cast<uintptr_t>(p) % (bf16 ? 2 : 4) != 0)
    fail("%s %s is not aligned to its elements", what, name);
}

// The stream of `stream_of`, or a new one on the current device.
inline std::shared_ptr<StreamRef> choose_stream(std::shared_ptr<StreamRef> shared) {
  if (shared) return shared;
  int dev = 0;
  HIPCK(hipGetDevice(&dev));
  return std::make_shared<StreamRef>(dev);
}

inline std::shared_ptr<StreamRef> shared_stream(const char* what, int64_t stream_of) {
  if (stream_of == 0) return nullptr;
  auto s = stream_of_handle(stream_of);
  if (!s) fail("%s stream_of %lld is not a live handle", what, (long long)stream_of);
  return s;
}

// The device of a shared stream, or the current one.
inline int device_of(const std::shared_ptr<StreamRef>& shared) {
  if (shared) return shared->device;
  int dev = 0;
  HIPCK(hipGetDevice(&dev));
  return dev;
}

inline int cu_count(int device) {
  int n = 0;
  HIPCK(hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, device));
  return n;
}
