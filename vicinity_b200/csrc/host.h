// Host-side helpers shared by the files that implement C entry points: error
// reporting through vg_last_error, the device guard and owning device buffers.
#pragma once

#include <cuda_runtime.h>

#include <cstddef>
#include <string>

#include "vicinity_gpu.h"

namespace vg {

void set_last_error(const char *msg);

inline int fail(int code, const std::string &msg) {
  set_last_error(msg.c_str());
  return code;
}

inline int cuda_fail(cudaError_t e, const char *what) {
  int code = e == cudaErrorMemoryAllocation ? VG_ERR_OUT_OF_MEMORY : VG_ERR_CUDA;
  cudaGetLastError();  // clear a sticky launch error so later calls start clean
  return fail(code, std::string(what) + ": " + cudaGetErrorString(e));
}

#define VG_CU(call)                                         \
  do {                                                      \
    cudaError_t vg_e_ = (call);                             \
    if (vg_e_ != cudaSuccess) return cuda_fail(vg_e_, #call); \
  } while (0)

#define VG_TRY(call)            \
  do {                          \
    int vg_s_ = (call);         \
    if (vg_s_ != VG_OK) return vg_s_; \
  } while (0)

struct DeviceGuard {
  int prev = -1;
  explicit DeviceGuard(int dev) {
    if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
    cudaSetDevice(dev);
  }
  ~DeviceGuard() {
    if (prev >= 0) cudaSetDevice(prev);
  }
};

// Owning device buffer with grow-only capacity.  reserve() discards contents.
struct DevBuf {
  void *p = nullptr;
  size_t cap = 0;
  DevBuf() = default;
  DevBuf(const DevBuf &) = delete;
  DevBuf &operator=(const DevBuf &) = delete;
  DevBuf(DevBuf &&o) noexcept : p(o.p), cap(o.cap) {
    o.p = nullptr;
    o.cap = 0;
  }
  DevBuf &operator=(DevBuf &&o) noexcept {
    if (this != &o) {
      release();
      p = o.p;
      cap = o.cap;
      o.p = nullptr;
      o.cap = 0;
    }
    return *this;
  }
  ~DevBuf() { release(); }
  cudaError_t reserve(size_t bytes) {
    if (bytes <= cap) return cudaSuccess;
    release();
    cudaError_t e = cudaMalloc(&p, bytes);
    if (e == cudaSuccess) cap = bytes;
    else p = nullptr;
    return e;
  }
  void release() {
    if (p) cudaFree(p);
    p = nullptr;
    cap = 0;
  }
  template <class T>
  T *as() const {
    return static_cast<T *>(p);
  }
};

inline bool is_device_ptr(const void *ptr) {
  if (!ptr) return false;
  cudaPointerAttributes a;
  if (cudaPointerGetAttributes(&a, ptr) != cudaSuccess) {
    cudaGetLastError();
    return false;
  }
  return a.type == cudaMemoryTypeDevice || a.type == cudaMemoryTypeManaged;
}

}  // namespace vg
