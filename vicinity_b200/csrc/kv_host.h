// Argument checks and the exception barrier shared by the entry points of the
// cache section of the C ABI (rotary.cu, kv_cache.cu).
#pragma once

#include <new>
#include <string>

#include "elements.cuh"
#include "host.h"

namespace vg {

// Runs an entry point's body; nothing throws across the ABI.
template <class F>
int guarded(F &&f) {
  try {
    try {
      return f();
    } catch (const std::bad_alloc &) {
      set_last_error("host memory");  // short: no allocation
      return VG_ERR_OTHER;
    } catch (const std::exception &e) {
      return fail(VG_ERR_OTHER, e.what());
    }
  } catch (...) {
    return VG_ERR_OTHER;
  }
}

inline int check_device(int device) {
  int count = 0;
  if (cudaGetDeviceCount(&count) != cudaSuccess || device < 0 || device >= count) {
    cudaGetLastError();
    return fail(VG_ERR_CUDA, "no CUDA device " + std::to_string(device) + " (the engine has no CPU path)");
  }
  return VG_OK;
}

inline int check_dtype(int dtype) {
  if (dtype != VG_F32 && dtype != VG_F16 && dtype != VG_BF16)
    return fail(VG_ERR_INVALID_PARAMETER, "dtype must be VG_F32, VG_F16 or VG_BF16");
  return VG_OK;
}

// An array of elements of `size` bytes.
inline int check_device_memory(const void *p, size_t size, int device, const char *name) {
  if (reinterpret_cast<uintptr_t>(p) % size)
    return fail(VG_ERR_INVALID_PARAMETER, std::string(name) + " is not aligned to its elements");
  cudaPointerAttributes a{};
  const bool known = p && cudaPointerGetAttributes(&a, p) == cudaSuccess;
  if (!known) cudaGetLastError();
  if (!known || !(a.type == cudaMemoryTypeManaged || (a.type == cudaMemoryTypeDevice && a.device == device)))
    return fail(VG_ERR_INVALID_PARAMETER,
                std::string(name) + " must be device memory of device " + std::to_string(device));
  return VG_OK;
}

// A tensor of `tokens` > 0 tokens: its memory, alignment and strides; an
// output's rows may not overlap.
inline int check_heads(const vg_heads *t, const char *name, size_t tokens, size_t dim, int dtype, int device,
                       bool output) {
  if (!t || !t->data) return fail(VG_ERR_INVALID_PARAMETER, std::string(name) + " is null");
  if (t->num_heads == 0 || t->num_heads > 65535)
    return fail(VG_ERR_INVALID_PARAMETER, std::string(name) + " must have 1 to 65535 heads");
  if (t->token_stride < 0 || t->head_stride < 0)
    return fail(VG_ERR_INVALID_PARAMETER, std::string(name) + " has a negative stride");
  // the last element's byte offset has to fit in 63 bits
  const __int128 reach = static_cast<__int128>(t->token_stride) * (tokens - 1) +
                         static_cast<__int128>(t->head_stride) * (t->num_heads - 1) + dim;
  if (reach > (static_cast<__int128>(1) << 60))
    return fail(VG_ERR_INVALID_PARAMETER, std::string(name) + " has strides out of range");
  if (output) {
    const int64_t T = static_cast<int64_t>(tokens), H = static_cast<int64_t>(t->num_heads), D = static_cast<int64_t>(dim);
    const int64_t ts = t->token_stride, hs = t->head_stride;
    const bool heads_in_token = (H == 1 || hs >= D) && (T == 1 || ts >= (H - 1) * hs + D);
    const bool tokens_in_head = (T == 1 || ts >= D) && (H == 1 || hs >= (T - 1) * ts + D);
    if (!heads_in_token && !tokens_in_head)
      return fail(VG_ERR_INVALID_PARAMETER, std::string(name) + " is written to: its rows must not overlap");
  }
  return check_device_memory(t->data, element_size(dtype), device, name);
}

inline Strided strided(const vg_heads &t) { return Strided{t.data, t.token_stride, t.head_stride}; }

}  // namespace vg
