// Loads and stores of 8 consecutive elements of a tensor in f32, binary16 or
// bfloat16, with one rounding to nearest on the way out.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <stdint.h>

#include "kv_cache.h"
#include "vicinity_gpu.h"

namespace vg {

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }

template <class T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// vec: p is 16-byte aligned.  Plain loads: an output may be its input, and then
// the memory is not read-only while the kernel runs.
template <class T>
__device__ __forceinline__ void load8(const T *p, bool vec, float (&x)[8]) {
  alignas(16) T e[8];
  if (vec) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i)
      reinterpret_cast<uint4 *>(e)[i] = reinterpret_cast<const uint4 *>(p)[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = p[i];
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = to_f32(e[i]);
}

template <class T>
__device__ __forceinline__ void store8(T *p, bool vec, const float (&x)[8]) {
  alignas(16) T e[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = from_f32<T>(x[i]);
  if (vec) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i)
      reinterpret_cast<uint4 *>(p)[i] = reinterpret_cast<uint4 *>(e)[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = e[i];
  }
}

// 8 consecutive 16-bit elements, binary16 or bfloat16 by a flag: for kernels
// that read or write them at their edges only.
__device__ __forceinline__ void load8_16(const void *base, int64_t at, bool f16, bool vec, float (&x)[8]) {
  if (f16) load8(static_cast<const __half *>(base) + at, vec, x);
  else load8(static_cast<const __nv_bfloat16 *>(base) + at, vec, x);
}
__device__ __forceinline__ void store8_16(void *base, int64_t at, bool f16, bool vec, const float (&x)[8]) {
  if (f16) store8(static_cast<__half *>(base) + at, vec, x);
  else store8(static_cast<__nv_bfloat16 *>(base) + at, vec, x);
}

// 16 elements as they lie in memory.
template <class T>
struct Raw16 {
  uint4 w[sizeof(T)];
  __device__ __forceinline__ void load(const T *p, bool vec) {
    if (vec) {
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(T)); ++i) w[i] = __ldg(reinterpret_cast<const uint4 *>(p) + i);
    } else {
      T *e = reinterpret_cast<T *>(w);
#pragma unroll
      for (int i = 0; i < 16; ++i) e[i] = p[i];
    }
  }
  __device__ __forceinline__ float at(int i) const { return to_f32(reinterpret_cast<const T *>(w)[i]); }
};

// Whether every row of a strided tensor starts on a 16-byte boundary.
inline bool rows_aligned(const Strided &t, size_t elem) {
  return reinterpret_cast<uintptr_t>(t.p) % 16 == 0 && (t.token * static_cast<int64_t>(elem)) % 16 == 0 &&
         (t.head * static_cast<int64_t>(elem)) % 16 == 0;
}

inline size_t element_size(int dtype) { return dtype == VG_F32 ? 4 : 2; }

// f(T{}) with T the element type of dtype (checked by the caller)
template <class F>
cudaError_t with_type(int dtype, F &&f) {
  if (dtype == VG_F32) return f(float{});
  if (dtype == VG_F16) return f(__half{});
  return f(__nv_bfloat16{});
}

}  // namespace vg
