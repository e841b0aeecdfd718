// Device helpers shared by the attention kernels of the 8-bit cache.
#pragma once

#include <cuda_fp16.h>

#include <stdint.h>

#include <atomic>

#include "elements.cuh"
#include "kv_cache.h"
#include "pipeline.cuh"

namespace vg {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
#define VG_INF __int_as_float(0x7f800000)

// A row has two references, which may lag by kLazy (fewer rescalings): nu of
// the scores x and mu = nu + lift of x + log2(value scale), lift a whole number.
// Probabilities are P = 2^(x + log2 vs - mu + kPShift) in binary16: at most
// 2^15, and they vanish below 2^-38 of the largest, which is a power of two when
// the references move to it (a row that one token dominates has its value, not
// rounded twice).  The denominator is the sum of 2^(x - nu) =
// P 2^(lift - kPShift) / vs in f32, which no value scale can overflow.  Where vs
// is so small beside the row's others that P would vanish in f32 too, its
// exponent is held at x - nu - kFar: 0 in binary16 all the same, but still there
// for the denominator.  nu starts at kUnseen, the lowest number: below every
// score but -inf, and differences stay defined.
constexpr float kUnseen = -3.402823466e38f;
// Scores beyond this (in binary logarithms) take their reference off before
// anything else is added, in two roundings instead of one multiply-add.
constexpr float kLargeScore = 1024.0f;
constexpr float kPShift = 13.0f, kLazy = 2.0f, kFar = 32.0f, kFarFactor = 4294967296.0f;

// 2 ulp; 0 below 2^-126
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}

// Two of the code bytes c of x (biased by 128), picked by the selector, as a
// binary16 pair: 0x6400 | u is 1024 + u.
template <uint32_t kSel>
__device__ __forceinline__ uint32_t half2_of(uint32_t x) {
  const uint32_t m = __byte_perm(x, 0x64646464u, kSel), bias = 0x64806480u;  // 1152
  const __half2 h = __hsub2(*reinterpret_cast<const __half2 *>(&m), *reinterpret_cast<const __half2 *>(&bias));
  return *reinterpret_cast<const uint32_t *>(&h);
}

// c += a b: A 16 x 16 and B 16 x 8 in binary16, C in f32
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void cp_async16(void *dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async4(void *dst, const void *src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// The power of two s (and 1 / s) that brings a row of largest magnitude `top`
// to [1, 2) (below 4 at the very end of the range); 1 where there is none.
__device__ __forceinline__ void row_scale(float top, float &s, float &inv) {
  const uint32_t e = __float_as_uint(top) >> 23;
  const uint32_t c = top == 0.0f || e >= 255u ? 127u : min(max(e, 1u), 253u);
  s = __uint_as_float(c << 23);
  inv = __uint_as_float((254u - c) << 23);
}

// log2 and reciprocal of a value scale (a power of two); a scale that is NaN
// counts as 1 here: the probabilities it meets are made NaN instead, so that
// the denominators stay what they are
__device__ __forceinline__ float log2_scale(float s) {
  return s == s ? static_cast<float>(static_cast<int>(__float_as_uint(s) >> 23) - 127) : 0.0f;
}
__device__ __forceinline__ float inverse_scale(float s) {
  return s == s ? __uint_as_float(0x7f000000u - __float_as_uint(s)) : 1.0f;
}

// What P of a block of value scale 2^lv takes: what is added to its scores, and
// what P is multiplied by for its share of the denominator.
struct PowerRefs {
  float nu, lift, ratio;
  __device__ __forceinline__ PowerRefs(float nu_, float lift_) {
    nu = nu_;
    lift = lift_;
    ratio = exp2_approx(lift - kPShift);
  }
  // added to x - nu, and to x itself (unless a score is so large that the rest is lost in it)
  __device__ __forceinline__ float shift(float lv) const { return fmaxf(lv + (kPShift - lift), -kFar); }
  __device__ __forceinline__ float exponent(float lv) const { return shift(lv) - nu; }
  __device__ __forceinline__ float share(float per_v) const { return fminf(per_v * ratio, kFarFactor); }
};

// Takes nu to within 1/2 of n, the largest x, and mu up to the largest
// x + log2 vs, which is n + over, where these are larger: the denominator l
// shrinks, the sum of values has to shrink by the result.  All in differences
// from the largest score, which stay exact however large the scores are.
__device__ __forceinline__ float raise_references(float &nu, float &lift, float n, float over, float &l) {
  const float at = fmaxf(nu, n), top = fmaxf((nu - at) + lift, (n - at) + over), less = rintf(-top);
  const float to = at + (top + less), by = nu - to;
  const float c = exp2_approx(by + (lift + less));
  l *= exp2_approx(by);
  nu = to;
  lift = -less;
  return c;
}

// Cached tokens that query qi of a sequence sees.
__device__ __forceinline__ uint32_t tokens_seen(const PlanSeq &ps, uint32_t qi, bool causal) {
  const uint32_t behind = ps.count - 1 - qi;
  return !causal ? ps.len : ps.len > behind ? ps.len - behind : 0;
}

// Allows a kernel its shared memory, once per device.
template <class Kernel>
cudaError_t allow_smem(Kernel *kern, size_t bytes, std::atomic<uint64_t> &done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || (dev < 64 && (done.load(std::memory_order_acquire) >> dev & 1))) return e;
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
  if (e == cudaSuccess && dev < 64) done.fetch_or(uint64_t(1) << dev, std::memory_order_release);
  return e;
}

// The result of one row from its sums: 8 dimensions from c on, and the lse.
__device__ __forceinline__ void finish_row(const AttendArgs &a, size_t token, uint32_t hq, uint32_t c, bool ovec,
                                           float nu, float lift, float sum, float (&y)[8]) {
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;  // no token seen: 0
  const float ratio = sum == 0.0f ? 0.0f : exp2_approx(lift - kPShift);
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = y[i] * inv * ratio;
  store8_16(a.out.p, static_cast<int64_t>(token) * a.out.token + static_cast<int64_t>(hq) * a.out.head + c,
            a.dtype == VG_F16, ovec, y);
  if (c == 0) {
    const float rest = log2f(sum);  // -inf: no token seen
    if (a.lse) a.lse[token * a.q_heads + hq] = (nu + rest) * kLn2;
    if (a.lse2) a.lse2[token * a.q_heads + hq] = sum == 0.0f ? make_float2(0.0f, VG_INF) : make_float2(nu, rest);
  }
}

}  // namespace vg
