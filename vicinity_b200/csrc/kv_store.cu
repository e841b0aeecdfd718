// Writing, reading and cutting down a key/value cache held in 8 bits.
//
// A block of `block` tokens of one (sequence, head) has one scale s for its
// keys and one for its values, a power of two, so x / s, the rounding of a
// code to a larger scale and code * s are exact in f32 (codes * s even in
// bfloat16): the stored codes are a function of the inputs alone, the same
// in any precision, at the price of up to one of the eight bits (a scale of
// max |x| / 127 would use the whole range, but rounds in every product).
#include "common.cuh"
#include "elements.cuh"
#include "kv_cache.h"

namespace vg {

namespace {

constexpr int kMinExp = -100, kMaxExp = 120;

__device__ __forceinline__ float pow2(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

// The smallest 2^e, e in [kMinExp, kMaxExp], with 127 * 2^e >= |x|, from the
// bits of |x|: |x| = m 2^(x-126), m in [0.5, 1); 127/128 has mantissa 0x7e0000.
__device__ __forceinline__ float scale_of(uint32_t absbits) {
  if (absbits >= 0x7f800000u) return __uint_as_float(0x7fffffffu);  // not finite: the block reads as NaN
  const int e = static_cast<int>(absbits >> 23) - 126 - 7 + ((absbits & 0x7fffffu) > 0x7e0000u ? 1 : 0);
  return pow2(min(max(e, kMinExp), kMaxExp));
}

// 1 / s of a scale (a power of two: exact; NaN stays NaN)
__device__ __forceinline__ float inverse(float s) {
  return s == s ? __uint_as_float(0x7f000000u - __float_as_uint(s)) : s;
}

__device__ __forceinline__ uint32_t code4(const float *x) {
  uint32_t r = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = min(max(__float2int_rn(x[i]), -127), 127);  // NaN: 0
    r |= static_cast<uint32_t>(c & 0xff) << (8 * i);
  }
  return r;
}

__device__ __forceinline__ void values4(uint32_t c, float s, float *x) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    x[i] = static_cast<float>(static_cast<int>(c << (24 - 8 * i)) >> 24) * s;
}

// Codes of scale `from` rounded to the scale `to` >= from.
__device__ __forceinline__ uint2 rescaled(uint2 c, float ratio) {
  float x[8];
  values4(c.x, ratio, x);
  values4(c.y, ratio, x + 4);
  return make_uint2(code4(x), code4(x + 4));
}

constexpr int kAppendThreads = 256;

// One CTA per (touched block, head, K or V).  Bound by memory: the new values
// are read once into registers (block * dim / 8 vectors of 8, at most 8 a
// thread), their largest magnitude is reduced over the CTA as bits (so
// infinities and NaN win), and the codes are written; the block's older codes
// are touched only if its scale grew.
template <class T>
__global__ void __launch_bounds__(kAppendThreads) kv_append_kernel(const KvView kv, const __grid_constant__ Plan plan,
                                                                   const Strided k, const Strided v, const bool kvec,
                                                                   const bool vvec) {
  __shared__ uint32_t part[kAppendThreads / 32];
  const PlanSeq &ps = plan.s[plan_find(plan, blockIdx.x)];
  const int which = blockIdx.z;
  const uint32_t head = blockIdx.y, nv = kv.dim / 8;
  const uint32_t b = (ps.len >> kv.block_shift) + (blockIdx.x - ps.unit0);
  const uint32_t blk0 = b << kv.block_shift;
  const uint32_t lo = max(ps.len, blk0), hi = min(ps.len + ps.count, blk0 + kv.block);
  const size_t r = static_cast<size_t>(ps.seq) * kv.heads + head;
  int8_t *codes = kv.codes[which] + (r * kv.stride + blk0) * kv.dim;
  float *scale = kv.scales[which] + r * (kv.stride >> kv.block_shift) + b;
  const Strided &in = which ? v : k;
  const bool vec = which ? vvec : kvec;
  const T *src = static_cast<const T *>(in.p) + static_cast<int64_t>(head) * in.head;
  const uint32_t total = (hi - lo) * nv;

  float x[8][8];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t e = threadIdx.x + i * kAppendThreads;
    if (e < total) {
      const uint32_t t = e / nv, c = e - t * nv;
      load8(src + static_cast<int64_t>(ps.row0 + lo - ps.len + t) * in.token + c * 8, vec, x[i]);
#pragma unroll
      for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(x[i][j]) & 0x7fffffffu);
    }
  }
  top = __reduce_max_sync(VG_FULL_MASK, top);
  if (lane_id() == 0) part[threadIdx.x >> 5] = top;
  const float s_old = lo > blk0 ? *scale : pow2(kMinExp);
  __syncthreads();  // the old scale has been read by all
#pragma unroll
  for (int w = 0; w < kAppendThreads / 32; ++w) top = max(top, part[w]);
  const float s_top = scale_of(top);
  const float s_new = s_old != s_old || s_top != s_top ? s_old + s_top : fmaxf(s_old, s_top);
  const float inv = inverse(s_new);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t e = threadIdx.x + i * kAppendThreads;
    if (e < total) {
      float y[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = x[i][j] * inv;
      *reinterpret_cast<uint2 *>(codes + (static_cast<size_t>(lo - blk0) * nv + e) * 8) =
          make_uint2(code4(y), code4(y + 4));
    }
  }
  if (lo > blk0 && s_new > s_old) {
    const float ratio = s_old * inv;  // 2^-k; rounds to 0 only where every code does
    for (uint32_t e = threadIdx.x; e < (lo - blk0) * nv; e += kAppendThreads) {
      uint2 *c = reinterpret_cast<uint2 *>(codes) + e;
      *c = rescaled(*c, ratio);
    }
  }
  if (threadIdx.x == 0) *scale = s_new;
  if (which == 0)
    for (uint32_t t = lo + threadIdx.x; t < hi; t += kAppendThreads) kv.weights[r * kv.stride + t] = 0.0f;
}

constexpr int kReadThreads = 256;

// One CTA per (tile of tokens, head, K or V): codes times their block's scale.
template <class T>
__global__ void __launch_bounds__(kReadThreads) kv_read_kernel(const KvView kv, const __grid_constant__ Plan plan,
                                                               const Strided k, const Strided v, const bool kvec,
                                                               const bool vvec) {
  const PlanSeq &ps = plan.s[plan_find(plan, blockIdx.x)];
  const int which = blockIdx.z;
  const uint32_t head = blockIdx.y, nv = kv.dim / 8;
  const uint32_t t0 = (blockIdx.x - ps.unit0) * kReadTile, n = min(kReadTile, ps.count - t0);
  const size_t r = static_cast<size_t>(ps.seq) * kv.heads + head;
  const int8_t *codes = kv.codes[which] + r * kv.stride * kv.dim;
  const float *scales = kv.scales[which] + r * (kv.stride >> kv.block_shift);
  const Strided &to = which ? v : k;
  const bool vec = which ? vvec : kvec;
  T *dst = static_cast<T *>(to.p) + static_cast<int64_t>(head) * to.head;
  for (uint32_t e = threadIdx.x; e < n * nv; e += kReadThreads) {
    const uint32_t i = e / nv, c = e - i * nv, t = ps.len + t0 + i;
    const uint2 w = *reinterpret_cast<const uint2 *>(codes + static_cast<size_t>(t) * kv.dim + c * 8);
    const float s = scales[t >> kv.block_shift];
    float x[8];
    values4(w.x, s, x);
    values4(w.y, s, x + 4);
    store8(dst + static_cast<int64_t>(ps.row0 + t0 + i) * to.token + c * 8, vec, x);
  }
}

// ---- eviction ---------------------------------------------------------------

constexpr int kSelectThreads = 1024;

// The order in which tokens are kept: recent ones first, then by weight
// (any NaN counts as the largest, -0 as 0), ties to the older.  In integers:
// the sign of a NaN is not defined after arithmetic.
__device__ __forceinline__ uint32_t keep_key(const float *w, uint32_t t, uint32_t recent0) {
  const float x = w[t];
  const uint32_t mag = __float_as_uint(x) & 0x7fffffffu;
  if (t >= recent0) return 0xffffffffu;
  if (mag > 0x7f800000u) return 0xfffffffeu;
  return mag == 0 ? 0x80000000u : order_key(x);
}

// One CTA per (sequence, head): radix selection of the budget-th largest key,
// eight bits at a time, then the kept tokens in order by a prefix sum over
// (key above the threshold, key equal to it and among the first of those).
__global__ void __launch_bounds__(kSelectThreads) kv_select_kernel(const KvView kv, const __grid_constant__ Plan plan,
                                                                   const uint32_t budget, const uint32_t recent,
                                                                   int32_t *kept) {
  __shared__ uint32_t hist[256];
  __shared__ uint32_t sh_prefix, sh_need;
  __shared__ uint32_t warp_sum[kSelectThreads / 32][2];
  const uint32_t entry = blockIdx.x, head = blockIdx.y;
  const PlanSeq &ps = plan.s[entry];
  const uint32_t len = ps.len;
  const float *w = kv.weights + (static_cast<size_t>(ps.seq) * kv.heads + head) * kv.stride;
  float *wd = kv.weights + (static_cast<size_t>(ps.row0) * kv.heads + head) * kv.stride;
  int32_t *out = kept + (static_cast<size_t>(entry) * kv.heads + head) * budget;
  const uint32_t keep = min(len, budget);
  for (uint32_t i = keep + threadIdx.x; i < budget; i += kSelectThreads) {
    out[i] = -1;
    if (i < kv.stride) wd[i] = 0.0f;
  }
  if (len <= budget) {
    for (uint32_t i = threadIdx.x; i < len; i += kSelectThreads) {
      out[i] = static_cast<int32_t>(i);
      wd[i] = w[i];
    }
    return;
  }
  const uint32_t recent0 = len - min(recent, len);
  uint32_t prefix = 0, need = budget;  // the need-th largest among the keys that start with prefix
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (uint32_t i = threadIdx.x; i < 256; i += kSelectThreads) hist[i] = 0;
    __syncthreads();
    for (uint32_t t = threadIdx.x; t < len; t += kSelectThreads) {
      const uint32_t key = keep_key(w, t, recent0);
      if (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8)))
        atomicAdd(&hist[(key >> shift) & 255u], 1u);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      uint32_t d = 255;
      while (hist[d] < need) need -= hist[d--];
      sh_prefix = prefix | (d << shift);
      sh_need = need;
    }
    __syncthreads();
    prefix = sh_prefix;
    need = sh_need;
    __syncthreads();
  }
  // prefix: the threshold; the first `need` keys equal to it are kept
  uint32_t base_gt = 0, base_eq = 0;
  const int warp = threadIdx.x >> 5, lane = lane_id();
  for (uint32_t t0 = 0; t0 < len; t0 += kSelectThreads) {
    const uint32_t t = t0 + threadIdx.x;
    const uint32_t key = t < len ? keep_key(w, t, recent0) : 0;
    const bool gt = t < len && key > prefix, eq = t < len && key == prefix;
    const uint32_t mg = __ballot_sync(VG_FULL_MASK, gt), me = __ballot_sync(VG_FULL_MASK, eq);
    if (lane == 0) {
      warp_sum[warp][0] = __popc(mg);
      warp_sum[warp][1] = __popc(me);
    }
    __syncthreads();
    uint32_t pg = base_gt, pe = base_eq, ag = 0, ae = 0;
    for (int i = 0; i < kSelectThreads / 32; ++i) {
      if (i < warp) {
        pg += warp_sum[i][0];
        pe += warp_sum[i][1];
      }
      ag += warp_sum[i][0];
      ae += warp_sum[i][1];
    }
    const uint32_t below = (1u << lane) - 1u;
    pg += __popc(mg & below);
    pe += __popc(me & below);
    if (gt || (eq && pe < need)) {
      const uint32_t at = pg + min(pe, need);
      out[at] = static_cast<int32_t>(t);
      wd[at] = w[t];
    }
    base_gt += ag;
    base_eq += ae;
    __syncthreads();
  }
}

constexpr int kGatherThreads = 256;

// One CTA per (destination block, head, K or V): its scale is the largest of
// its tokens' scales (NaN if one is), and each token's codes are moved, rounded
// to that scale where their own is smaller.
__global__ void __launch_bounds__(kGatherThreads) kv_gather_kernel(const KvView kv, const __grid_constant__ Plan plan,
                                                                   const uint32_t budget, const int32_t *kept) {
  __shared__ float from[128];
  __shared__ int32_t at[128];
  __shared__ uint32_t top;
  const uint32_t entry = plan_find(plan, blockIdx.x);
  const PlanSeq &ps = plan.s[entry];
  const int which = blockIdx.z;
  const uint32_t head = blockIdx.y, nv = kv.dim / 8;
  const uint32_t b = blockIdx.x - ps.unit0, blk0 = b << kv.block_shift;
  const uint32_t n = min(kv.block, min(ps.len, budget) - blk0);
  const size_t nb = kv.stride >> kv.block_shift;
  const size_t rs = static_cast<size_t>(ps.seq) * kv.heads + head, rd = static_cast<size_t>(ps.row0) * kv.heads + head;
  const int8_t *src = kv.codes[which] + rs * kv.stride * kv.dim;
  int8_t *dst = kv.codes[which] + (rd * kv.stride + blk0) * kv.dim;
  if (threadIdx.x == 0) top = 0;
  __syncthreads();
  if (threadIdx.x < n) {
    const int32_t t = kept[(static_cast<size_t>(entry) * kv.heads + head) * budget + blk0 + threadIdx.x];
    at[threadIdx.x] = t;
    const float s = kv.scales[which][rs * nb + (static_cast<uint32_t>(t) >> kv.block_shift)];
    from[threadIdx.x] = s;
    atomicMax(&top, __float_as_uint(s) & 0x7fffffffu);  // positive: ordered by their bits, NaN last
  }
  __syncthreads();
  const float s_new = __uint_as_float(top), inv = inverse(s_new);
  for (uint32_t e = threadIdx.x; e < n * nv; e += kGatherThreads) {
    const uint32_t i = e / nv, c = e - i * nv;
    uint2 w = *reinterpret_cast<const uint2 *>(src + static_cast<size_t>(at[i]) * kv.dim + c * 8);
    const float ratio = from[i] * inv;
    if (ratio < 1.0f) w = rescaled(w, ratio);
    *reinterpret_cast<uint2 *>(dst + static_cast<size_t>(e) * 8) = w;
  }
  if (threadIdx.x == 0) kv.scales[which][rd * nb + b] = s_new;
}

}  // namespace

cudaError_t launch_kv_append(const KvView &kv, const Plan &plan, int dtype, const Strided &k, const Strided &v,
                             cudaStream_t s) {
  if (plan.units == 0) return cudaSuccess;
  const bool kvec = rows_aligned(k, element_size(dtype)), vvec = rows_aligned(v, element_size(dtype));
  return with_type(dtype, [&](auto t) {
    kv_append_kernel<decltype(t)><<<dim3(plan.units, kv.heads, 2), kAppendThreads, 0, s>>>(kv, plan, k, v, kvec, vvec);
    return cudaGetLastError();
  });
}

cudaError_t launch_kv_read(const KvView &kv, const Plan &plan, int dtype, const Strided &k, const Strided &v,
                           cudaStream_t s) {
  if (plan.units == 0) return cudaSuccess;
  const bool kvec = rows_aligned(k, element_size(dtype)), vvec = rows_aligned(v, element_size(dtype));
  return with_type(dtype, [&](auto t) {
    kv_read_kernel<decltype(t)><<<dim3(plan.units, kv.heads, 2), kReadThreads, 0, s>>>(kv, plan, k, v, kvec, vvec);
    return cudaGetLastError();
  });
}

cudaError_t launch_kv_select(const KvView &kv, const Plan &plan, uint32_t budget, uint32_t recent, int32_t *kept,
                             cudaStream_t s) {
  kv_select_kernel<<<dim3(plan.n, kv.heads), kSelectThreads, 0, s>>>(kv, plan, budget, recent, kept);
  return cudaGetLastError();
}

cudaError_t launch_kv_gather(const KvView &kv, const Plan &plan, uint32_t budget, const int32_t *kept,
                             cudaStream_t s) {
  if (plan.units == 0) return cudaSuccess;
  kv_gather_kernel<<<dim3(plan.units, kv.heads, 2), kGatherThreads, 0, s>>>(kv, plan, budget, kept);
  return cudaGetLastError();
}

}  // namespace vg
