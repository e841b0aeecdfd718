// Writing, reading and cutting down a key/value cache held in 8 bits.
//
// A block of `block` tokens of one (sequence, head) has one scale s for its
// keys and one for its values, a power of two, so x / s, the rounding of a
// code to a larger scale and code * s are exact in f32 (codes * s even in
// bfloat16): the stored codes are a function of the inputs alone, the same
// in any precision, at the price of up to one of the eight bits (a scale of
// max |x| / 127 would use the whole range, but rounds in every product).
#include "chain.cuh"
#include "common.cuh"
#include "elements.cuh"
#include "kv_cache.h"

#include <algorithm>
#include <type_traits>

namespace vg {

namespace {

__device__ __forceinline__ float pow2(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

// The smallest 2^e, e in [kMinScaleExp, kMaxScaleExp], with 127 * 2^e >= |x|, from the
// bits of |x|: |x| = m 2^(x-126), m in [0.5, 1); 127/128 has mantissa 0x7e0000.
__device__ __forceinline__ float scale_of(uint32_t absbits) {
  if (absbits >= 0x7f800000u) return __uint_as_float(0x7fffffffu);  // not finite: the block reads as NaN
  const int e = static_cast<int>(absbits >> 23) - 126 - 7 + ((absbits & 0x7fffffu) > 0x7e0000u ? 1 : 0);
  return pow2(min(max(e, kMinScaleExp), kMaxScaleExp));
}

// 1 / s of a scale (a power of two: exact; NaN stays NaN)
__device__ __forceinline__ float inverse(float s) {
  return s == s ? __uint_as_float(0x7f000000u - __float_as_uint(s)) : s;
}

// Codes are rounded by adding 1.5 * 2^23: the sum's last byte is the nearest
// integer (ties to even) of a value below 2^22, and x times a power of two is
// exact inside the multiply-add.  The conversion instruction has a quarter of
// its rate.
__device__ __forceinline__ uint32_t rounded(float x, float factor) {
  return __float_as_uint(fmaf(x, factor, 12582912.0f));
}
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// 16 codes of raw elements.  exotic: the scale is NaN, or so large that it was
// clamped -- codes may saturate, and are 0 for NaN.
template <class T>
__device__ __forceinline__ uint4 codes16(const Raw16<T> &x, float inv, bool exotic) {
  uint32_t r[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) r[i] = rounded(x.at(i), inv);
  if (exotic) {
#pragma unroll
    for (int i = 0; i < 16; ++i) r[i] = min(max(__float2int_rn(x.at(i) * inv), -127), 127);  // NaN: 0
  }
  return make_uint4(pack4(r[0], r[1], r[2], r[3]), pack4(r[4], r[5], r[6], r[7]), pack4(r[8], r[9], r[10], r[11]),
                    pack4(r[12], r[13], r[14], r[15]));
}

// The value of byte i of a word of codes: biased by 128 it is the last byte of
// 2^23 + 128 + code (the conversion instruction has a quarter of the rate).
__device__ __forceinline__ float code_at(uint32_t c, int i) {
  return __uint_as_float(__byte_perm(c ^ 0x80808080u, 0x4b000000u, 0x7540 | i)) - 8388736.0f;
}

// Codes rounded to a larger scale; ratio = 2^-k (0 where every code vanishes).
__device__ __forceinline__ uint32_t rescaled4(uint32_t c, float ratio) {
  return pack4(rounded(code_at(c, 0), ratio), rounded(code_at(c, 1), ratio), rounded(code_at(c, 2), ratio),
               rounded(code_at(c, 3), ratio));
}
__device__ __forceinline__ uint4 rescaled(uint4 c, float ratio) {
  return make_uint4(rescaled4(c.x, ratio), rescaled4(c.y, ratio), rescaled4(c.z, ratio), rescaled4(c.w, ratio));
}

// A CTA's work: neighbouring CTAs take the heads of one block of tokens, whose
// rows lie next to each other in the caller's tensors.
struct StoreUnit {
  uint32_t unit, head;
  int which;  // 0: keys, 1: values
};
__device__ __forceinline__ StoreUnit store_unit(const KvView &kv) {
  const uint32_t u = blockIdx.x / kv.heads;
  return {u >> 1, blockIdx.x - u * kv.heads, static_cast<int>(u & 1)};
}
template <class P>
unsigned store_grid(const KvView &kv, const P &plan) { return plan.units * 2 * kv.heads; }

constexpr int kStoreThreads = 256;

// Item e of a block is 16 elements, chunk e % per of token e / per, per = dim / 16
// (2, 4, 6 or 8); e < 2^11.
__device__ __forceinline__ uint32_t item_token(uint32_t e, uint32_t per) {
  return (e * (per == 6 ? 10923u : 65536u / per)) >> 16;
}

// One CTA per (touched block, head, K or V).  Bound by memory: the new values
// are read once into registers (kItems of 16 a thread), their largest magnitude
// is reduced over the CTA as bits (so infinities and NaN win), and the codes
// are written; the block's older codes are touched only if its scale grew.
// 16,384 tokens x 8 heads x 128, keys and values in bf16: 22 us, 4.5 TB/s (the
// time between a CTA's loads and its stores is not covered by others' loads).
template <class T, int kItems, class P>
__global__ void __launch_bounds__(kStoreThreads) kv_append_kernel(const __grid_constant__ KvView kv,
                                                                  const __grid_constant__ P plan,
                                                                  const __grid_constant__ Strided k,
                                                                  const __grid_constant__ Strided v, const bool kvec,
                                                                  const bool vvec) {
  __shared__ uint32_t part[kStoreThreads / 32];
  const StoreUnit u = store_unit(kv);
  const PlanSeq &ps = plan.s[plan_find(plan, u.unit)];
  const uint32_t per = kv.dim / 16;
  const uint32_t b = (ps.len >> kv.block_shift) + (u.unit - ps.unit0);
  const uint32_t blk0 = b << kv.block_shift;
  const uint32_t lo = max(ps.len, blk0), hi = min(ps.len + ps.count, blk0 + kv.block);
  const size_t r = static_cast<size_t>(ps.seq) * kv.heads + u.head;
  uint4 *codes = reinterpret_cast<uint4 *>((u.which ? kv.codes[1] : kv.codes[0]) + (r * kv.stride + blk0) * kv.dim);
  float *scale = (u.which ? kv.scales[1] : kv.scales[0]) + r * (kv.stride >> kv.block_shift) + b;
  const Strided &in = u.which ? v : k;
  const bool vec = u.which ? vvec : kvec;
  const T *src = static_cast<const T *>(in.p) + static_cast<int64_t>(u.head) * in.head +
                 static_cast<int64_t>(ps.row0 + lo - ps.len) * in.token;
  const uint32_t total = (hi - lo) * per;

  Raw16<T> x[kItems];
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const uint32_t e = threadIdx.x + i * kStoreThreads, t = item_token(e, per);
    if (e < total) x[i].load(src + static_cast<int64_t>(t) * in.token + (e - t * per) * 16, vec);
  }
  const float s_old = lo > blk0 ? *scale : pow2(kMinScaleExp);
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < kItems; ++i)
    if (threadIdx.x + i * kStoreThreads < total) {
#pragma unroll
      for (int j = 0; j < 16; ++j) top = max(top, __float_as_uint(x[i].at(j)) & 0x7fffffffu);
    }
  top = __reduce_max_sync(VG_FULL_MASK, top);
  if (lane_id() == 0) part[threadIdx.x >> 5] = top;
  __syncthreads();  // the old scale has been read by all
#pragma unroll
  for (int w = 0; w < kStoreThreads / 32; ++w) top = max(top, part[w]);
  const float s_top = scale_of(top);
  const float s_new = s_old != s_old || s_top != s_top ? s_old + s_top : fmaxf(s_old, s_top);
  const float inv = inverse(s_new);
  const bool exotic = !(s_new < pow2(kMaxScaleExp));
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const uint32_t e = threadIdx.x + i * kStoreThreads;
    if (e < total) codes[(lo - blk0) * per + e] = codes16(x[i], inv, exotic);
  }
  if (lo > blk0 && s_new > s_old) {
    const float ratio = s_old * inv;
    for (uint32_t e = threadIdx.x; e < (lo - blk0) * per; e += kStoreThreads) codes[e] = rescaled(codes[e], ratio);
  }
  if (threadIdx.x == 0) *scale = s_new;
  if (u.which == 0)
    for (uint32_t t = lo + threadIdx.x; t < hi; t += kStoreThreads) kv.weights[r * kv.stride + t] = 0.0f;
}

// One CTA per (tile of tokens, head, K or V): codes times their block's scale.
// Bound by memory: the same 16,384 tokens into bf16 19 us, 5.3 TB/s.
template <class T, class P>
__global__ void __launch_bounds__(kStoreThreads) kv_read_kernel(const __grid_constant__ KvView kv,
                                                                const __grid_constant__ P plan,
                                                                const __grid_constant__ Strided k,
                                                                const __grid_constant__ Strided v, const bool kvec,
                                                                const bool vvec) {
  const StoreUnit u = store_unit(kv);
  const PlanSeq &ps = plan.s[plan_find(plan, u.unit)];
  const uint32_t per = kv.dim / 16;
  const uint32_t t0 = (u.unit - ps.unit0) * kReadTile, n = min(kReadTile, ps.count - t0);
  const size_t r = static_cast<size_t>(ps.seq) * kv.heads + u.head;
  const uint4 *codes =
      reinterpret_cast<const uint4 *>((u.which ? kv.codes[1] : kv.codes[0]) + (r * kv.stride + ps.len + t0) * kv.dim);
  const float *scales = (u.which ? kv.scales[1] : kv.scales[0]) + r * (kv.stride >> kv.block_shift);
  const Strided &to = u.which ? v : k;
  const bool vec = u.which ? vvec : kvec;
  T *dst = static_cast<T *>(to.p) + static_cast<int64_t>(u.head) * to.head +
           static_cast<int64_t>(ps.row0 + t0) * to.token;
  constexpr int kItems = 2;  // loads in flight
  for (uint32_t e0 = threadIdx.x; e0 < n * per; e0 += kItems * kStoreThreads) {
    uint4 w[kItems];
    float s[kItems];
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const uint32_t e = e0 + i * kStoreThreads;
      if (e < n * per) {
        w[i] = __ldg(codes + e);
        s[i] = __ldg(scales + ((ps.len + t0 + item_token(e, per)) >> kv.block_shift));
      }
    }
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const uint32_t e = e0 + i * kStoreThreads, t = item_token(e, per);
      if (e >= n * per) continue;
      T *out = dst + static_cast<int64_t>(t) * to.token + (e - t * per) * 16;
      const uint32_t c[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = code_at(c[2 * h + (j >> 2)], j & 3) * s[i];
        store8(out + 8 * h, vec, x);
      }
    }
  }
}

// ---- eviction ---------------------------------------------------------------

constexpr uint32_t kSelectThreads = 1024;

// The order in which tokens are kept: recent ones first, then by weight
// (any NaN counts as the largest, -0 as 0), ties to the older.  In integers:
// the sign of a NaN is not defined after arithmetic.
constexpr uint32_t kNewest = 0xffffffffu, kNone = 0x80000000u;  // keys of recent tokens and of weight 0
__device__ __forceinline__ uint32_t keep_key(float x, bool newest) {
  const uint32_t b = __float_as_uint(x), mag = b & 0x7fffffffu;
  uint32_t k = mag == 0 ? kNone : order_key(x);
  k = mag > 0x7f800000u ? kNewest - 1 : k;
  return newest ? kNewest : k;
}

// One CTA per (sequence, head): radix selection of the budget-th largest key by
// its first 12, then 10, then 10 bits, and the kept tokens in order by a prefix
// sum over (key above the threshold, key equal to it and among the first of
// those).  A thread takes kHeld consecutive tokens, in registers (kOne: the row
// is one round of the CTA), or round after round, read again in every pass.
// Bound by issue and latency: some 30 instructions a token on one SM, three
// histograms in shared memory with their scans, or fewer -- the search stops
// when a bin is kept whole.  12 bits spread weights of a few exponents over
// enough bins; the two keys that many tokens share, recent ones and weight 0,
// are counted in registers.  64 rows of 16,384 tokens: 14 us (4 MB: the memory
// would take 1); by bisection over a cluster of CTAs, two bits a step, 26.
template <bool kOne, uint32_t kHeld, class P>
__global__ void __launch_bounds__(kSelectThreads) kv_select_kernel(const __grid_constant__ KvView kv,
                                                                   const __grid_constant__ P plan,
                                                                   const uint32_t budget, const uint32_t recent,
                                                                   int32_t *kept) {
  __shared__ __align__(16) uint32_t hist[4096];
  __shared__ uint32_t warp_sum[2][32], sh_digit, sh_need, sh_count;
  chain_release();
  const uint32_t head = blockIdx.x, entry = blockIdx.y;
  const PlanSeq &ps = plan.s[entry];
  const uint32_t len = ps.len;
  const float *w = kv.weights + (static_cast<size_t>(ps.seq) * kv.heads + head) * kv.stride;
  float *wd = kv.weights + (static_cast<size_t>(ps.row0) * kv.heads + head) * kv.stride;
  int32_t *out = kept + (static_cast<size_t>(entry) * kv.heads + head) * budget;
  const uint32_t tid = threadIdx.x, threads = blockDim.x;
  for (uint32_t i = min(len, budget) + tid; i < budget; i += threads) {
    out[i] = -1;
    wd[i] = 0.0f;
  }
  if (len <= budget) {
    for (uint32_t i = tid; i < len; i += threads) {
      out[i] = static_cast<int32_t>(i);
      wd[i] = w[i];
    }
    return;
  }
  const uint32_t recent0 = len - min(recent, len);
  const int warp = tid >> 5, warps = threads >> 5, lane = lane_id();
  const uint32_t rounds = kOne ? 1 : (len + threads * kHeld - 1) / (threads * kHeld);
  // The keys of a round.  A row's memory goes on to a multiple of kKvPad
  // tokens, so whole vectors may be read where a token of them is held.
  uint32_t key[kHeld];
  uint32_t first = 0, mine = 0;
  auto load = [&](uint32_t round) {
    first = (round * threads + tid) * kHeld;
    mine = first < len ? min(kHeld, len - first) : 0;
#pragma unroll
    for (uint32_t i = 0; i < kHeld; i += 4) {
      float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (i < mine) x = *reinterpret_cast<const float4 *>(w + first + i);
      key[i] = keep_key(x.x, first + i >= recent0);
      key[i + 1] = keep_key(x.y, first + i + 1 >= recent0);
      key[i + 2] = keep_key(x.z, first + i + 2 >= recent0);
      key[i + 3] = keep_key(x.w, first + i + 3 >= recent0);
    }
  };
  if (kOne) load(0);

  uint32_t cut = 0, need = budget;  // kept: keys above cut, and the first `need` that equal it
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = 20 - 10 * pass;
    const uint32_t bins = pass ? 1024 : 4096;
    for (uint32_t i = tid; i < bins / 4; i += threads) reinterpret_cast<uint4 *>(hist)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    uint32_t newest = 0, none = 0;
    for (uint32_t r = 0; r < rounds; ++r) {
      if (!kOne) load(r);
#pragma unroll
      for (uint32_t i = 0; i < kHeld; ++i) {
        const uint32_t x = key[i];
        if (i >= mine) continue;
        if (pass) {
          if (x >> (shift + 10) == cut >> (shift + 10)) atomicAdd(hist + (x >> shift & 1023u), 1u);
        } else if (x == kNewest) {
          ++newest;
        } else if (x == kNone) {
          ++none;
        } else {
          atomicAdd(hist + (x >> 20), 1u);
        }
      }
    }
    if (pass == 0) {
      newest = __reduce_add_sync(VG_FULL_MASK, newest);
      none = __reduce_add_sync(VG_FULL_MASK, none);
      if (lane == 0 && newest) atomicAdd(hist + (kNewest >> 20), newest);
      if (lane == 0 && none) atomicAdd(hist + (kNone >> 20), none);
    }
    __syncthreads();
    // groups of four bins, from the top: the one that holds the need-th key
    const uint32_t groups = bins / 4, own = (groups + threads - 1) / threads;
    uint32_t sum = 0;
    for (uint32_t i = tid * own; i < min(groups, (tid + 1) * own); ++i) {
      const uint4 h = reinterpret_cast<const uint4 *>(hist)[groups - 1 - i];
      sum += h.x + h.y + h.z + h.w;
    }
    uint32_t inc = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t y = __shfl_up_sync(VG_FULL_MASK, inc, d);
      if (lane >= d) inc += y;
    }
    if (lane == 31) warp_sum[0][warp] = inc;
    __syncthreads();
    inc += __reduce_add_sync(VG_FULL_MASK, lane < warp ? warp_sum[0][lane] : 0);
    if (inc - sum < need && need <= inc) {
      uint32_t left = need - (inc - sum), d = bins - 1 - tid * own * 4;
      while (hist[d] < left) left -= hist[d--];
      sh_digit = d;
      sh_need = left;
      sh_count = hist[d];
    }
    __syncthreads();
    cut |= sh_digit << shift;
    need = sh_need;
    if (need == sh_count && cut) {  // the whole bin is kept: the keys from its first one on
      --cut;
      need = 0;
      break;
    }
  }

  uint32_t gt0 = 0, eq0 = 0;  // of the rounds before
  for (uint32_t r = 0; r < rounds; ++r) {
    if (!kOne) load(r);
    uint32_t gt = 0, eq = 0;
#pragma unroll
    for (uint32_t i = 0; i < kHeld; ++i) {
      gt += i < mine && key[i] > cut ? 1u : 0u;
      eq += i < mine && key[i] == cut ? 1u : 0u;
    }
    uint32_t both = gt | eq << 16;  // of a round: at most 2^14 each
    const uint32_t own = both;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t y = __shfl_up_sync(VG_FULL_MASK, both, d);
      if (lane >= d) both += y;
    }
    if (lane == 31) warp_sum[r & 1][warp] = both;
    __syncthreads();
    const uint32_t ws = lane < warps ? warp_sum[r & 1][lane] : 0;
    both += __reduce_add_sync(VG_FULL_MASK, lane < warp ? ws : 0) - own;
    const uint32_t all = __reduce_add_sync(VG_FULL_MASK, ws);
    gt = gt0 + (both & 0xffffu);
    eq = eq0 + (both >> 16);
#pragma unroll
    for (uint32_t i = 0; i < kHeld; ++i) {
      if (i >= mine) continue;
      const bool above = key[i] > cut, equal = key[i] == cut;
      if (above || (equal && eq < need)) {
        const uint32_t at = gt + min(eq, need);
        out[at] = static_cast<int32_t>(first + i);
        wd[at] = key[i] < kNewest - 1 ? key_to_float(key[i]) : w[first + i];
      }
      gt += above ? 1u : 0u;
      eq += equal ? 1u : 0u;
    }
    gt0 += all & 0xffffu;
    eq0 += all >> 16;
  }
}

// One CTA per (destination block, head): per keys and values the block's scale
// is the largest of its tokens' scales (NaN if one is), and each token's codes
// are moved, rounded to that scale where their own is smaller.  Bound by memory
// behind a chain of three loads (place, scale, codes); keys and values together
// have twice the bytes in flight behind it.  8 sequences x 8 heads x 2,048
// tokens (68 MB): 14 us from the selection's end, before which it has started.
template <int kItems, class P>
__global__ void __launch_bounds__(kStoreThreads) kv_gather_kernel(const __grid_constant__ KvView kv,
                                                                  const __grid_constant__ P plan,
                                                                  const uint32_t budget, const int32_t *kept) {
  __shared__ float from[2][128];
  __shared__ int32_t at[128];
  __shared__ uint32_t top[2];
  const uint32_t unit = blockIdx.x / kv.heads, head = blockIdx.x - unit * kv.heads;
  const uint32_t entry = plan_find(plan, unit);
  const PlanSeq &ps = plan.s[entry];
  const uint32_t per = kv.dim / 16;
  const uint32_t b = unit - ps.unit0, blk0 = b << kv.block_shift;
  const uint32_t n = min(kv.block, min(ps.len, budget) - blk0);
  const size_t nb = kv.stride >> kv.block_shift;
  const size_t rs = static_cast<size_t>(ps.seq) * kv.heads + head;
  const size_t rd = static_cast<size_t>(ps.row0) * kv.heads + head;
  if (threadIdx.x < 2) top[threadIdx.x] = 0;
  __syncthreads();
  chain_wait();  // the selection
  const uint32_t token = threadIdx.x & 127, which = threadIdx.x >> 7;
  if (token < n) {
    const int32_t t = kept[(static_cast<size_t>(entry) * kv.heads + head) * budget + blk0 + token];
    const float s = (which ? kv.scales[1] : kv.scales[0])[rs * nb + (static_cast<uint32_t>(t) >> kv.block_shift)];
    at[token] = t;  // both halves of the CTA write the same
    from[which][token] = s;
    atomicMax(&top[which], __float_as_uint(s) & 0x7fffffffu);  // positive: ordered by their bits, NaN last
  }
  __syncthreads();
  uint4 w[2][kItems];
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const uint32_t e = threadIdx.x + i * kStoreThreads, t = item_token(e, per);
    if (e >= n * per) continue;
    const size_t src = (rs * kv.stride + at[t]) * per + (e - t * per);
    w[0][i] = __ldg(reinterpret_cast<const uint4 *>(kv.codes[0]) + src);
    w[1][i] = __ldg(reinterpret_cast<const uint4 *>(kv.codes[1]) + src);
  }
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const float s_new = __uint_as_float(top[c]), inv = inverse(s_new);
    uint4 *dst = reinterpret_cast<uint4 *>(kv.codes[c]) + (rd * kv.stride + blk0) * per;
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const uint32_t e = threadIdx.x + i * kStoreThreads;
      if (e >= n * per) continue;
      const float ratio = from[c][item_token(e, per)] * inv;
      dst[e] = ratio < 1.0f ? rescaled(w[c][i], ratio) : w[c][i];
    }
    if (threadIdx.x == 0) kv.scales[c][rd * nb + b] = s_new;
  }
}

// f(the number of items of 16 elements that a thread takes of a block)
template <class F>
cudaError_t with_items(const KvView &kv, F &&f) {
  const uint32_t n = kv.block * (kv.dim / 16);
  if (n <= kStoreThreads) return f(std::integral_constant<int, 1>{});
  if (n <= 2 * kStoreThreads) return f(std::integral_constant<int, 2>{});
  return f(std::integral_constant<int, 4>{});
}

}  // namespace

cudaError_t launch_kv_append(const KvView &kv, const Plan &plan, int dtype, const Strided &k, const Strided &v,
                             cudaStream_t s) {
  if (plan.units == 0) return cudaSuccess;
  const bool kvec = rows_aligned(k, element_size(dtype)), vvec = rows_aligned(v, element_size(dtype));
  return with_plan(plan, [&](const auto &p) {
    return with_type(dtype, [&](auto t) {
      return with_items(kv, [&](auto items) {
        kv_append_kernel<decltype(t), items.value>
            <<<store_grid(kv, p), kStoreThreads, 0, s>>>(kv, p, k, v, kvec, vvec);
        return cudaGetLastError();
      });
    });
  });
}

cudaError_t launch_kv_read(const KvView &kv, const Plan &plan, int dtype, const Strided &k, const Strided &v,
                           cudaStream_t s) {
  if (plan.units == 0) return cudaSuccess;
  const bool kvec = rows_aligned(k, element_size(dtype)), vvec = rows_aligned(v, element_size(dtype));
  return with_plan(plan, [&](const auto &p) {
    return with_type(dtype, [&](auto t) {
      kv_read_kernel<decltype(t)><<<store_grid(kv, p), kStoreThreads, 0, s>>>(kv, p, k, v, kvec, vvec);
      return cudaGetLastError();
    });
  });
}

cudaError_t launch_kv_select(const KvView &kv, const Plan &plan, uint32_t budget, uint32_t recent, int32_t *kept,
                             cudaStream_t s) {
  uint32_t longest = 1;
  for (uint32_t i = 0; i < plan.n; ++i) longest = std::max(longest, plan.s[i].len);
  // the fewest tokens a thread that hold the row: short rows cost few rounds
  // of shared-memory additions
  const uint32_t threads = longest <= 256 * 4 ? 256 : kSelectThreads;
  return with_plan(plan, [&](const auto &p) {
    using P = std::decay_t<decltype(p)>;
    auto *kern = longest <= threads * 4    ? kv_select_kernel<true, 4, P>
                 : longest <= threads * 8  ? kv_select_kernel<true, 8, P>
                 : longest <= threads * 16 ? kv_select_kernel<true, 16, P>
                                           : kv_select_kernel<false, 16, P>;
    kern<<<dim3(kv.heads, p.n), threads, 0, s>>>(kv, p, budget, recent, kept);
    return cudaGetLastError();
  });
}

cudaError_t launch_kv_gather(const KvView &kv, const Plan &plan, uint32_t budget, const int32_t *kept,
                             cudaStream_t s) {
  if (plan.units == 0) return cudaSuccess;
  return with_plan(plan, [&](const auto &p) {
    return with_items(kv, [&](auto items) {
      return launch_chained(kv_gather_kernel<items.value, std::decay_t<decltype(p)>>, p.units * kv.heads,
                            kStoreThreads, 0, s, kv, p, budget, kept);
    });
  });
}

}  // namespace vg
