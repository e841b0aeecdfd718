// Rotary positions: every pair (a, b) of a head becomes
//   m (a cos t - b sin t, a sin t + b cos t),  t = position * frequency,
// or, transposed, the same with -sin (the map that takes gradients back).
//
// Bound by memory: each value is read and written once.  The angle is reduced
// to a fraction of a turn in 64 bits -- in 32 an angle at position 10^5 would
// be off by a hundredth -- and its sine and cosine are computed once per
// (token, frequency) of a CTA, in shared memory, for all heads the CTA takes.
// 16,384 tokens x 40 heads x 128 in bf16: 55 us, 6.1 TB/s.
#include "common.cuh"
#include "elements.cuh"
#include "kv_cache.h"
#include "kv_host.h"

#include <algorithm>
#include <cmath>

namespace vg {

namespace {

constexpr int kRotaryThreads = 256;
constexpr size_t kFillCtas = 2 * 148;  // two CTAs for each SM

struct RotaryArgs {
  const int64_t *pos;
  uint32_t tokens, dim;       // dim: of the head
  uint32_t q_heads, heads;    // heads: of q and k
  uint32_t heads_per_cta, tokens_per_cta;
  uint32_t items;             // work items per (token, head): of pairs, then of copied dimensions
  uint32_t pair_items;
  Strided q, qo, k, ko;
  bool transpose;
};

template <int N>
__device__ __forceinline__ void sines(const float *p, float (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N / 4; ++i) {
    const float4 v = reinterpret_cast<const float4 *>(p)[i];
    x[4 * i] = v.x, x[4 * i + 1] = v.y, x[4 * i + 2] = v.z, x[4 * i + 3] = v.w;
  }
}

// An item is 8 pairs (halves), 4 pairs (adjacent) or 8 copied elements with
// vec, one pair or one element without.
template <class T, bool kVec, bool kInterleaved>
__global__ void __launch_bounds__(kRotaryThreads) rotary_kernel(const __grid_constant__ RotaryTable tab,
                                                                const __grid_constant__ RotaryArgs a) {
  extern __shared__ __align__(16) float cs[];  // [tokens_per_cta][2][pairs]: m cos, m sin
  const uint32_t t0 = blockIdx.x * a.tokens_per_cta, nt = min(a.tokens_per_cta, a.tokens - t0);
  const uint32_t h0 = blockIdx.y * a.heads_per_cta, nh = min(a.heads_per_cta, a.heads - h0);
  for (uint32_t e = threadIdx.x; e < nt * tab.pairs; e += kRotaryThreads) {
    const uint32_t t = e / tab.pairs, i = e - t * tab.pairs;
    double turn = static_cast<double>(a.pos[t0 + t]) * tab.turns[i];
    turn -= rint(turn);
    float s, c;
    sincospif(static_cast<float>(2.0 * turn), &s, &c);
    s *= tab.magnitude;
    cs[e + t * tab.pairs] = c * tab.magnitude;
    cs[e + (t + 1) * tab.pairs] = a.transpose ? -s : s;
  }
  __syncthreads();
  const uint32_t n = nt * nh * a.items;
  for (uint32_t e = threadIdx.x; e < n; e += kRotaryThreads) {
    const uint32_t th = e / a.items, item = e - th * a.items;
    const uint32_t t = th / nh, h = h0 + th - t * nh;
    const bool is_q = h < a.q_heads;
    const Strided &in = is_q ? a.q : a.k, &out = is_q ? a.qo : a.ko;
    const int64_t hh = is_q ? h : h - a.q_heads;
    const T *src = static_cast<const T *>(in.p) + static_cast<int64_t>(t0 + t) * in.token + hh * in.head;
    T *dst = static_cast<T *>(out.p) + static_cast<int64_t>(t0 + t) * out.token + hh * out.head;
    const float *fc = cs + 2 * t * tab.pairs, *fs = fc + tab.pairs;
    if (item >= a.pair_items) {
      const uint32_t d = 2 * tab.pairs + (item - a.pair_items) * (kVec ? 8 : 1);
      if (kVec) {
        float x[8];
        load8(src + d, true, x);
        store8(dst + d, true, x);
      } else {
        dst[d] = src[d];
      }
    } else if (kVec && kInterleaved) {
      float x[8], y[8], c[4], s[4];
      load8(src + item * 8, true, x);
      sines<4>(fc + item * 4, c);
      sines<4>(fs + item * 4, s);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        y[2 * j] = x[2 * j] * c[j] - x[2 * j + 1] * s[j];
        y[2 * j + 1] = x[2 * j] * s[j] + x[2 * j + 1] * c[j];
      }
      store8(dst + item * 8, true, y);
    } else if (kVec) {
      float x[8], y[8], u[8], v[8], c[8], s[8];
      load8(src + item * 8, true, x);
      load8(src + tab.pairs + item * 8, true, y);
      sines<8>(fc + item * 8, c);
      sines<8>(fs + item * 8, s);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        u[j] = x[j] * c[j] - y[j] * s[j];
        v[j] = x[j] * s[j] + y[j] * c[j];
      }
      store8(dst + item * 8, true, u);
      store8(dst + tab.pairs + item * 8, true, v);
    } else {
      const uint32_t ia = kInterleaved ? 2 * item : item, ib = kInterleaved ? 2 * item + 1 : item + tab.pairs;
      const float c = fc[item], s = fs[item];
      const float x = to_f32(src[ia]), y = to_f32(src[ib]);
      dst[ia] = from_f32<T>(x * c - y * s);
      dst[ib] = from_f32<T>(x * s + y * c);
    }
  }
}

}  // namespace

cudaError_t launch_rotary(const RotaryTable &tab, int dtype, uint32_t dim, const int64_t *pos, size_t tokens,
                          const Strided &q, const Strided &qo, uint32_t q_heads, const Strided &k, const Strided &ko,
                          uint32_t k_heads, bool transpose, cudaStream_t s) {
  const size_t es = element_size(dtype);
  const uint32_t rot = 2 * tab.pairs;
  const bool vec = tab.pairs % (tab.interleaved ? 4 : 8) == 0 && dim % 8 == 0 && rows_aligned(q, es) &&
                   rows_aligned(qo, es) && (k_heads == 0 || (rows_aligned(k, es) && rows_aligned(ko, es)));
  const bool in_place = q.p == qo.p && (k_heads == 0 || k.p == ko.p);
  RotaryArgs a{};
  a.pos = pos;
  a.tokens = static_cast<uint32_t>(tokens);
  a.dim = dim;
  a.q_heads = q_heads;
  a.heads = q_heads + k_heads;
  a.pair_items = vec ? tab.pairs / (tab.interleaved ? 4 : 8) : tab.pairs;
  a.items = a.pair_items + (in_place ? 0 : vec ? (dim - rot) / 8 : dim - rot);
  a.q = q;
  a.qo = qo;
  a.k = k;
  a.ko = ko;
  a.transpose = transpose;
  // a CTA takes about 256 sines for its tokens and all heads; with few tokens,
  // one token and a share of the heads, so that the GPU is filled
  a.tokens_per_cta = std::max(1u, 256u / tab.pairs);
  // (at most 2^24 items a CTA: they are counted in 32 bits)
  a.heads_per_cta = std::min(a.heads, std::max(1u, (1u << 24) / (a.tokens_per_cta * std::max(1u, a.items))));
  if (tokens < a.tokens_per_cta * kFillCtas) {
    a.tokens_per_cta = 1;
    const uint32_t parts = static_cast<uint32_t>(std::max<size_t>(1, kFillCtas / tokens));
    a.heads_per_cta = std::min(
        a.heads_per_cta,
        std::max(std::max(1u, kRotaryThreads / 2 / std::max(1u, a.items)), (a.heads + parts - 1) / parts));
  }
  const dim3 grid(static_cast<uint32_t>((tokens + a.tokens_per_cta - 1) / a.tokens_per_cta),
                  (a.heads + a.heads_per_cta - 1) / a.heads_per_cta);
  const size_t smem = static_cast<size_t>(a.tokens_per_cta) * tab.pairs * sizeof(float2);
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    auto *kern = vec ? (tab.interleaved ? rotary_kernel<T, true, true> : rotary_kernel<T, true, false>)
                     : (tab.interleaved ? rotary_kernel<T, false, true> : rotary_kernel<T, false, false>);
    kern<<<grid, kRotaryThreads, smem, s>>>(tab, a);
    return cudaGetLastError();
  });
}

}  // namespace vg

using namespace vg;

struct vg_rotary {
  RotaryTable table{};
  double freq[128];
};

extern "C" {

int vg_rotary_create(const vg_rotary_params *params, vg_rotary **out) {
  return guarded([&]() -> int {
    if (!params || !out) return fail(VG_ERR_INVALID_PARAMETER, "null argument");
    *out = nullptr;
    const vg_rotary_params &p = *params;
    if (p.dim < 2 || p.dim > 256 || p.dim % 2)
      return fail(VG_ERR_INVALID_CONFIG, "invalid config `dim`: rotary dimensions must be even, 2 to 256");
    if (!std::isfinite(p.base) || p.base <= 1.0)
      return fail(VG_ERR_INVALID_CONFIG, "invalid config `base`: must be finite and greater than 1");
    if (p.scaling < VG_ROTARY_PLAIN || p.scaling > VG_ROTARY_BY_PARTS)
      return fail(VG_ERR_INVALID_CONFIG, "invalid config `scaling`: must be a VG_ROTARY_ kind");
    if (p.scaling != VG_ROTARY_PLAIN && (!std::isfinite(p.factor) || p.factor < 1.0))
      return fail(VG_ERR_INVALID_CONFIG, "invalid config `factor`: must be finite and at least 1");
    if (p.scaling == VG_ROTARY_BY_PARTS &&
        (!std::isfinite(p.original_length) || p.original_length <= 0.0 || !std::isfinite(p.high_turns) ||
         !(p.low_turns >= 0.0) || !(p.high_turns > p.low_turns)))
      return fail(VG_ERR_INVALID_CONFIG,
                  "invalid config: by-parts scaling takes original_length > 0 and 0 <= low_turns < high_turns");
    if (!std::isfinite(p.magnitude) || p.magnitude <= 0.0)
      return fail(VG_ERR_INVALID_CONFIG, "invalid config `magnitude`: must be finite and greater than 0");
    const double two_pi = 6.283185307179586476925;
    vg_rotary *r = new vg_rotary;
    r->table.pairs = static_cast<uint32_t>(p.dim / 2);
    r->table.interleaved = p.interleaved != 0;
    r->table.magnitude = static_cast<float>(p.magnitude);
    for (uint32_t i = 0; i < r->table.pairs; ++i) {
      double f = std::pow(p.base, -2.0 * i / static_cast<double>(p.dim));
      if (p.scaling == VG_ROTARY_LINEAR) f /= p.factor;
      if (p.scaling == VG_ROTARY_BY_PARTS) {
        const double turns = p.original_length * f / two_pi;
        const double g = std::min(1.0, std::max(0.0, (turns - p.low_turns) / (p.high_turns - p.low_turns)));
        f = (1.0 - g) * f / p.factor + g * f;
      }
      r->freq[i] = f;
      r->table.turns[i] = f / two_pi;
    }
    *out = r;
    return VG_OK;
  });
}

int vg_rotary_destroy(vg_rotary *r) {
  delete r;
  return VG_OK;
}

int vg_rotary_frequencies(const vg_rotary *r, double *out) {
  return guarded([&]() -> int {
    if (!r || !out) return fail(VG_ERR_INVALID_PARAMETER, "null argument");
    std::copy(r->freq, r->freq + r->table.pairs, out);
    return VG_OK;
  });
}

int vg_rotary_apply(const vg_rotary *r, int dtype, size_t head_dim, const int64_t *positions, size_t tokens,
                    const vg_heads *q, const vg_heads *q_out, const vg_heads *k, const vg_heads *k_out,
                    int transpose, int device, void *stream) {
  return guarded([&]() -> int {
    if (!r) return fail(VG_ERR_INVALID_PARAMETER, "null rotary table");
    VG_TRY(check_dtype(dtype));
    if (head_dim < 2 * r->table.pairs || head_dim > 4096)
      return fail(VG_ERR_DIMENSION_MISMATCH, "head_dim must be at least the rotated dimensions, at most 4096");
    if (tokens > 0x7fffffffull) return fail(VG_ERR_INVALID_PARAMETER, "at most 2^31 - 1 tokens");
    if (!k != !k_out) return fail(VG_ERR_INVALID_PARAMETER, "k and k_out go together");
    VG_TRY(check_device(device));
    if (tokens == 0) return VG_OK;
    DeviceGuard g(device);
    VG_TRY(check_device_memory(positions, sizeof(int64_t), device, "positions"));
    const vg_heads *in[2] = {q, k}, *out[2] = {q_out, k_out};
    const char *names[2][2] = {{"q", "q_out"}, {"k", "k_out"}};
    for (int i = 0; i < (k ? 2 : 1); ++i) {
      VG_TRY(check_heads(in[i], names[i][0], tokens, head_dim, dtype, device, false));
      VG_TRY(check_heads(out[i], names[i][1], tokens, head_dim, dtype, device, true));
      if (in[i]->num_heads != out[i]->num_heads)
        return fail(VG_ERR_DIMENSION_MISMATCH, std::string(names[i][1]) + " must have the heads of its input");
      if (in[i]->data == out[i]->data &&
          (in[i]->token_stride != out[i]->token_stride || in[i]->head_stride != out[i]->head_stride))
        return fail(VG_ERR_INVALID_PARAMETER, std::string(names[i][1]) + " in place must have its input's strides");
    }
    const Strided none{};
    VG_CU(launch_rotary(r->table, dtype, static_cast<uint32_t>(head_dim), positions, tokens, strided(*q),
                        strided(*q_out), static_cast<uint32_t>(q->num_heads), k ? strided(*k) : none,
                        k ? strided(*k_out) : none, k ? static_cast<uint32_t>(k->num_heads) : 0u, transpose != 0,
                        static_cast<cudaStream_t>(stream)));
    return VG_OK;
  });
}

}  // extern "C"
