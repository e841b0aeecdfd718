// Attention over a key/value cache held in 8 bits.
#include "common.cuh"
#include "elements.cuh"
#include "kv_cache.h"

namespace vg {

namespace {

constexpr int kRowWarps = 4;

// First version: one warp per (query row, head), the tokens one after another
// with a running maximum and sum; a lane holds dim / 32 dimensions.
template <class T>
__global__ void __launch_bounds__(kRowWarps * 32) attend_rows_kernel(const __grid_constant__ AttendArgs a,
                                                                     const __grid_constant__ Plan plan) {
  const PlanSeq &ps = plan.s[plan_find(plan, blockIdx.x)];
  const uint32_t j = blockIdx.x - ps.unit0, h = blockIdx.y * kRowWarps + (threadIdx.x >> 5);
  if (h >= a.q_heads) return;
  const int lane = lane_id();
  const KvView &kv = a.kv;
  const size_t r = static_cast<size_t>(ps.seq) * kv.heads + h / a.group;
  const uint32_t per = kv.dim / 32;
  const T *q = static_cast<const T *>(a.q.p) + static_cast<int64_t>(ps.row0 + j) * a.q.token +
               static_cast<int64_t>(h) * a.q.head;
  float qv[4], o[4] = {};
  for (uint32_t i = 0; i < 4; ++i) qv[i] = i < per ? to_f32(q[lane + 32 * i]) * a.scale : 0.0f;
  const uint32_t behind = ps.count - 1 - j;
  const uint32_t sees = a.causal ? (ps.len > behind ? ps.len - behind : 0) : ps.len;
  const size_t nb = kv.stride >> kv.block_shift;
  const int8_t *kc = kv.codes[0] + r * kv.stride * kv.dim, *vc = kv.codes[1] + r * kv.stride * kv.dim;
  const float *ks = kv.scales[0] + r * nb, *vs = kv.scales[1] + r * nb;
  float m = -__int_as_float(0x7f800000), l = 0.0f;
  for (uint32_t t = 0; t < sees; ++t) {
    float d = 0.0f;
    for (uint32_t i = 0; i < per; ++i) d += qv[i] * static_cast<float>(kc[static_cast<size_t>(t) * kv.dim + lane + 32 * i]);
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) d += __shfl_xor_sync(VG_FULL_MASK, d, w);
    const float s = d * ks[t >> kv.block_shift];
    const float mn = s > m || s != s ? s : m;
    const float c = expf(m - mn), p = expf(s - mn);
    l = l * c + p;
    const float pv = p * vs[t >> kv.block_shift];
    for (uint32_t i = 0; i < per; ++i)
      o[i] = o[i] * c + pv * static_cast<float>(vc[static_cast<size_t>(t) * kv.dim + lane + 32 * i]);
    m = mn;
  }
  T *out = static_cast<T *>(a.out.p) + static_cast<int64_t>(ps.row0 + j) * a.out.token +
           static_cast<int64_t>(h) * a.out.head;
  for (uint32_t i = 0; i < per; ++i) out[lane + 32 * i] = from_f32<T>(sees ? o[i] / l : 0.0f);
  if (lane == 0) a.lse[static_cast<size_t>(ps.row0 + j) * a.q_heads + h] = m + logf(l);
}

// One warp per (cached token, key/value head): its probabilities, recomputed
// from the rows' lse, summed over the queries and heads that share it.
template <class T>
__global__ void __launch_bounds__(kRowWarps * 32) weigh_rows_kernel(const __grid_constant__ AttendArgs a,
                                                                    const __grid_constant__ Plan plan) {
  const PlanSeq &ps = plan.s[plan_find(plan, blockIdx.x)];
  const uint32_t t = (blockIdx.x - ps.unit0) * kRowWarps + (threadIdx.x >> 5), g = blockIdx.y;
  if (t >= ps.len) return;
  const int lane = lane_id();
  const KvView &kv = a.kv;
  const size_t r = static_cast<size_t>(ps.seq) * kv.heads + g;
  const uint32_t per = kv.dim / 32;
  const float ks = kv.scales[0][r * (kv.stride >> kv.block_shift) + (t >> kv.block_shift)] * a.scale;
  float kvv[4];
  for (uint32_t i = 0; i < 4; ++i)
    kvv[i] = i < per ? ks * static_cast<float>(kv.codes[0][(r * kv.stride + t) * kv.dim + lane + 32 * i]) : 0.0f;
  float sum = 0.0f;
  for (uint32_t j = 0; j < ps.count; ++j) {
    if (a.causal && t + (ps.count - 1 - j) >= ps.len) continue;
    for (uint32_t h = g * a.group; h < (g + 1) * a.group; ++h) {
      const T *q = static_cast<const T *>(a.q.p) + static_cast<int64_t>(ps.row0 + j) * a.q.token +
                   static_cast<int64_t>(h) * a.q.head;
      float d = 0.0f;
      for (uint32_t i = 0; i < per; ++i) d += to_f32(q[lane + 32 * i]) * kvv[i];
#pragma unroll
      for (int w = 16; w > 0; w >>= 1) d += __shfl_xor_sync(VG_FULL_MASK, d, w);
      sum += expf(d - a.lse[static_cast<size_t>(ps.row0 + j) * a.q_heads + h]);
    }
  }
  if (lane == 0) kv.weights[r * kv.stride + t] += sum;
}

}  // namespace

cudaError_t launch_kv_attend_rows(const AttendArgs &a, const Plan &plan, cudaStream_t s) {
  if (plan.units == 0) return cudaSuccess;
  const dim3 grid(plan.units, (a.q_heads + kRowWarps - 1) / kRowWarps);
  if (a.dtype == VG_F16) attend_rows_kernel<__half><<<grid, kRowWarps * 32, 0, s>>>(a, plan);
  else attend_rows_kernel<__nv_bfloat16><<<grid, kRowWarps * 32, 0, s>>>(a, plan);
  return cudaGetLastError();
}

cudaError_t launch_kv_weigh_rows(const AttendArgs &a, const Plan &plan, cudaStream_t s) {
  if (plan.units == 0) return cudaSuccess;
  const dim3 grid(plan.units, a.kv.heads);
  if (a.dtype == VG_F16) weigh_rows_kernel<__half><<<grid, kRowWarps * 32, 0, s>>>(a, plan);
  else weigh_rows_kernel<__nv_bfloat16><<<grid, kRowWarps * 32, 0, s>>>(a, plan);
  return cudaGetLastError();
}

}  // namespace vg
