// C ABI of the key/value cache (include/vicinity_gpu.h): the handle, its
// device memory, the launch plans made from host-side lengths, and checks.
#include <algorithm>
#include <cmath>
#include <memory>
#include <string>
#include <vector>

#include "kv_cache.h"
#include "kv_host.h"

using namespace vg;

struct vg_kv_cache {
  int device = 0;
  vg_kv_params params{};
  KvView view{};
  DevBuf codes[2], scales[2], weights;
  std::vector<uint32_t> len;  // tokens of each sequence once all enqueued work is done
  DevBuf ws_lse, ws_kept, ws_part, ws_scores, ws_tiles;
  int *h_err = nullptr, *d_err = nullptr;  // error flag of bounded device waits, in mapped pinned host memory
  // Work is ordered across streams: each call's stream first waits for the
  // event recorded after the last call's work.
  cudaEvent_t done = nullptr;

  ~vg_kv_cache() {
    if (done) {
      cudaEventSynchronize(done);
      cudaEventDestroy(done);
    }
    if (h_err) cudaFreeHost(h_err);
  }
};

namespace {

// The device work of one call, between begin() and the end of the scope.
class Work {
 public:
  Work(vg_kv_cache *kv, void *stream) : kv_(kv), s_(static_cast<cudaStream_t>(stream)) {}
  ~Work() {  // also after a failed launch: what was enqueued before it is ordered
    if (begun_) cudaEventRecord(kv_->done, s_);
  }
  int begin() {
    cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
    VG_CU(cudaStreamIsCapturing(s_, &cap));
    if (cap != cudaStreamCaptureStatusNone)
      return fail(VG_ERR_UNSUPPORTED, "unsupported: key/value cache calls cannot be captured into a CUDA graph");
    if (const int code = *reinterpret_cast<volatile int *>(kv_->h_err))
      return fail(VG_ERR_CUDA, "an earlier attention call gave up a wait on the device (code " + std::to_string(code) +
                                   "): its results are not valid");
    VG_CU(cudaStreamWaitEvent(s_, kv_->done, 0));
    begun_ = true;
    return VG_OK;
  }

 private:
  vg_kv_cache *kv_;
  cudaStream_t s_;
  bool begun_ = false;
};

uint32_t ceil_div(uint32_t a, uint32_t b) { return a / b + (a % b != 0); }

// Rows of all sequences; refuses totals that do not fit the packed row index.
int total_rows(const vg_kv_cache *kv, const uint32_t *counts, size_t *out) {
  size_t n = 0;
  for (size_t s = 0; s < kv->params.num_seqs; ++s) n += counts[s];
  if (n > 0x7fffffffull) return fail(VG_ERR_INVALID_PARAMETER, "at most 2^31 - 1 tokens per call");
  *out = n;
  return VG_OK;
}

// A launch over (unit, head, K or V) has a one-dimensional grid.
int check_grid(const vg_kv_cache *kv, uint64_t units) {
  if (units * 2 * kv->view.heads > 0x7fffffffull) return fail(VG_ERR_INVALID_PARAMETER, "too many tokens in one call");
  return VG_OK;
}

// Calls launch(plan) for the sequences with a count, kPlanSeqs at a time.
// entry(seq, PlanSeq&) fills in len and count and returns the entry's units.
// Sequences that `take` refuses are passed over.
template <class Take, class Entry, class Launch>
int for_plans_of(const vg_kv_cache *kv, const uint32_t *counts, Take &&take, Entry &&entry, Launch &&launch) {
  Plan plan;
  plan.n = plan.units = 0;
  uint32_t row = 0;
  uint64_t units = 0;
  const size_t ns = kv->params.num_seqs;
  for (size_t s = 0; s < ns; ++s) {
    if (counts[s] && take(counts[s])) {
      PlanSeq &e = plan.s[plan.n++];
      e.seq = static_cast<uint32_t>(s);
      e.len = kv->len[s];
      e.count = counts[s];
      e.row0 = row;
      e.unit0 = static_cast<uint32_t>(units);
      units += entry(s, e);
      if (units > 0x7fffffffull) return fail(VG_ERR_INVALID_PARAMETER, "too many tokens in one call");
    }
    row += counts[s];
    if (plan.n == kPlanSeqs || (s + 1 == ns && plan.n)) {
      plan.units = static_cast<uint32_t>(units);
      VG_TRY(launch(plan));
      plan.n = 0;
      units = 0;
    }
  }
  return VG_OK;
}

template <class Entry, class Launch>
int for_plans(const vg_kv_cache *kv, const uint32_t *counts, Entry &&entry, Launch &&launch) {
  return for_plans_of(kv, counts, [](uint32_t) { return true; }, entry, [&](Plan &plan) -> int {
    VG_TRY(check_grid(kv, plan.units));
    VG_CU(launch(plan));
    return VG_OK;
  });
}

// Re-counts a plan's units: units_of(entry) each.
template <class Units>
int set_units(Plan &plan, Units &&units_of) {
  uint64_t units = 0;
  for (uint32_t i = 0; i < plan.n; ++i) {
    plan.s[i].unit0 = static_cast<uint32_t>(units);
    units += units_of(plan.s[i]);
    if (units > 0x7fffffffull) return fail(VG_ERR_INVALID_PARAMETER, "too many tokens in one call");
  }
  plan.units = static_cast<uint32_t>(units);
  return VG_OK;
}

// Tokens per work unit when the tokens of every sequence are cut into chunks.
// Units run `slots` at a time, so w waves of chunks of c tokens take about
// w (c + kUnitCost), and joining the chunks kJoinCost more: of one to four full
// waves, and of leaving the sequences whole, the cheapest.  per_chunk(entry):
// units of one chunk of it.  Costs are in tokens of a unit: a unit's start and
// end take about 1 us, a join 4 us, where the decoding kernel's take 3 to 4 us per
// 512 tokens.
constexpr uint32_t kUnitCost = 128, kJoinCost = 512, kMaxWaves = 4;

template <class PerChunk>
uint32_t pick_chunk(const Plan &plan, uint64_t slots, uint32_t quantum, PerChunk &&per_chunk) {
  uint32_t longest = 1;
  for (uint32_t i = 0; i < plan.n; ++i) longest = std::max(longest, plan.s[i].len);
  const auto units = [&](uint32_t chunk) {
    uint64_t n = 0;
    for (uint32_t i = 0; i < plan.n; ++i) n += std::max(1u, ceil_div(plan.s[i].len, chunk)) * per_chunk(plan.s[i]);
    return n;
  };
  const uint32_t least = std::max(1u, ceil_div(ceil_div(longest, kMaxSplits), quantum));
  const uint32_t whole = std::max(least, ceil_div(longest, quantum));
  const auto cost_of = [&](uint32_t c) {
    return (units(c * quantum) + slots - 1) / slots * (uint64_t(c) * quantum + kUnitCost) + (c < whole ? kJoinCost : 0);
  };
  uint32_t best = whole;
  uint64_t cost = cost_of(whole);
  for (uint32_t w = 1; w <= kMaxWaves; ++w) {
    uint32_t lo = least, hi = whole;  // the smallest chunk that makes at most w waves
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo) / 2;
      if (units(mid * quantum) <= w * slots) hi = mid;
      else lo = mid + 1;
    }
    const uint64_t c = cost_of(lo);
    if (c < cost) {
      cost = c;
      best = lo;
    }
  }
  return best * quantum;
}

constexpr size_t kScoreBytes = size_t(1) << 30;  // stored scores of one launch, at most
constexpr uint64_t kSlots = 148 * 2;             // CTAs that run at once, of the decoding and the tile kernel
constexpr uint32_t kDecodeQuantum = 32;

// Working memory of `bytes`.  To replace a buffer waits for the device, so what
// grows with the sequences is made for the longest they can get (`most`, where
// that is known), and anything else at least doubles.
int reserve(DevBuf &b, size_t bytes, size_t most = 0) {
  if (bytes <= b.cap) return VG_OK;
  if (b.reserve(std::max({bytes, most, 2 * b.cap})) != cudaSuccess) {
    cudaGetLastError();  // no room for more than is needed
    VG_CU(b.reserve(bytes));
  }
  return VG_OK;
}

// Query tiles of a plan's rows, for the tile kernels.
int query_tiles(vg_kv_cache *kv, AttendArgs &a, Plan &plan, cudaStream_t s) {
  uint64_t blocks = 0;
  for (uint32_t i = 0; i < plan.n; ++i) {
    plan.s[i].block0 = static_cast<uint32_t>(blocks);
    blocks += ceil_div(plan.s[i].count * a.group, kTileRows);
  }
  const size_t n = blocks * kv->view.heads, bytes = query_tile_bytes(kv->view.dim);
  VG_TRY(reserve(kv->ws_tiles, n * (bytes + kTileRows * sizeof(float))));
  a.q_tiles = kv->ws_tiles.as<uint8_t>();
  a.q_factor = reinterpret_cast<float *>(a.q_tiles + n * bytes);
  VG_CU(launch_kv_query_tiles(a, plan, static_cast<uint32_t>(blocks), s));
  return VG_OK;
}

int weigh_tiles(AttendArgs &a, Plan &plan, cudaStream_t s) {
  VG_TRY(set_units(plan, [](const PlanSeq &e) { return ceil_div(e.len, kWeighRows); }));
  VG_CU(launch_kv_weigh_tiles(a, plan, s));
  return VG_OK;
}

// max_ctas: what a plan that is cut can have at any lengths, where it is known.
int reserve_parts(vg_kv_cache *kv, AttendArgs &a, const Plan &plan, uint32_t part_rows, size_t max_ctas = 0) {
  const size_t rows = static_cast<size_t>(plan.units) * kv->view.heads * part_rows;
  const size_t row_bytes = kv->view.dim * sizeof(float) + sizeof(float4);
  VG_TRY(reserve(kv->ws_part, rows * row_bytes, max_ctas * part_rows * row_bytes));
  a.part_o = kv->ws_part.as<float>();
  a.part_ml = reinterpret_cast<float4 *>(a.part_o + rows * kv->view.dim);
  return VG_OK;
}

// Sequences of at most kDecodeRows rows per key/value head.
int attend_decode(vg_kv_cache *kv, AttendArgs a, Plan &plan, cudaStream_t s) {
  uint32_t max_rows = 0;
  for (uint32_t i = 0; i < plan.n; ++i) max_rows = std::max(max_rows, plan.s[i].count * a.group);
  a.chunk = pick_chunk(plan, kSlots, kDecodeQuantum, [&](const PlanSeq &) { return uint64_t(kv->view.heads); });
  bool split = false;
  size_t scores = 0, most = 0, chunks = 0;  // the latter two: of sequences at their capacity
  const uint32_t cap = static_cast<uint32_t>(kv->params.capacity);
  for (uint32_t i = 0; i < plan.n; ++i) {
    PlanSeq &e = plan.s[i];
    split |= e.len > a.chunk;
    e.aux = scores;
    const size_t rows = static_cast<size_t>(kv->view.heads) * ((e.count * a.group + 1) & ~1u);
    scores += rows * (static_cast<size_t>(ceil_div(e.len, 16)) * 16);
    most += rows * (static_cast<size_t>(ceil_div(cap, 16)) * 16);
    chunks += static_cast<size_t>(kv->view.heads) * ceil_div(cap, kDecodeQuantum);
  }
  VG_TRY(set_units(plan, [&](const PlanSeq &e) { return std::max(1u, ceil_div(e.len, a.chunk)); }));
  if (split) VG_TRY(reserve_parts(kv, a, plan, kDecodeRows, std::min<size_t>(kMaxWaves * kSlots, chunks)));
  const bool keep = a.lse2 && scores * sizeof(float) <= kScoreBytes;
  if (keep) {
    VG_TRY(reserve(kv->ws_scores, std::max<size_t>(scores, 1) * sizeof(float),
                   std::min(most * sizeof(float), kScoreBytes)));
    a.scores = kv->ws_scores.as<float>();
  } else if (a.lse2) {  // before the attention: its outputs may take the queries' place
    VG_TRY(query_tiles(kv, a, plan, s));
  }
  VG_CU(launch_kv_attend_decode(a, plan, max_rows, s));
  if (split) VG_CU(launch_kv_attend_join(a, plan, kDecodeRows, max_rows, s));
  if (keep) {
    VG_TRY(set_units(plan, [](const PlanSeq &e) { return ceil_div(e.len, kWeighTile); }));
    VG_CU(launch_kv_weigh_scores(a, plan, s));
  } else if (a.lse2) {
    VG_TRY(weigh_tiles(a, plan, s));
  }
  return VG_OK;
}

// Sequences of more rows, in units of `tiles` row tiles.
int attend_tiles(vg_kv_cache *kv, AttendArgs a, Plan &plan, uint32_t tiles, cudaStream_t s) {
  const uint32_t unit_rows = tiles * kTileRows;
  const auto blocks = [&](const PlanSeq &e) { return ceil_div(e.count * a.group, unit_rows); };
  VG_TRY(query_tiles(kv, a, plan, s));
  a.chunk = pick_chunk(plan, kSlots / tiles, kTileRows,
                       [&](const PlanSeq &e) { return uint64_t(kv->view.heads) * blocks(e); });
  VG_TRY(set_units(plan, [&](const PlanSeq &e) { return uint64_t(blocks(e)) * std::max(1u, ceil_div(e.len, a.chunk)); }));
  uint32_t max_rows = 0;  // of the sequences that are cut
  for (uint32_t i = 0; i < plan.n; ++i)
    if (plan.s[i].len > a.chunk) max_rows = std::max(max_rows, plan.s[i].count * a.group);
  if (max_rows) VG_TRY(reserve_parts(kv, a, plan, unit_rows));
  VG_CU(launch_kv_attend_tiles(a, plan, tiles, s));
  if (max_rows) VG_CU(launch_kv_attend_join(a, plan, unit_rows, max_rows, s));
  if (a.lse2) VG_TRY(weigh_tiles(a, plan, s));
  return VG_OK;
}

}  // namespace

extern "C" {

int vg_kv_create(const vg_kv_params *params, int device, vg_kv_cache **out) {
  return guarded([&]() -> int {
    if (!params || !out) return fail(VG_ERR_INVALID_PARAMETER, "null argument");
    *out = nullptr;
    const vg_kv_params &p = *params;
    if (p.num_seqs == 0 || p.num_kv_heads == 0 || p.num_kv_heads > 65535 || p.capacity == 0 ||
        p.capacity > (1ull << 30))
      return fail(VG_ERR_INVALID_CONFIG,
                  "invalid config: num_seqs >= 1, num_kv_heads 1 to 65535 and capacity 1 to 2^30 are needed");
    if (p.head_dim != 32 && p.head_dim != 64 && p.head_dim != 96 && p.head_dim != 128)
      return fail(VG_ERR_INVALID_CONFIG, "invalid config `head_dim`: must be 32, 64, 96 or 128");
    if (p.block_tokens != 16 && p.block_tokens != 32 && p.block_tokens != 64 && p.block_tokens != 128)
      return fail(VG_ERR_INVALID_CONFIG, "invalid config `block_tokens`: must be 16, 32, 64 or 128");
    if (p.num_seqs > (1ull << 31) / p.num_kv_heads)
      return fail(VG_ERR_INVALID_CONFIG, "invalid config: num_seqs * num_kv_heads must be at most 2^31");
    VG_TRY(check_device(device));
    DeviceGuard g(device);
    auto kv = std::make_unique<vg_kv_cache>();
    kv->device = device;
    kv->params = p;
    kv->len.assign(p.num_seqs, 0);
    const size_t stride = (p.capacity + kKvPad - 1) / kKvPad * kKvPad;
    const size_t rows = p.num_seqs * p.num_kv_heads;
    if (rows > (size_t(1) << 50) / (stride * p.head_dim))
      return fail(VG_ERR_OUT_OF_MEMORY, "the cache does not fit any device");
    for (int i = 0; i < 2; ++i) {
      VG_CU(kv->codes[i].reserve(rows * stride * p.head_dim));
      VG_CU(kv->scales[i].reserve(rows * (stride / p.block_tokens) * sizeof(float)));
      kv->view.codes[i] = kv->codes[i].as<int8_t>();
      kv->view.scales[i] = kv->scales[i].as<float>();
    }
    VG_CU(kv->weights.reserve(rows * stride * sizeof(float)));
    VG_CU(cudaMemsetAsync(kv->weights.p, 0, rows * stride * sizeof(float), nullptr));
    VG_CU(cudaStreamSynchronize(nullptr));
    VG_CU(cudaEventCreateWithFlags(&kv->done, cudaEventDisableTiming));
    VG_CU(cudaHostAlloc(reinterpret_cast<void **>(&kv->h_err), sizeof(int), cudaHostAllocMapped));
    *kv->h_err = 0;
    VG_CU(cudaHostGetDevicePointer(reinterpret_cast<void **>(&kv->d_err), kv->h_err, 0));
    kv->view.weights = kv->weights.as<float>();
    kv->view.heads = static_cast<uint32_t>(p.num_kv_heads);
    kv->view.dim = static_cast<uint32_t>(p.head_dim);
    kv->view.block = static_cast<uint32_t>(p.block_tokens);
    kv->view.block_shift = p.block_tokens == 16 ? 4 : p.block_tokens == 32 ? 5 : p.block_tokens == 64 ? 6 : 7;
    kv->view.stride = static_cast<uint32_t>(stride);
    *out = kv.release();
    return VG_OK;
  });
}

int vg_kv_destroy(vg_kv_cache *kv) {
  if (!kv) return VG_OK;
  DeviceGuard g(kv->device);
  delete kv;
  return VG_OK;
}

int vg_kv_get_info(const vg_kv_cache *kv, vg_kv_info *out) {
  return guarded([&]() -> int {
    if (!kv || !out) return fail(VG_ERR_INVALID_PARAMETER, "null argument");
    *out = vg_kv_info{};
    out->num_seqs = kv->params.num_seqs;
    out->capacity = kv->params.capacity;
    out->num_kv_heads = kv->params.num_kv_heads;
    out->head_dim = kv->params.head_dim;
    out->block_tokens = kv->params.block_tokens;
    out->weight_stride = kv->view.stride;
    out->device_bytes = kv->codes[0].cap + kv->codes[1].cap + kv->scales[0].cap + kv->scales[1].cap + kv->weights.cap +
                        kv->ws_lse.cap + kv->ws_kept.cap + kv->ws_part.cap + kv->ws_scores.cap + kv->ws_tiles.cap;
    out->device = kv->device;
    return VG_OK;
  });
}

int vg_kv_lengths(const vg_kv_cache *kv, uint32_t *out) {
  return guarded([&]() -> int {
    if (!kv || !out) return fail(VG_ERR_INVALID_PARAMETER, "null argument");
    std::copy(kv->len.begin(), kv->len.end(), out);
    return VG_OK;
  });
}

int vg_kv_truncate(vg_kv_cache *kv, const uint32_t *lengths) {
  return guarded([&]() -> int {
    if (!kv || !lengths) return fail(VG_ERR_INVALID_PARAMETER, "null argument");
    for (size_t s = 0; s < kv->len.size(); ++s)
      if (lengths[s] > kv->len[s])
        return fail(VG_ERR_INVALID_PARAMETER, "sequence " + std::to_string(s) + " holds " +
                                                  std::to_string(kv->len[s]) + " tokens: cannot be truncated to " +
                                                  std::to_string(lengths[s]));
    std::copy(lengths, lengths + kv->len.size(), kv->len.begin());
    return VG_OK;
  });
}

int vg_kv_weights(const vg_kv_cache *kv, float **out) {
  return guarded([&]() -> int {
    if (!kv || !out) return fail(VG_ERR_INVALID_PARAMETER, "null argument");
    *out = kv->view.weights;
    return VG_OK;
  });
}

int vg_kv_append(vg_kv_cache *kv, const uint32_t *counts, int dtype, const vg_heads *k, const vg_heads *v,
                 void *stream) {
  return guarded([&]() -> int {
    if (!kv || !counts) return fail(VG_ERR_INVALID_PARAMETER, "null argument");
    VG_TRY(check_dtype(dtype));
    size_t rows = 0;
    VG_TRY(total_rows(kv, counts, &rows));
    for (size_t s = 0; s < kv->len.size(); ++s)
      if (counts[s] > kv->params.capacity - kv->len[s])
        return fail(VG_ERR_INVALID_PARAMETER, "sequence " + std::to_string(s) + " would pass its capacity of " +
                                                  std::to_string(kv->params.capacity) + " tokens");
    if (rows == 0) return VG_OK;
    DeviceGuard g(kv->device);
    VG_TRY(check_heads(k, "k", rows, kv->params.head_dim, dtype, kv->device, false));
    VG_TRY(check_heads(v, "v", rows, kv->params.head_dim, dtype, kv->device, false));
    if (k->num_heads != kv->params.num_kv_heads || v->num_heads != kv->params.num_kv_heads)
      return fail(VG_ERR_DIMENSION_MISMATCH, "k and v must have the cache's key/value heads");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    Work work(kv, stream);
    VG_TRY(work.begin());
    const uint32_t sh = kv->view.block_shift;
    VG_TRY(for_plans(
        kv, counts,
        [&](size_t, PlanSeq &e) { return ((e.len + e.count - 1) >> sh) - (e.len >> sh) + 1; },
        [&](const Plan &plan) { return launch_kv_append(kv->view, plan, dtype, strided(*k), strided(*v), s); }));
    for (size_t i = 0; i < kv->len.size(); ++i) kv->len[i] += counts[i];
    return VG_OK;
  });
}

int vg_kv_attend(vg_kv_cache *kv, const uint32_t *counts, int dtype, const vg_heads *q, const vg_heads *out,
                 float *lse, float scale, int flags, void *stream) {
  return guarded([&]() -> int {
    if (!kv || !counts) return fail(VG_ERR_INVALID_PARAMETER, "null argument");
    VG_TRY(check_dtype(dtype));
    if (dtype == VG_F32) return fail(VG_ERR_UNSUPPORTED, "unsupported: queries are VG_F16 or VG_BF16");
    if (!std::isfinite(scale)) return fail(VG_ERR_INVALID_PARAMETER, "scale must be finite");
    if (flags & ~(VG_KV_CAUSAL | VG_KV_ACCUMULATE)) return fail(VG_ERR_INVALID_PARAMETER, "unknown flags");
    size_t rows = 0;
    VG_TRY(total_rows(kv, counts, &rows));
    if (rows == 0) return VG_OK;
    DeviceGuard g(kv->device);
    VG_TRY(check_heads(q, "q", rows, kv->params.head_dim, dtype, kv->device, false));
    VG_TRY(check_heads(out, "out", rows, kv->params.head_dim, dtype, kv->device, true));
    if (q->num_heads % kv->params.num_kv_heads)
      return fail(VG_ERR_DIMENSION_MISMATCH, "the query heads must be a multiple of the cache's key/value heads");
    if (out->num_heads != q->num_heads) return fail(VG_ERR_DIMENSION_MISMATCH, "out must have the heads of q");
    if (out->data == q->data && ((rows > 1 && out->token_stride != q->token_stride) ||
                                 (q->num_heads > 1 && out->head_stride != q->head_stride)))
      return fail(VG_ERR_INVALID_PARAMETER, "out in place must have the strides of q");
    if (rows * (q->num_heads / kv->params.num_kv_heads) > 0x7fffffffull)
      return fail(VG_ERR_INVALID_PARAMETER, "too many queries in one call");
    if (lse) VG_TRY(check_device_memory(lse, sizeof(float), kv->device, "lse"));
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    Work work(kv, stream);
    VG_TRY(work.begin());
    AttendArgs a{};
    a.kv = kv->view;
    a.dtype = dtype;
    a.q = strided(*q);
    a.out = strided(*out);
    a.q_heads = static_cast<uint32_t>(q->num_heads);
    a.group = a.q_heads / kv->view.heads;
    a.scale = scale;
    a.causal = (flags & VG_KV_CAUSAL) != 0;
    a.lse = lse;
    a.error = kv->d_err;
    if (flags & VG_KV_ACCUMULATE) {
      VG_TRY(reserve(kv->ws_lse, rows * a.q_heads * sizeof(float2)));
      a.lse2 = kv->ws_lse.as<float2>();
    }
    // by the rows of a key/value head: 16 in the decoding kernel, one row tile, more
    const auto no_units = [](size_t, PlanSeq &) { return 0u; };
    const auto rows_of = [&](uint32_t count) { return uint64_t(count) * a.group; };
    VG_TRY(for_plans_of(kv, counts, [&](uint32_t c) { return rows_of(c) <= kDecodeRows; }, no_units,
                        [&](Plan &plan) { return attend_decode(kv, a, plan, s); }));
    VG_TRY(for_plans_of(kv, counts, [&](uint32_t c) { return rows_of(c) > kDecodeRows && rows_of(c) <= kTileRows; },
                        no_units, [&](Plan &plan) { return attend_tiles(kv, a, plan, 1, s); }));
    VG_TRY(for_plans_of(kv, counts, [&](uint32_t c) { return rows_of(c) > kTileRows; }, no_units,
                        [&](Plan &plan) { return attend_tiles(kv, a, plan, 2, s); }));
    return VG_OK;
  });
}

int vg_kv_evict(vg_kv_cache *kv, size_t n, const uint32_t *src, const uint32_t *dst, size_t budget, size_t recent,
                int32_t *kept, void *stream) {
  return guarded([&]() -> int {
    if (!kv || (n && (!src || !dst))) return fail(VG_ERR_INVALID_PARAMETER, "null argument");
    if (budget == 0 || budget > kv->params.capacity)
      return fail(VG_ERR_INVALID_PARAMETER, "budget must be 1 to the capacity");
    if (recent > budget) return fail(VG_ERR_INVALID_PARAMETER, "recent must be at most budget");
    std::vector<char> seen(kv->len.size(), 0);
    for (size_t i = 0; i < n; ++i)
      for (uint32_t s : {src[i], dst[i]}) {
        if (s >= kv->len.size())
          return fail(VG_ERR_INVALID_PARAMETER, "no sequence " + std::to_string(s) + ": the cache's are below " +
                                                    std::to_string(kv->len.size()));
        if (seen[s]) return fail(VG_ERR_INVALID_PARAMETER, "sequence " + std::to_string(s) + " appears twice");
        seen[s] = 1;
      }
    if (n == 0) return VG_OK;
    DeviceGuard g(kv->device);
    if (kept) VG_TRY(check_device_memory(kept, sizeof(int32_t), kv->device, "kept"));
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    Work work(kv, stream);
    VG_TRY(work.begin());
    const size_t row = kv->params.num_kv_heads * budget;
    if (!kept) {
      VG_TRY(reserve(kv->ws_kept, n * row * sizeof(int32_t)));
      kept = kv->ws_kept.as<int32_t>();
    }
    Plan plan;
    for (size_t i0 = 0; i0 < n; i0 += kPlanSeqs) {
      plan.n = static_cast<uint32_t>(std::min<size_t>(n - i0, kPlanSeqs));
      uint64_t units = 0;
      for (uint32_t i = 0; i < plan.n; ++i) {
        PlanSeq &e = plan.s[i];
        e.seq = src[i0 + i];
        e.len = kv->len[e.seq];
        e.count = static_cast<uint32_t>(budget);
        e.row0 = dst[i0 + i];
        e.unit0 = static_cast<uint32_t>(units);
        units += ceil_div(std::min(e.len, e.count), kv->view.block);
      }
      VG_TRY(check_grid(kv, units));
      plan.units = static_cast<uint32_t>(units);
      VG_CU(launch_kv_select(kv->view, plan, static_cast<uint32_t>(budget), static_cast<uint32_t>(recent),
                             kept + i0 * row, s));
      VG_CU(launch_kv_gather(kv->view, plan, static_cast<uint32_t>(budget), kept + i0 * row, s));
    }
    for (size_t i = 0; i < n; ++i) kv->len[dst[i]] = std::min(kv->len[src[i]], static_cast<uint32_t>(budget));
    return VG_OK;
  });
}

int vg_kv_read(vg_kv_cache *kv, const uint32_t *starts, const uint32_t *counts, int dtype, const vg_heads *k,
               const vg_heads *v, void *stream) {
  return guarded([&]() -> int {
    if (!kv || !starts || !counts) return fail(VG_ERR_INVALID_PARAMETER, "null argument");
    VG_TRY(check_dtype(dtype));
    size_t rows = 0;
    VG_TRY(total_rows(kv, counts, &rows));
    for (size_t s = 0; s < kv->len.size(); ++s)
      if (counts[s] && (starts[s] > kv->len[s] || counts[s] > kv->len[s] - starts[s]))
        return fail(VG_ERR_INVALID_PARAMETER, "sequence " + std::to_string(s) + " holds only " +
                                                  std::to_string(kv->len[s]) + " tokens");
    if (rows == 0) return VG_OK;
    DeviceGuard g(kv->device);
    VG_TRY(check_heads(k, "k", rows, kv->params.head_dim, dtype, kv->device, true));
    VG_TRY(check_heads(v, "v", rows, kv->params.head_dim, dtype, kv->device, true));
    if (k->num_heads != kv->params.num_kv_heads || v->num_heads != kv->params.num_kv_heads)
      return fail(VG_ERR_DIMENSION_MISMATCH, "k and v must have the cache's key/value heads");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    Work work(kv, stream);
    VG_TRY(work.begin());
    VG_TRY(for_plans(
        kv, counts,
        [&](size_t seq, PlanSeq &e) {
          e.len = starts[seq];
          return ceil_div(e.count, kReadTile);
        },
        [&](const Plan &plan) { return launch_kv_read(kv->view, plan, dtype, strided(*k), strided(*v), s); }));
    return VG_OK;
  });
}

}  // extern "C"

namespace {

// Scales of a host or device array as the kernels take them: their exponents
// are used as they are.
int check_scales(const float *scales, size_t n, const char *name, cudaStream_t s) {
  std::vector<uint32_t> bits(std::min<size_t>(n, size_t(1) << 18));
  for (size_t at = 0; at < n; at += bits.size()) {
    const size_t m = std::min(n - at, bits.size());
    VG_CU(cudaMemcpyAsync(bits.data(), scales + at, m * sizeof(float), cudaMemcpyDefault, s));
    VG_CU(cudaStreamSynchronize(s));
    for (size_t i = 0; i < m; ++i) {
      const uint32_t b = bits[i], e = b >> 23;  // the sign would be the exponent's ninth bit
      const bool nan = (b & 0x7fffffffu) > 0x7f800000u;
      if (!nan && ((b & 0x7fffffu) || e < 127 + kMinScaleExp || e > 127 + kMaxScaleExp))
        return fail(VG_ERR_INVALID_PARAMETER,
                    std::string(name) + " must be scales: powers of two in [2^-100, 2^120], or NaN (entry " +
                        std::to_string(at + i) + ")");
    }
  }
  return VG_OK;
}

// What a strided copy takes as the distance between rows, on any device so far.
constexpr size_t kMaxPitch = 0x7fffffff;

// `rows` rows of `bytes` each between a host or device array and the cache:
// one copy for all heads (32 heads of 4,096 tokens x 128 from device arrays:
// 102 us a load, 549 with a copy for each head and array).
int copy_rows(void *dst, size_t dst_pitch, const void *src, size_t src_pitch, size_t bytes, size_t rows,
              cudaStream_t s) {
  if (std::max(dst_pitch, src_pitch) <= kMaxPitch) {
    VG_CU(cudaMemcpy2DAsync(dst, dst_pitch, src, src_pitch, bytes, rows, cudaMemcpyDefault, s));
    return VG_OK;
  }
  for (size_t i = 0; i < rows; ++i)
    VG_CU(cudaMemcpyAsync(static_cast<char *>(dst) + i * dst_pitch, static_cast<const char *>(src) + i * src_pitch,
                          bytes, cudaMemcpyDefault, s));
  return VG_OK;
}

// The arrays of one sequence in the cache, and what a row of each holds of `length` tokens.
struct SequenceRows {
  int8_t *codes[2];
  float *scales[2], *weights;
  size_t code_bytes, scale_bytes, weight_bytes;     // of a head
  size_t code_pitch, scale_pitch, weight_pitch;     // from head to head
  SequenceRows(const KvView &w, size_t seq, size_t length) {
    const size_t r = seq * w.heads, nb = w.stride >> w.block_shift;
    for (int i = 0; i < 2; ++i) {
      codes[i] = w.codes[i] + r * w.stride * w.dim;
      scales[i] = w.scales[i] + r * nb;
    }
    weights = w.weights + r * w.stride;
    code_bytes = length * w.dim;
    scale_bytes = ((length + w.block - 1) >> w.block_shift) * sizeof(float);
    weight_bytes = length * sizeof(float);
    code_pitch = static_cast<size_t>(w.stride) * w.dim;
    scale_pitch = nb * sizeof(float);
    weight_pitch = w.stride * sizeof(float);
  }
};

}  // namespace

extern "C" {

int vg_kv_load(vg_kv_cache *kv, size_t seq, size_t length, const int8_t *k_codes, const float *k_scales,
               const int8_t *v_codes, const float *v_scales, const float *weights, void *stream) {
  return guarded([&]() -> int {
    if (!kv) return fail(VG_ERR_INVALID_PARAMETER, "null argument");
    if (seq >= kv->len.size()) return fail(VG_ERR_INVALID_PARAMETER, "no sequence " + std::to_string(seq));
    if (length > kv->params.capacity) return fail(VG_ERR_INVALID_PARAMETER, "length is over the capacity");
    if (length && (!k_codes || !k_scales || !v_codes || !v_scales))
      return fail(VG_ERR_INVALID_PARAMETER, "null codes or scales");
    DeviceGuard g(kv->device);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    Work work(kv, stream);
    VG_TRY(work.begin());
    const SequenceRows to(kv->view, seq, length);
    const size_t heads = kv->view.heads;
    const int8_t *codes[2] = {k_codes, v_codes};
    const float *scales[2] = {k_scales, v_scales};
    if (length) {
      for (int i = 0; i < 2; ++i)
        VG_TRY(check_scales(scales[i], heads * (to.scale_bytes / sizeof(float)), i ? "v_scales" : "k_scales", s));
      for (int i = 0; i < 2; ++i) {
        VG_TRY(copy_rows(to.codes[i], to.code_pitch, codes[i], to.code_bytes, to.code_bytes, heads, s));
        VG_TRY(copy_rows(to.scales[i], to.scale_pitch, scales[i], to.scale_bytes, to.scale_bytes, heads, s));
      }
      if (weights) VG_TRY(copy_rows(to.weights, to.weight_pitch, weights, to.weight_bytes, to.weight_bytes, heads, s));
      else VG_CU(cudaMemsetAsync(to.weights, 0, to.weight_pitch * heads, s));  // past the length too: unused
    }
    VG_CU(cudaStreamSynchronize(s));
    kv->len[seq] = static_cast<uint32_t>(length);
    return VG_OK;
  });
}

int vg_kv_export(vg_kv_cache *kv, size_t seq, int8_t *k_codes, float *k_scales, int8_t *v_codes, float *v_scales,
                 float *weights, void *stream) {
  return guarded([&]() -> int {
    if (!kv) return fail(VG_ERR_INVALID_PARAMETER, "null argument");
    if (seq >= kv->len.size()) return fail(VG_ERR_INVALID_PARAMETER, "no sequence " + std::to_string(seq));
    const size_t length = kv->len[seq];
    if (length && (!k_codes || !k_scales || !v_codes || !v_scales))
      return fail(VG_ERR_INVALID_PARAMETER, "null codes or scales");
    DeviceGuard g(kv->device);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    Work work(kv, stream);
    VG_TRY(work.begin());
    const SequenceRows from(kv->view, seq, length);
    const size_t heads = kv->view.heads;
    int8_t *codes[2] = {k_codes, v_codes};
    float *scales[2] = {k_scales, v_scales};
    if (length) {
      for (int i = 0; i < 2; ++i) {
        VG_TRY(copy_rows(codes[i], from.code_bytes, from.codes[i], from.code_pitch, from.code_bytes, heads, s));
        VG_TRY(copy_rows(scales[i], from.scale_bytes, from.scales[i], from.scale_pitch, from.scale_bytes, heads, s));
      }
      if (weights)
        VG_TRY(copy_rows(weights, from.weight_bytes, from.weights, from.weight_pitch, from.weight_bytes, heads, s));
    }
    VG_CU(cudaStreamSynchronize(s));
    return VG_OK;
  });
}

}  // extern "C"
