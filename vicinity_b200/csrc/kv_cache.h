// Device-side view of a key/value cache and the launchers of its kernels
// (rotary.cu, kv_store.cu, kv_attend.cu, kv_attend_tc.cu).
//
// Layout, per (sequence, key/value head) row r = seq * heads + head:
//   codes   int8 [2: K, V][rows][stride][dim]   token-major
//   scales  f32  [2][rows][stride / block]      powers of two
//   weights f32  [rows][stride]
// stride is the capacity rounded up to kKvPad tokens, so a tile of up to
// kKvPad tokens that starts on a multiple of its size is one contiguous range
// inside the row, whatever the sequence's length.  Memory past a sequence's
// length holds finite codes but any scale: readers select, never multiply,
// it away.
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace vg {

constexpr uint32_t kKvPad = 128;
constexpr int kMinScaleExp = -100, kMaxScaleExp = 120;  // scales are 2^e, or NaN
// Sequences per launch: the plan travels as a kernel argument, 8 KB or, up to
// kSmallPlan of them, half a KB (which takes 1.2 us less to launch).
constexpr int kPlanSeqs = 256, kSmallPlan = 16;

struct KvView {
  int8_t *codes[2];
  float *scales[2];
  float *weights;
  uint32_t heads, dim, block, block_shift, stride;
};

// One sequence of a launch.  unit0: the first of the launch's work units that
// belongs to it (what a unit is, the kernel says).
struct PlanSeq {
  uint32_t seq;    // slot in the cache
  uint32_t len;    // tokens cached when the kernel runs
  uint32_t count;  // tokens of this call
  uint32_t row0;   // first of them in the packed tensors
  uint32_t unit0;
  uint32_t block0;  // the first of the launch's blocks of kTileRows rows that belongs to it
  uint64_t aux;     // offset of its scores
};
template <int N>
struct PlanOf {
  uint32_t n, units;
  PlanSeq s[N];
};
using Plan = PlanOf<kPlanSeqs>;

// f(the plan in the smallest form that holds it)
template <class F>
cudaError_t with_plan(const Plan &plan, F &&f) {
  if (plan.n > kSmallPlan) return f(plan);
  PlanOf<kSmallPlan> small;
  small.n = plan.n;
  small.units = plan.units;
  for (uint32_t i = 0; i < plan.n; ++i) small.s[i] = plan.s[i];
  return f(small);
}

struct Strided {
  void *p;
  int64_t token, head;  // strides in elements
};

// Entry of the plan that work unit u belongs to (entries without units are skipped).
template <class P>
__device__ __forceinline__ uint32_t plan_find(const P &plan, uint32_t u) {
  uint32_t lo = 0, hi = plan.n;  // last entry with unit0 <= u
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) >> 1;
    if (plan.s[mid].unit0 <= u) lo = mid;
    else hi = mid;
  }
  return lo;
}

// ---- rotary.cu ----
struct RotaryTable {
  double turns[128];  // frequency / (2 pi)
  uint32_t pairs;
  int interleaved;
  float magnitude;
};
cudaError_t launch_rotary(const RotaryTable &t, int dtype, uint32_t dim, const int64_t *pos, size_t tokens,
                          const Strided &q, const Strided &qo, uint32_t q_heads, const Strided &k, const Strided &ko,
                          uint32_t k_heads, bool transpose, cudaStream_t s);

// ---- kv_store.cu ----
// Units: the blocks that a sequence's new tokens touch (len: before the append).
cudaError_t launch_kv_append(const KvView &kv, const Plan &plan, int dtype, const Strided &k, const Strided &v,
                             cudaStream_t s);
// Units: tiles of kReadTile tokens of [len, len + count) -- len is the first token read.
constexpr uint32_t kReadTile = 64;
cudaError_t launch_kv_read(const KvView &kv, const Plan &plan, int dtype, const Strided &k, const Strided &v,
                           cudaStream_t s);
// Selection: entry i keeps min(len, count = budget) tokens of sequence seq;
// kept i32 [entries][heads][budget].  row0 is the destination sequence.
cudaError_t launch_kv_select(const KvView &kv, const Plan &plan, uint32_t budget, uint32_t recent, int32_t *kept,
                             cudaStream_t s);
// Units: blocks of the destination.
cudaError_t launch_kv_gather(const KvView &kv, const Plan &plan, uint32_t budget, const int32_t *kept,
                             cudaStream_t s);

// ---- kv_attend.cu ----
constexpr int kDecodeRows = 16;      // rows (queries x heads that share a key/value head) of the decoding kernel
constexpr uint32_t kMaxSplits = 512;  // chunks of one sequence that are joined
struct AttendArgs {
  KvView kv;
  int dtype;
  Strided q, out;
  uint32_t q_heads, group;
  float scale;      // softmax scale
  bool causal;
  float *lse;       // [rows][q_heads] natural log (nullable)
  // [rows][q_heads] log2 for the weights, as a score and the rest; (0, inf) where no token is seen (nullable)
  float2 *lse2;
  // Splitting over the tokens: a unit takes `chunk` tokens; a sequence of more
  // than one unit leaves [unit][head][row of 16 or 128] partial sums
  uint32_t chunk;
  float *part_o;    // [..][dim]
  float4 *part_ml;  // [..] (references nu and mu - nu, denominator, -)
  // Scores x of the call's rows, for the weights (nullable): entry e has
  // [heads][len rounded up to 16][rows rounded up to 2] from scores + plan.s[e].aux
  float *scores;
  // Query tiles of the tile kernels, [row block][head], and the factors of
  // their rows, [row block][head][kTileRows]
  uint8_t *q_tiles;
  float *q_factor;
  int *error;       // set nonzero when a bounded wait gives up (host-mapped)
};
// Sequences of at most kDecodeRows rows per key/value head.  Units: chunks (at least one per sequence).
cudaError_t launch_kv_attend_decode(const AttendArgs &a, const Plan &plan, uint32_t max_rows, cudaStream_t s);
// Joins the partial sums of sequences that have more than one unit.
cudaError_t launch_kv_attend_join(const AttendArgs &a, const Plan &plan, uint32_t part_rows, uint32_t max_rows,
                                  cudaStream_t s);
// Adds the probabilities of stored scores to the weights.  Units: kWeighTile tokens.
constexpr uint32_t kWeighTile = 256;
cudaError_t launch_kv_weigh_scores(const AttendArgs &a, const Plan &plan, cudaStream_t s);

// ---- kv_attend_tc.cu ----
constexpr int kTileRows = 128;
size_t query_tile_bytes(uint32_t dim);
// blocks: row blocks of the plan (per head)
cudaError_t launch_kv_query_tiles(const AttendArgs &a, const Plan &plan, uint32_t blocks, cudaStream_t s);
// tiles: 1 or 2 row tiles a unit.  Units: blocks of tiles * kTileRows rows times chunks (at least one) of each sequence.
cudaError_t launch_kv_attend_tiles(const AttendArgs &a, const Plan &plan, uint32_t tiles, cudaStream_t s);
// Weights from recomputed scores.  Units: kWeighRows tokens.
constexpr uint32_t kWeighRows = 128;
cudaError_t launch_kv_weigh_tiles(const AttendArgs &a, const Plan &plan, cudaStream_t s);

}  // namespace vg
