// Attention over a key/value cache held in 8 bits.
//
// Scores are x = log2(e) scale q.k and the reference mu of a row's exponentials is
// the running maximum of x + log2(value scale): with P = 2^(x + log2 vs - mu) the
// sum of P times the value codes needs no other factor, and the denominator is
// the sum of P / vs (powers of two: exact), held relative to the running maximum
// nu of x alone.  Codes are exact in binary16, and a query row is scaled by a
// power of two into its range, so both products run on the tensor cores in
// binary16 with f32 sums; only P is rounded, to 11 bits: in more the second
// product would take two binary16 parts, twice the products of a kernel that
// is bound by them, for an error that an output in 16 bits hardly shows: f16
// outputs err by 2.1e-4 to 2.3e-4 of their norm against 2.05e-4 to 2.1e-4 in f32.
#include "chain.cuh"
#include "common.cuh"
#include "elements.cuh"
#include "kv_attend.cuh"
#include "kv_cache.h"

#include <algorithm>
#include <type_traits>

namespace vg {

namespace {

// ---- up to 16 query rows per key/value head ----------------------------------
//
// One token of decoding, or a few: bound by reading the codes once.  A CTA
// (two on an SM) takes (sequence, head, chunk of tokens); each of its warps walks its own
// 16-token steps, which it copies into its own shared-memory ring (cp.async,
// kRing - 1 steps ahead, no barrier between warps), converts to binary16 in
// registers and multiplies with mma.sync m16n8k16.  Tokens, then dimensions,
// are the 16 rows of a product and the queries its 8 columns (kCols: one or two
// groups of them): with the queries as rows, most of the 16 would be empty and
// there would be twice as many products.  Scores come out with a token per
// row; movmatrix turns the probabilities into the second product's operand.
// The order of the dimensions inside a product is free, so a lane takes whole
// words of a token: dim / 4 consecutive key dimensions, dim / 8 consecutive
// value dimensions.
// 131,101 tokens x 8 heads x 128, 4 rows a head (268 MB): 49 us, 5.5 TB/s; the
// copies alone take 46, the rest is the start and the end of the CTAs.
constexpr int kStep = 16;  // tokens per step: one scale each for keys and values (blocks are multiples of 16)

// byte offset of (token, byte of its row) in a stage: 16-byte chunks XORed so
// that the lanes of one load phase hit different banks
template <int D>
__device__ __forceinline__ uint32_t swz(uint32_t tok, uint32_t byte) {
  if (D == 128) return tok * D + (byte ^ ((tok & 7u) << 4));
  if (D == 64) return tok * D + (byte ^ (((tok >> 1) & 3u) << 4));
  return tok * D + byte;
}

// N words at byte offset `at` (a multiple of their size) of a row's chunk
template <int D, int N>
__device__ __forceinline__ void row_words(const uint8_t *st, uint32_t tok, uint32_t at, uint32_t (&w)[N]) {
  if (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const uint4 x = *reinterpret_cast<const uint4 *>(st + swz<D>(tok, at + 16 * i));
      w[4 * i] = x.x;
      w[4 * i + 1] = x.y;
      w[4 * i + 2] = x.z;
      w[4 * i + 3] = x.w;
    }
  } else if (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const uint2 x = *reinterpret_cast<const uint2 *>(st + swz<D>(tok, at + 8 * i));
      w[2 * i] = x.x;
      w[2 * i + 1] = x.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = *reinterpret_cast<const uint32_t *>(st + swz<D>(tok, at + 4 * i));
  }
}

// References of joined partial sums: the larger nu, and the lift from there to the larger mu.
__device__ __forceinline__ void join_references(float &nu, float &lift, float nu2, float lift2) {
  const float at = fmaxf(nu, nu2);
  lift = fmaxf(nu - at + lift, nu2 - at + lift2);
  nu = at;
}

// transposes an 8 x 8 matrix of binary16 (lane 4 r + c holds columns 2 c, 2 c + 1 of row r)
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// Warps of a CTA and their rings' stages, by kCols: what the registers of two
// CTAs on an SM allow, and some 64 KB on their way to an SM at any time.
template <int kCols>
struct Dec {
  static constexpr int warps = kCols == 1 ? 8 : 6, ring = kCols == 1 ? 3 : 4;
};

template <int D, int kCols, bool kScores, class P>
__global__ void __launch_bounds__(Dec<kCols>::warps * 32, 2)
    attend_decode_kernel(const __grid_constant__ AttendArgs a, const __grid_constant__ P plan, const bool qvec,
                         const bool ovec) {
  constexpr int kPlane = kStep * D;                    // bytes of one step's keys (or values)
  constexpr int kStage = 2 * kPlane + 16;              // and the two scales
  constexpr int kDecWarps = Dec<kCols>::warps, kRing = Dec<kCols>::ring;
  constexpr int kK = D / 16;                           // key words per lane and token = k-steps
  constexpr int kV = D / 32;                           // value words per lane and token
  constexpr uint32_t kRowsMax = 8 * kCols;
  extern __shared__ __align__(16) uint8_t dec_smem[];
  chain_release();
  const int warp = threadIdx.x >> 5, lane = lane_id(), n = lane >> 2, j = lane & 3;
  uint8_t *ring = dec_smem + warp * (kRing * kStage);
  const KvView &kv = a.kv;
  const uint32_t unit = blockIdx.x, entry = plan_find(plan, unit), head = blockIdx.y;
  const PlanSeq &ps = plan.s[entry];
  const uint32_t t0 = (unit - ps.unit0) * a.chunk, t1 = min(ps.len, t0 + a.chunk);
  const size_t r = static_cast<size_t>(ps.seq) * kv.heads + head;
  const int8_t *kc = kv.codes[0] + r * kv.stride * D, *vc = kv.codes[1] + r * kv.stride * D;
  const size_t nb = kv.stride >> kv.block_shift;
  const float *ks = kv.scales[0] + r * nb, *vs = kv.scales[1] + r * nb;

  const uint32_t steps = t1 > t0 ? (t1 - t0 + kStep - 1) / kStep : 0;
  auto fetch = [&](uint32_t step, uint32_t slot) {  // always one group, empty past the end
    if (step < steps) {
      uint8_t *st = ring + slot * kStage;
      const uint32_t t = t0 + step * kStep;
      const size_t at = static_cast<size_t>(t) * D + lane * 16;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        const uint32_t c = lane + 32 * i, tok = c / (D / 16), byte = (c % (D / 16)) * 16;
        cp_async16(st + swz<D>(tok, byte), kc + at + 512 * i);
        cp_async16(st + kPlane + swz<D>(tok, byte), vc + at + 512 * i);
      }
      if (lane < 2) cp_async4(st + 2 * kPlane + lane * 4, (lane ? vs : ks) + (t >> kv.block_shift));
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < kRing - 1; ++i) fetch(warp + i * kDecWarps, i);

  // the queries as B fragments: lane (n, j) holds its dimensions of row n of each group
  const uint32_t rows = ps.count * a.group;
  const uint32_t row_stride = (rows + 1) & ~1u;  // of the scores: [token][row_stride]
  float *scores = a.scores + ps.aux + static_cast<size_t>(head) * row_stride * ((ps.len + kStep - 1) / kStep * kStep);
  float q_scale[kCols];
  uint32_t qb[kCols][kK][2];
#pragma unroll
  for (int g = 0; g < kCols; ++g) {
    const uint32_t row = n + 8 * g;
    float x[D / 4];
    if (row < rows) {
      const uint32_t qi = row / a.group;
      const int64_t at = static_cast<int64_t>(ps.row0 + qi) * a.q.token +
                   static_cast<int64_t>(head * a.group + row - qi * a.group) * a.q.head + j * (D / 4);
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
        load8_16(a.q.p, at + 8 * i, a.dtype == VG_F16, qvec, *reinterpret_cast<float(*)[8]>(x + 8 * i));
    } else {
#pragma unroll
      for (int i = 0; i < D / 4; ++i) x[i] = 0.0f;
    }
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < D / 4; ++i) top = fmaxf(top, fabsf(x[i]));
    top = fmaxf(top, __shfl_xor_sync(VG_FULL_MASK, top, 1));
    top = fmaxf(top, __shfl_xor_sync(VG_FULL_MASK, top, 2));
    float inv;
    row_scale(top, q_scale[g], inv);
    q_scale[g] *= fabsf(a.scale) * kLog2e;
    if (a.scale < 0.0f) inv = -inv;  // factors of the products are not negative
#pragma unroll
    for (int s = 0; s < kK; ++s) {
      qb[g][s][0] = pack_half2(x[4 * s] * inv, x[4 * s + 1] * inv);
      qb[g][s][1] = pack_half2(x[4 * s + 2] * inv, x[4 * s + 3] * inv);
    }
  }
  // results: a lane has rows 2 j and 2 j + 1 of each group, tokens n and n + 8
  uint32_t lim[2 * kCols], all_see = t1;
  float qs[2 * kCols];
#pragma unroll
  for (int h = 0; h < 2 * kCols; ++h) {
    const uint32_t row = 8 * (h >> 1) + 2 * j + (h & 1);
    qs[h] = __shfl_sync(VG_FULL_MASK, q_scale[h >> 1], 4 * (2 * j + (h & 1)));
    lim[h] = row < rows ? tokens_seen(ps, row / a.group, a.causal) : t1;
    all_see = min(all_see, lim[h]);
  }
  all_see = __reduce_min_sync(VG_FULL_MASK, all_see);

  float o[kCols][D / 16][4];
#pragma unroll
  for (int g = 0; g < kCols; ++g)
#pragma unroll
    for (int i = 0; i < D / 16; ++i) o[g][i][0] = o[g][i][1] = o[g][i][2] = o[g][i][3] = 0.0f;
  float nu[2 * kCols], lift[2 * kCols], l[2 * kCols];
#pragma unroll
  for (int h = 0; h < 2 * kCols; ++h) {
    nu[h] = kUnseen;
    lift[h] = 0.0f;
    l[h] = 0.0f;
  }

  uint32_t slot = 0;
  for (uint32_t step = warp; step < steps; step += kDecWarps) {
    fetch(step + (kRing - 1) * kDecWarps, slot == 0 ? kRing - 1 : slot - 1);
    cp_async_wait<kRing - 1>();
    __syncwarp();
    const uint8_t *st = ring + slot * kStage;
    slot = slot + 1 == kRing ? 0 : slot + 1;
    const uint32_t t = t0 + step * kStep;
    float s[kCols][4] = {};  // (token n, rows 2 j, 2 j + 1), (token n + 8, ...)
    {
      uint32_t w0[kK], w1[kK];
      row_words<D>(st, n, j * (D / 4), w0);
      row_words<D>(st, n + 8, j * (D / 4), w1);
#pragma unroll
      for (int c = 0; c < kK; ++c) {
        const uint32_t x0 = w0[c] ^ 0x80808080u, x1 = w1[c] ^ 0x80808080u;
        const uint32_t ka[4] = {half2_of<0x4140>(x0), half2_of<0x4140>(x1), half2_of<0x4342>(x0), half2_of<0x4342>(x1)};
#pragma unroll
        for (int g = 0; g < kCols; ++g) mma_f16(s[g], ka, qb[g][c][0], qb[g][c][1]);
      }
    }
    const float2 scale = *reinterpret_cast<const float2 *>(st + 2 * kPlane);  // of keys, of values
    const float lv = log2_scale(scale.y), per_v = inverse_scale(scale.y);
    float f[2 * kCols];
#pragma unroll
    for (int h = 0; h < 2 * kCols; ++h) f[h] = scale.x * qs[h];
    if (t + kStep > all_see) {  // where a factor is 0 or NaN, -inf would not stay: scores from here on
#pragma unroll
      for (int h = 0; h < 2 * kCols; ++h) {
        float &x = s[h >> 1][h & 1], &y = s[h >> 1][2 + (h & 1)];
        x = t + n < lim[h] ? x * f[h] : -VG_INF;
        y = t + n + 8 < lim[h] ? y * f[h] : -VG_INF;
        f[h] = 1.0f;
      }
    }
    if (kScores) {
#pragma unroll
      for (int g = 0; g < kCols; ++g)
        if (8u * g + 2 * j < rows) {
          float *sc = scores + static_cast<size_t>(t + n) * row_stride + 8 * g + 2 * j;
          *reinterpret_cast<float2 *>(sc) = make_float2(s[g][0] * f[2 * g], s[g][1] * f[2 * g + 1]);
          *reinterpret_cast<float2 *>(sc + 8 * row_stride) = make_float2(s[g][2] * f[2 * g], s[g][3] * f[2 * g + 1]);
        }
    }
    bool raise = false;
#pragma unroll
    for (int h = 0; h < 2 * kCols; ++h) {
      const float above = __fmul_rn(fmaxf(s[h >> 1][h & 1], s[h >> 1][2 + (h & 1)]), f[h]) - nu[h];
      raise |= fmaxf(above, above + (lv - lift[h])) > kLazy;
    }
    if (__any_sync(VG_FULL_MASK, raise)) {
#pragma unroll
      for (int h = 0; h < 2 * kCols; ++h) {
        float x = __fmul_rn(fmaxf(s[h >> 1][h & 1], s[h >> 1][2 + (h & 1)]), f[h]);
#pragma unroll
        for (int w = 4; w < 32; w <<= 1) x = fmaxf(x, __shfl_xor_sync(VG_FULL_MASK, x, w));
        const float c = raise_references(nu[h], lift[h], x, lv, l[h]);
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          o[h >> 1][i][h & 1] *= c;
          o[h >> 1][i][2 + (h & 1)] *= c;
        }
      }
    }
    uint32_t pb[kCols][2];
#pragma unroll
    for (int g = 0; g < kCols; ++g) {
      float p[4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const PowerRefs refs(nu[2 * g + h], lift[2 * g + h]);
        const float shift = refs.shift(lv);
        p[h] = exp2_approx(__fmul_rn(s[g][h], f[2 * g + h]) - nu[2 * g + h] + shift);
        p[2 + h] = exp2_approx(__fmul_rn(s[g][2 + h], f[2 * g + h]) - nu[2 * g + h] + shift);
        l[2 * g + h] = fmaf(p[h] + p[2 + h], refs.share(per_v), l[2 * g + h]);
        if (scale.y != scale.y) {  // the values read as NaN: so does every row that sees one of them
          if (t + n < lim[2 * g + h]) p[h] = scale.y;
          if (t + n + 8 < lim[2 * g + h]) p[2 + h] = scale.y;
        }
      }
      pb[g][0] = transposed(pack_half2(p[0], p[1]));
      pb[g][1] = transposed(pack_half2(p[2], p[3]));
    }
    {
      uint32_t w[4][kV];  // tokens 2 j, 2 j + 1, 2 j + 8, 2 j + 9
#pragma unroll
      for (int c = 0; c < 4; ++c)
        row_words<D>(st + kPlane, 2 * j + (c & 1) + 8 * (c >> 1), n * (D / 8), w[c]);
#pragma unroll
      for (int c = 0; c < kV; ++c) {
#pragma unroll
        for (int hi = 0; hi < 2; ++hi) {
          const uint32_t sel = hi ? 0x7362u : 0x5140u;
          const uint32_t x0 = __byte_perm(w[0][c], w[1][c], sel) ^ 0x80808080u;
          const uint32_t x1 = __byte_perm(w[2][c], w[3][c], sel) ^ 0x80808080u;
          const uint32_t va[4] = {half2_of<0x4140>(x0), half2_of<0x4342>(x0), half2_of<0x4140>(x1), half2_of<0x4342>(x1)};
#pragma unroll
          for (int g = 0; g < kCols; ++g) mma_f16(o[g][2 * c + hi], va, pb[g][0], pb[g][1]);
        }
      }
    }
    __syncwarp();  // the slot is free for the next fetch
  }

  // join the warps, then write the rows out or, one chunk of several, as partial sums
#pragma unroll
  for (int h = 0; h < 2 * kCols; ++h)
#pragma unroll
    for (int w = 4; w < 32; w <<= 1) l[h] += __shfl_xor_sync(VG_FULL_MASK, l[h], w);
  cp_async_wait<0>();
  __syncthreads();
  // [warp][row][D], rows padded so that a lane's pairs of dimensions spread over the banks
  constexpr int kPad = D + 2;
  float *so = reinterpret_cast<float *>(dec_smem);
  float4 *sml = reinterpret_cast<float4 *>(so + kDecWarps * kRowsMax * kPad);  // [warp][row]
#pragma unroll
  for (int h = 0; h < 2 * kCols; ++h) {
    const uint32_t row = 8 * (h >> 1) + 2 * j + (h & 1);
    float *dst = so + (warp * kRowsMax + row) * kPad + n * (D / 8);
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
      *reinterpret_cast<float2 *>(dst + 2 * i) = make_float2(o[h >> 1][i][h & 1], o[h >> 1][i][2 + (h & 1)]);
    if (n == 0) sml[warp * kRowsMax + row] = make_float4(nu[h], lift[h], l[h], 0.0f);
  }
  __syncthreads();
  const bool whole = ps.len <= a.chunk;
  for (uint32_t e = threadIdx.x; e < rows * (D / 8); e += kDecWarps * 32) {
    const uint32_t row = e / (D / 8), c = e % (D / 8) * 8;
    // the largest nu, and the lift from there to the largest mu
    float top_nu = kUnseen, top_lift = kUnseen, sum = 0.0f, y[8] = {};
#pragma unroll
    for (int w = 0; w < kDecWarps; ++w) top_nu = fmaxf(top_nu, sml[w * kRowsMax + row].x);
#pragma unroll
    for (int w = 0; w < kDecWarps; ++w) {
      const float4 ml = sml[w * kRowsMax + row];
      top_lift = fmaxf(top_lift, ml.x - top_nu + ml.y);
    }
#pragma unroll
    for (int w = 0; w < kDecWarps; ++w) {
      const float4 ml = sml[w * kRowsMax + row];
      const float f = exp2_approx(ml.x - top_nu + (ml.y - top_lift));
      sum += exp2_approx(ml.x - top_nu) * ml.z;
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] += f * so[(w * kRowsMax + row) * kPad + c + i];
    }
    if (whole) {
      const uint32_t qi = row / a.group, hq = head * a.group + row - qi * a.group;
      finish_row(a, static_cast<size_t>(ps.row0) + qi, hq, c, ovec, top_nu, top_lift, sum, y);
    } else {
      const size_t at = (static_cast<size_t>(unit) * kv.heads + head) * kDecodeRows + row;
      float *dst = a.part_o + at * D + c;
      *reinterpret_cast<float4 *>(dst) = make_float4(y[0], y[1], y[2], y[3]);
      *reinterpret_cast<float4 *>(dst + 4) = make_float4(y[4], y[5], y[6], y[7]);
      if (c == 0) a.part_ml[at] = make_float4(top_nu, top_lift, sum, 0.0f);
    }
  }
}

// ---- joining the chunks of a sequence -------------------------------------------

// One CTA per (row, head, sequence): 32-byte slices of the row's partial sums,
// groups of threads taking every kGroups-th chunk.  Latency: about 5 us.  (By
// the last CTA of the first kernel instead of a launch: 14 us for 74 chunks.)
constexpr int kJoinThreads = 256;

template <class P>
__global__ void __launch_bounds__(kJoinThreads) attend_join_kernel(const __grid_constant__ AttendArgs a,
                                                                   const __grid_constant__ P plan,
                                                                   const uint32_t part_rows, const bool ovec) {
  __shared__ float weight[kMaxSplits];
  __shared__ float2 red[kJoinThreads / 32];
  __shared__ float acc[kJoinThreads * 8];
  chain_release();
  chain_wait();
  const PlanSeq &ps = plan.s[blockIdx.z];
  const uint32_t head = blockIdx.y, row = blockIdx.x, D = a.kv.dim, rows = ps.count * a.group;
  if (ps.len <= a.chunk || row >= rows) return;
  const uint32_t ns = (ps.len + a.chunk - 1) / a.chunk;
  const size_t step = static_cast<size_t>(a.kv.heads) * part_rows;
  // a sequence's units: its row blocks, the last one first, and the chunks of each
  const uint32_t block = (rows + part_rows - 1) / part_rows - 1 - row / part_rows;
  const size_t first =
      ((static_cast<size_t>(ps.unit0) + block * ns) * a.kv.heads + head) * part_rows + row % part_rows;
  const int warp = threadIdx.x >> 5;
  float nu = kUnseen, lift = 0.0f;
  for (uint32_t i = threadIdx.x; i < ns; i += kJoinThreads) {
    const float4 ml = a.part_ml[first + i * step];
    join_references(nu, lift, ml.x, ml.y);
  }
#pragma unroll
  for (int w = 16; w > 0; w >>= 1) {
    const float nu2 = __shfl_xor_sync(VG_FULL_MASK, nu, w), lift2 = __shfl_xor_sync(VG_FULL_MASK, lift, w);
    join_references(nu, lift, nu2, lift2);
  }
  if (lane_id() == 0) red[warp] = make_float2(nu, lift);
  __syncthreads();
  for (int w = 0; w < kJoinThreads / 32; ++w) join_references(nu, lift, red[w].x, red[w].y);
  __syncthreads();
  float sum = 0.0f;
  for (uint32_t i = threadIdx.x; i < ns; i += kJoinThreads) {
    const float4 ml = a.part_ml[first + i * step];
    weight[i] = exp2_approx(ml.x - nu + (ml.y - lift));
    sum += exp2_approx(ml.x - nu) * ml.z;
  }
#pragma unroll
  for (int w = 16; w > 0; w >>= 1) sum += __shfl_xor_sync(VG_FULL_MASK, sum, w);
  if (lane_id() == 0) red[warp].x = sum;
  __syncthreads();
  sum = 0.0f;
  for (int w = 0; w < kJoinThreads / 32; ++w) sum += red[w].x;
  const uint32_t per = D / 8, groups = kJoinThreads / per, g = threadIdx.x / per, c = threadIdx.x % per * 8;
  float y[8] = {};
  if (g < groups) {
#pragma unroll 2
    for (uint32_t i = g; i < ns; i += groups) {
      const float4 *src = reinterpret_cast<const float4 *>(a.part_o + (first + i * step) * D + c);
      const float4 u = src[0], v = src[1];
      const float f = weight[i];
      y[0] += f * u.x, y[1] += f * u.y, y[2] += f * u.z, y[3] += f * u.w;
      y[4] += f * v.x, y[5] += f * v.y, y[6] += f * v.z, y[7] += f * v.w;
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[threadIdx.x * 8 + i] = y[i];
  __syncthreads();
  if (g == 0) {
    for (uint32_t w = 1; w < groups; ++w)
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] += acc[(w * per + threadIdx.x) * 8 + i];
    const uint32_t qi = row / a.group, hq = head * a.group + row - qi * a.group;
    finish_row(a, static_cast<size_t>(ps.row0) + qi, hq, c, ovec, nu, lift, sum, y);
  }
}

// Weights from stored scores: a thread takes one token of one head.  Storing
// and reading 4 bytes a row and token replaces reading the keys again.
template <class P>
__global__ void __launch_bounds__(kWeighTile) weigh_scores_kernel(const __grid_constant__ AttendArgs a,
                                                                  const __grid_constant__ P plan) {
  chain_wait();
  const PlanSeq &ps = plan.s[plan_find(plan, blockIdx.x)];
  const uint32_t t = (blockIdx.x - ps.unit0) * kWeighTile + threadIdx.x, head = blockIdx.y;
  if (t >= ps.len) return;
  const uint32_t rows = ps.count * a.group, stride = (rows + 1) & ~1u;
  const float *sc =
      a.scores + ps.aux + (static_cast<size_t>(head) * ((ps.len + kStep - 1) / kStep * kStep) + t) * stride;
  const float2 *lse = a.lse2 + static_cast<size_t>(ps.row0) * a.q_heads + head * a.group;
  float sum = 0.0f;
  for (uint32_t row = 0; row < rows; row += 2) {
    const float2 x = *reinterpret_cast<const float2 *>(sc + row);
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) {
      if (row + h >= rows) break;
      const uint32_t qi = (row + h) / a.group;
      const float y = h ? x.y : x.x;
      const float2 ref = lse[static_cast<size_t>(qi) * a.q_heads + row + h - qi * a.group];
      const float p = exp2_approx(y - ref.x - ref.y);
      sum += y == -VG_INF ? 0.0f : p;  // not seen
    }
  }
  float *w = a.kv.weights + (static_cast<size_t>(ps.seq) * a.kv.heads + head) * a.kv.stride + t;
  *w += sum;
}

template <int D, int kCols, bool kScores>
cudaError_t decode(const AttendArgs &a, const Plan &plan, cudaStream_t s) {
  constexpr int warps = Dec<kCols>::warps;
  constexpr size_t ring = warps * Dec<kCols>::ring * (2 * kStep * D + 16);
  constexpr size_t join = warps * 8 * kCols * ((D + 2) * sizeof(float) + sizeof(float4));
  constexpr size_t smem = std::max(ring, join);
  return with_plan(plan, [&](const auto &p) {
    static std::atomic<uint64_t> allowed{0};
    auto *kern = attend_decode_kernel<D, kCols, kScores, std::decay_t<decltype(p)>>;
    const cudaError_t e = allow_smem(kern, smem, allowed);
    if (e != cudaSuccess) return e;
    kern<<<dim3(p.units, a.kv.heads), warps * 32, smem, s>>>(a, p, rows_aligned(a.q, 2), rows_aligned(a.out, 2));
    return cudaGetLastError();
  });
}

template <int D>
cudaError_t decode_rows(const AttendArgs &a, const Plan &plan, uint32_t rows, cudaStream_t s) {
  if (rows <= 8) return a.scores ? decode<D, 1, true>(a, plan, s) : decode<D, 1, false>(a, plan, s);
  return a.scores ? decode<D, 2, true>(a, plan, s) : decode<D, 2, false>(a, plan, s);
}

}  // namespace

cudaError_t launch_kv_attend_decode(const AttendArgs &a, const Plan &plan, uint32_t max_rows, cudaStream_t s) {
  if (plan.units == 0) return cudaSuccess;
  switch (a.kv.dim) {
    case 32: return decode_rows<32>(a, plan, max_rows, s);
    case 64: return decode_rows<64>(a, plan, max_rows, s);
    case 96: return decode_rows<96>(a, plan, max_rows, s);
    default: return decode_rows<128>(a, plan, max_rows, s);
  }
}

cudaError_t launch_kv_attend_join(const AttendArgs &a, const Plan &plan, uint32_t part_rows, uint32_t max_rows,
                                  cudaStream_t s) {
  return with_plan(plan, [&](const auto &p) {
    return launch_chained(attend_join_kernel<std::decay_t<decltype(p)>>, dim3(max_rows, a.kv.heads, p.n), kJoinThreads,
                          0, s, a, p, part_rows, rows_aligned(a.out, 2));
  });
}

cudaError_t launch_kv_weigh_scores(const AttendArgs &a, const Plan &plan, cudaStream_t s) {
  if (plan.units == 0) return cudaSuccess;
  return with_plan(plan, [&](const auto &p) {
    return launch_chained(weigh_scores_kernel<std::decay_t<decltype(p)>>, dim3(p.units, a.kv.heads), kWeighTile, 0, s,
                          a, p);
  });
}

}  // namespace vg
