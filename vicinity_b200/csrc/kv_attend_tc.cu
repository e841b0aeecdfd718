// Attention of many queries over the 8-bit cache on the 5th-generation tensor
// cores (tcgen05), and the weights of its tokens.
//
// The rows of a key/value head are its queries times the query heads that share
// it; a tile is 128 rows (the lanes of the TMEM accumulator) by 128 tokens.
// Bound by the two products, 4 dim flops per (row, token), and as much by one
// ex2 each; the codes are read from L2 by every row block.  1,024 queries x 32
// heads x 128 over 16,384 tokens (266 GFLOP): 314 us after 9 for the query tiles,
// 0.85 PFLOP/s, tensor and exponential pipes 54 % busy.  Product and softmax of a row tile follow each
// other, two tiles take turns, and what is left is the time between a product's
// end and the start of what waits for it; a third tile has no room in TMEM.
// Their weights (133 GFLOP and the exponentials again): 210 us, the exponential
// pipe 74 % busy.  See kv_attend.cu for the scaling of scores and
// probabilities.
//
// attend_tile_kernel, one CTA per (sequence, head, kTiles row tiles, chunk of
// tokens).  Two row tiles share the converted codes and take turns: the
// products of one run while the other is in its softmax.  A sequence of one row
// tile gets a CTA of half the size, two of which share an SM instead.
//   4 warps per row tile  softmax: one row per thread, S from TMEM, P back into its place
//   4 warps               load codes, convert them to binary16 tiles in shared memory
//                         (keys as they are; values transposed: tokens are the
//                         contraction of the second product)
//   1 warp                copies the query tiles, issues S = Q K^T and O += P V
// With two row tiles the softmax warps hold their row's 128 scores in
// registers: the block is launched with 128 a thread (16 warps, three of them
// idle) and moves them to 176 for softmax, 96 for conversion and 64 for the
// rest.  Half-size CTAs read S twice instead, 32 scores at a time in loops of
// little code.
// Every wait is bounded: a protocol error sets the error flag and the kernel
// drains its copies and products, frees its TMEM and returns.
#include "chain.cuh"
#include "common.cuh"
#include "elements.cuh"
#include "f32x2.cuh"
#include "kv_attend.cuh"
#include "kv_cache.h"
#include "umma.cuh"

#include <algorithm>
#include <type_traits>

namespace vg {

namespace {

constexpr int kRows = kTileRows;              // 128
constexpr uint32_t kTok = 128;                // tokens per tile
constexpr uint32_t kKBlockBytes = kRows * 128;  // 64 binary16 columns of a 128-row tile
constexpr int kThreads = 288;                 // of the weights' kernel
constexpr uint32_t kTmemColumns = 256;        // its two accumulators

__device__ __forceinline__ uint32_t f16_idesc(uint32_t n) {  // D f32, A and B binary16 K-major, M = 128
  return (1u << 4) | ((n >> 3) << 17) | ((kRows >> 4) << 24);
}

// Matrix descriptors differ in their low word only (umma_desc of an address in
// the first 256 KB); kDescHigh is the rest.
constexpr uint32_t kDescHigh = (1024u >> 4) | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t desc_low(uint32_t saddr) { return (saddr & 0x3FFFFu) >> 4 | 1u << 16; }

__device__ __forceinline__ void umma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
      "mov.b64 da, {%1, %5};\n\t"
      "mov.b64 db, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"(kDescHigh)
      : "memory");
}

// A from TMEM: binary16 pairs, 8 columns per K-step of 16
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\t"
      "mov.b64 db, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"(kDescHigh)
      : "memory");
}

// d = a b^T over `steps` K-steps of two K-major tiles of 128-row K-blocks (low descriptor words)
__device__ __forceinline__ void umma_rows(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, int steps) {
#pragma unroll
  for (int k = 0; k < 8; k += 2) {
    if (k >= steps) break;
    const uint32_t off = (k >> 2) * (kKBlockBytes >> 4) + (k & 3) * 2;
    umma_ss(d, a + off, b + off, idesc, k != 0);
    umma_ss(d, a + off + 2, b + off + 2, idesc, 1);
  }
}

__device__ __forceinline__ void tmem_ld8_nowait(uint32_t taddr, uint32_t *v) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
               : "r"(taddr));
}

__device__ __forceinline__ void tmem_wait_ld16(uint32_t *v) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]),
                 "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15])::
                   "memory");
}

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t *v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Registers of the calling warpgroup's threads, drawn from what the block was launched with.
template <int kCount, bool kMore>
__device__ __forceinline__ void set_registers() {
  if (kMore) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kCount));
  else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kCount));
}

__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Byte of (row, 16-byte chunk c of 8 binary16 columns) in a K-major tile of 128-byte swizzled rows.
__device__ __forceinline__ uint32_t tile_byte(uint32_t rows, uint32_t row, uint32_t c) {
  return (c >> 3) * (rows * 128) + row * 128 + (((c & 7u) ^ (row & 7u)) << 4);
}

// ---- key tile: 128 tokens x D, as they lie -------------------------------------

// 16 codes each: item = (token, 16-byte chunk)
template <int D, int kWorkers>
struct KeyTile {
  static constexpr int kItems = kTok * (D / 16) / kWorkers;
  uint4 w[kItems];
  __device__ __forceinline__ void load(const int8_t *codes, uint32_t tid) {
#pragma unroll
    for (int i = 0; i < kItems; ++i) w[i] = __ldg(reinterpret_cast<const uint4 *>(codes) + tid + i * kWorkers);
  }
  __device__ __forceinline__ void store(uint8_t *tile, uint32_t tid) const {
    // where a step of kWorkers items is whole tokens, a thread's chunk stays
    constexpr bool kWhole = kWorkers % (D / 16) == 0;
    const uint32_t tok0 = tid / (D / 16), c0 = tid % (D / 16);
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const uint32_t e = tid + i * kWorkers;
      const uint32_t tok = kWhole ? tok0 : e / (D / 16), c = kWhole ? c0 : e % (D / 16);
      const uint32_t x[4] = {w[i].x ^ 0x80808080u, w[i].y ^ 0x80808080u, w[i].z ^ 0x80808080u, w[i].w ^ 0x80808080u};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        // the lanes of the second K-block store their halves in the other
        // order: eight lanes of a token meet eight different bank groups
        const uint32_t hh = (c & 4u) ? 1 - h : h;
        const uint32_t a = hh ? x[2] : x[0], b = hh ? x[3] : x[1];
        // (16 and more tokens further: a multiple of 8 rows, the same swizzle)
        uint8_t *dst = tile + tile_byte(kTok, tok, 2 * c + hh) + (kWhole ? i * (kWorkers / (D / 16)) * 128 : 0);
        *reinterpret_cast<uint4 *>(dst) =
            make_uint4(half2_of<0x4140>(a), half2_of<0x4342>(a), half2_of<0x4140>(b), half2_of<0x4342>(b));
      }
    }
  }
};

// ---- value tile: D x 128 tokens -------------------------------------------------

// Item = (8 tokens, 4 dimensions): a word of each token, transposed in
// registers.  Dimension 4 i + d is row d D/4 + i of the tile, so that
// neighbouring lanes store neighbouring rows (no bank conflicts).
template <int D>
struct ValueTile {
  static constexpr int kItems = (kTok / 8) * (D / 4) / 128;
  static constexpr bool kWhole = 128 % (D / 4) == 0;  // as for the keys
  uint32_t w[kItems][8];
  __device__ __forceinline__ void load(const int8_t *codes, uint32_t tid) {
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const uint32_t e = tid + i * 128, u = kWhole ? tid / (D / 4) : e / (D / 4), c = kWhole ? tid % (D / 4) : e % (D / 4);
      const uint32_t *p = reinterpret_cast<const uint32_t *>(codes) + u * 8 * (D / 4) + c + (kWhole ? i * 128 * 8 : 0);
#pragma unroll
      for (int k = 0; k < 8; ++k) w[i][k] = __ldg(p + k * (D / 4));
    }
  }
  __device__ __forceinline__ void store(uint8_t *tile, uint32_t tid) const {
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const uint32_t e = tid + i * 128;
      const uint32_t u = (kWhole ? tid / (D / 4) + i * (128 / (D / 4)) : e / (D / 4));
      const uint32_t c = kWhole ? tid % (D / 4) : e % (D / 4);
      uint32_t out[4][4];  // [dimension][token pair]
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t a = __byte_perm(w[i][2 * k], w[i][2 * k + 1], 0x5140) ^ 0x80808080u;
        const uint32_t b = __byte_perm(w[i][2 * k], w[i][2 * k + 1], 0x7362) ^ 0x80808080u;
        out[0][k] = half2_of<0x4140>(a);
        out[1][k] = half2_of<0x4342>(a);
        out[2][k] = half2_of<0x4140>(b);
        out[3][k] = half2_of<0x4342>(b);
      }
#pragma unroll
      for (int d = 0; d < 4; ++d)
        *reinterpret_cast<uint4 *>(tile + tile_byte(D, d * (D / 4) + c, u)) =
            make_uint4(out[d][0], out[d][1], out[d][2], out[d][3]);
    }
  }
};

// ---- query tiles -----------------------------------------------------------------

// Rows of a block of 128 as a binary16 tile, each scaled by a power of two
// into the range (and by the sign of the softmax scale), with the factor that
// turns its products with key codes times their scale into scores.
constexpr int kImageThreads = 256;

template <class P>
__global__ void __launch_bounds__(kImageThreads) query_tiles_kernel(const __grid_constant__ AttendArgs a,
                                                                    const __grid_constant__ P plan,
                                                                    const bool qvec) {
  chain_release();
  const uint32_t D = a.kv.dim, head = blockIdx.y;
  uint32_t lo = 0, hi = plan.n;  // the entry that row block blockIdx.x belongs to
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) >> 1;
    if (plan.s[mid].block0 <= blockIdx.x) lo = mid;
    else hi = mid;
  }
  const PlanSeq &ps = plan.s[lo];
  const uint32_t rows = ps.count * a.group, c = threadIdx.x & 15, sub = threadIdx.x >> 4;
  const size_t at = static_cast<size_t>(blockIdx.x) * a.kv.heads + head;
  uint8_t *tile = a.q_tiles + at * ((D + 63) / 64) * kKBlockBytes;
  float *qf = a.q_factor + at * kRows;
  const bool neg = a.scale < 0.0f;
  for (uint32_t r = sub; r < kRows; r += kImageThreads / 16) {
    const uint32_t row = (blockIdx.x - ps.block0) * kRows + r;
    float x[8] = {};
    if (row < rows && c < D / 8) {
      const uint32_t qi = row / a.group;
      load8_16(a.q.p,
               static_cast<int64_t>(ps.row0 + qi) * a.q.token +
                static_cast<int64_t>(head * a.group + row - qi * a.group) * a.q.head + c * 8,
               a.dtype == VG_F16, qvec, x);
    }
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[i]));
#pragma unroll
    for (int w = 8; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor_sync(VG_FULL_MASK, top, w));
    float s, inv;
    row_scale(top, s, inv);
    if (neg) inv = -inv;
    if (c < D / 8)
      *reinterpret_cast<uint4 *>(tile + tile_byte(kRows, r, c)) =
          make_uint4(pack_half2(x[0] * inv, x[1] * inv), pack_half2(x[2] * inv, x[3] * inv),
                     pack_half2(x[4] * inv, x[5] * inv), pack_half2(x[6] * inv, x[7] * inv));
    if (c == 0) qf[r] = row < rows ? s * fabsf(a.scale) * kLog2e : 0.0f;
  }
}

// ---- attention ---------------------------------------------------------------------

template <int D, int kTiles>
struct TileSmem {  // offsets from a 1024-byte boundary; kTiles stages of codes
  static constexpr uint32_t kQ = ((D + 63) / 64) * kKBlockBytes, kK = kQ, kV = 2 * D * 128;
  static constexpr uint32_t k = kTiles * kQ, v = k + kTiles * kK, table = v + kTiles * kV;
  static constexpr uint32_t bars = table + 2 * 8 * sizeof(float4);
  static constexpr size_t bytes = 1024 + bars + 32 * 8;
};

template <int D, int kTiles, class P>
__global__ void __launch_bounds__(kTiles == 2 ? 512 : 288, 3 - kTiles)
    attend_tile_kernel(const __grid_constant__ AttendArgs a, const __grid_constant__ P plan, const bool ovec) {
  using Smem = TileSmem<D, kTiles>;
  constexpr int kSoftWarps = 4 * kTiles, kMmaWarp = kSoftWarps + 4;
  constexpr uint32_t kColumns = 256 * kTiles;  // per row tile: S (P in its first half) and O
  extern __shared__ uint8_t tile_raw[];
  const uint32_t raw = smem_u32(tile_raw);
  uint8_t *sm = tile_raw + (((raw + 1023u) & ~1023u) - raw);  // swizzled tiles need 1024-byte alignment
  uint8_t *sQ = sm, *sK = sm + Smem::k, *sV = sm + Smem::v;
  // per 16 tokens: (key scale, log2 of the value scale, its reciprocal, whether one of them is NaN)
  float4 *table = reinterpret_cast<float4 *>(sm + Smem::table);  // [2][8]
  uint64_t *bars = reinterpret_cast<uint64_t *>(sm + Smem::bars);
  uint64_t *qfull = bars, *drain = bars + 1, *tfull = bars + 2;           // tfull[2]
  uint64_t *kfull = bars + 4, *kempty = bars + 6, *vfull = bars + 8, *vempty = bars + 10;  // [kTiles] stages
  uint64_t *sfull = bars + 12, *pvdone = bars + 14;                       // [kTiles] row tiles
  uint64_t *pfull = bars + 16;                                            // [kTiles][2] halves of a tile's tokens
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 20);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = lane_id();

  const KvView &kv = a.kv;
  const uint32_t unit = blockIdx.x, head = blockIdx.y;
  const PlanSeq &ps = plan.s[plan_find(plan, unit)];
  constexpr uint32_t kUnitRows = kRows * kTiles;
  const uint32_t rows = ps.count * a.group, ns = max(1u, (ps.len + a.chunk - 1) / a.chunk);
  const uint32_t nrb = (rows + kUnitRows - 1) / kUnitRows;
  const uint32_t rb = nrb - 1 - (unit - ps.unit0) / ns, sp = (unit - ps.unit0) % ns;  // last rows, which see most, first
  const uint32_t last = min(rows, (rb + 1) * kUnitRows) - 1;
  const uint32_t row_tiles = (last - rb * kUnitRows) / kRows + 1;  // of the unit's kTiles
  const uint32_t t0 = sp * a.chunk, t1 = min(tokens_seen(ps, last / a.group, a.causal), t0 + a.chunk);
  const uint32_t tiles = t1 > t0 ? (t1 - t0 + kTok - 1) / kTok : 0;
  const size_t r = static_cast<size_t>(ps.seq) * kv.heads + head, nb = kv.stride >> kv.block_shift;
  const size_t q_at = static_cast<size_t>(ps.block0 + rb * kTiles) * kv.heads + head;  // + heads per row tile

  if (threadIdx.x == 0) {
    mbar_init(qfull, 1);
    mbar_init(drain, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(tfull + i, 1);
      mbar_init(kfull + i, 4);
      mbar_init(kempty + i, 1);
      mbar_init(vfull + i, 4);
      mbar_init(vempty + i, 1);
      mbar_init(sfull + i, 1);
      // the warps of a row tile that have rows
      const uint32_t from = rb * kUnitRows + i * kRows, some = rows > from ? min(4u, (rows - from + 31) / 32) : 4u;
      mbar_init(pfull + 2 * i, some);
      mbar_init(pfull + 2 * i + 1, some);
      mbar_init(pvdone + i, 1);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_smem();
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(kColumns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  chain_release();  // not before this CTA has its TMEM: a successor that waits may hold some
  chain_wait();     // the query tiles
  const uint32_t tmem = *tmem_slot;  // row tile x: S at 128 x, O at 128 (kTiles + x)
  auto give_up = [&](int code) {
    *abort_flag = 1;
    if (a.error) *reinterpret_cast<volatile int *>(a.error) = code;
  };

  if (warp >= kMmaWarp) {
    // ---- query tiles and products ----
    if (kTiles == 2) set_registers<64, false>();
    if (warp == kMmaWarp && lane == 0 && tiles) {
      mbar_arrive_expect_tx(qfull, row_tiles * Smem::kQ);
      for (uint32_t x = 0; x < row_tiles; ++x)
        bulk_copy_g2s(sQ + x * Smem::kQ, a.q_tiles + (q_at + static_cast<size_t>(x) * kv.heads) * Smem::kQ, Smem::kQ,
                      qfull);
      bool ok = mbar_wait_sleep(qfull, 0);
      const uint32_t dQ = desc_low(smem_u32(sQ)), dK = desc_low(smem_u32(sK)), dV = desc_low(smem_u32(sV));
      auto scores = [&](uint32_t x, uint32_t i) {  // S of row tile x and token tile i
        const uint32_t st = i % kTiles;
        if (x == 0) {
          ok = ok && mbar_wait(kfull + st, (i / kTiles) & 1);
          if (!ok) return;
          tc_fence_after();
        }
        umma_rows(tmem + x * kTok, dQ + x * (Smem::kQ >> 4), dK + st * (Smem::kK >> 4), f16_idesc(kTok), D / 16);
        umma_commit(sfull + x);
        if (x + 1 == row_tiles) umma_commit(kempty + st);
      };
      for (uint32_t x = 0; ok && x < row_tiles; ++x) scores(x, 0);
      for (uint32_t i = 0; ok && i < tiles; ++i) {
        const uint32_t st = i % kTiles;
        for (uint32_t x = 0; ok && x < row_tiles; ++x) {
          ok = !*abort_flag && (x || mbar_wait(vfull + st, (i / kTiles) & 1));
          // Alone, a row tile's products start with the first half of P.  With
          // two, the other tile's fill that time, and one uninterrupted run of
          // eight is faster (chunks of 1,024 queries: 325 against 361 us).
          if (kTiles == 2) ok = ok && mbar_wait(pfull + 2 * x, i & 1) && mbar_wait(pfull + 2 * x + 1, i & 1);
          tc_fence_after();
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (kTiles == 1) {
              ok = ok && mbar_wait(pfull + h, i & 1);
              tc_fence_after();
            }
            if (!ok) break;
            const uint32_t b = dV + st * (Smem::kV >> 4) + h * (D * 128 >> 4);
            const uint32_t d = tmem + (kTiles + x) * kTok, p = tmem + x * kTok + h * 32;
            umma_ts(d, p, b, f16_idesc(D), (i | h) != 0);
#pragma unroll
            for (int k = 1; k < 4; ++k) umma_ts(d, p + k * 8, b + k * 2, f16_idesc(D), 1);
          }
          if (!ok) break;
          umma_commit(pvdone + x);
          if (x + 1 == row_tiles) umma_commit(vempty + st);
          // the next S takes the place of the P just used
          if (i + 1 < tiles && (ok = mbar_wait(pvdone + x, i & 1))) scores(x, i + 1);
        }
      }
      if (!ok) give_up(1);
      umma_commit(drain);  // every product issued is complete before TMEM is released
      mbar_wait(drain, 0);
    }
  } else if (warp >= kSoftWarps) {
    // ---- codes to binary16 tiles ----
    if (kTiles == 2) set_registers<96, false>();
    const uint32_t tid = threadIdx.x - kSoftWarps * 32;
    const int8_t *kc = kv.codes[0] + (r * kv.stride + t0) * D, *vc = kv.codes[1] + (r * kv.stride + t0) * D;
    const float *ks = kv.scales[0] + r * nb, *vs = kv.scales[1] + r * nb;
    KeyTile<D, 128> key;
    ValueTile<D> value;
    float2 scale = make_float2(1.0f, 1.0f);  // of group `lane` of the tile (first warp)
    auto load_keys = [&](uint32_t i) {
      key.load(kc + static_cast<size_t>(i) * kTok * D, tid);
      const uint32_t t = t0 + i * kTok + tid * 16;
      if (tid < 8 && t < ps.len) scale = make_float2(__ldg(ks + (t >> kv.block_shift)), __ldg(vs + (t >> kv.block_shift)));
    };
    if (tiles) load_keys(0);
    bool ok = true;
    for (uint32_t i = 0; i < tiles; ++i) {
      const uint32_t st = i % kTiles, before = (i / kTiles - 1) & 1;  // phase of the stage's last use
      value.load(vc + static_cast<size_t>(i) * kTok * D, tid);
      // The stage's keys have been used and, two tiles ago, the table's entries
      // (with one stage: waited for before the last tile's values).
      ok = i < kTiles || (mbar_wait_sleep(kempty + st, before) && (kTiles == 1 || mbar_wait_sleep(vempty + st, before)));
      if (!__all_sync(VG_FULL_MASK, ok)) {
        ok = false;
        break;
      }
      if (tid < 8)
        table[(i & 1) * 8 + tid] =
            make_float4(scale.x == scale.x ? scale.x : 1.0f, log2_scale(scale.y), inverse_scale(scale.y),
                        scale.x != scale.x ? 2.0f : scale.y != scale.y ? 1.0f : 0.0f);
      if (tid < 32) {
        __syncwarp();
        if (lane == 0) mbar_arrive(tfull + (i & 1));
      }
      key.store(sK + st * Smem::kK, tid);
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(kfull + st);
      if (i + 1 < tiles) load_keys(i + 1);
      if (!__all_sync(VG_FULL_MASK, i < kTiles || mbar_wait_sleep(vempty + st, before))) {
        ok = false;
        break;
      }
      value.store(sV + st * Smem::kV, tid);
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(vfull + st);
    }
    if (!ok) give_up(2);
  } else {
    // ---- softmax: thread = row = TMEM lane ----
    if (kTiles == 2) set_registers<176, true>();
    const uint32_t x = warp >> 2, wr = threadIdx.x & 127;
    const uint32_t row = rb * kUnitRows + threadIdx.x;
    const bool valid = row < rows;
    const uint32_t qi = row / a.group;
    const uint32_t lim = valid ? tokens_seen(ps, qi, a.causal) : 0xffffffffu;
    const uint32_t warp_lim = __reduce_min_sync(VG_FULL_MASK, lim);
    const uint32_t my_tiles = row - lane < rows ? tiles : 0;  // a warp without rows has nothing to do
    const float f_row = my_tiles == 0 ? 0.0f : a.q_factor[(q_at + static_cast<size_t>(x) * kv.heads) * kRows + wr];
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t pS = tmem + x * kTok + lane_base, pO = tmem + (kTiles + x) * kTok + lane_base;
    float nu = kUnseen, lift = 0.0f, l = 0.0f;
    float poison = 0.0f;  // whether the row has seen values (1) or keys (2) that read as NaN
    // products of 32 tokens from `from` on that the row does not see
    auto hide = [&](uint32_t *v, uint32_t from) {
#pragma unroll
      for (int k = 0; k < 32; ++k)
        if (from + k >= lim) v[k] = 0xff800000u;
    };
    // largest score (n) and score plus log2 of the value scale (m) of 32
    // products; the factors are above 0, so that -inf stays -inf
    auto largest = [&](const uint32_t *v, const float4 *tab, float &m, float &n) {
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const float4 e = tab[g];
        float top = -VG_INF;
#pragma unroll
        for (int k = 0; k < 16; ++k) top = fmaxf(top, __uint_as_float(v[16 * g + k]));
        const float x = __fmul_rn(top, fmaxf(f_row * e.x, 1e-37f));
        n = fmaxf(n, x);
        m = fmaxf(m, x + e.y);
      }
    };
    // Large scores: 32 products become scores less nu; over: the largest of
    // these plus log2 of the value scale
    auto subtract = [&](uint32_t *v, const float4 *tab, float &over) {
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const float4 e = tab[g];
        const float f = fmaxf(f_row * e.x, 1e-37f);
        float top = -VG_INF;
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const float x = __fmul_rn(__uint_as_float(v[16 * g + k]), f) - nu;
          v[16 * g + k] = __float_as_uint(x);
          top = fmaxf(top, x);
        }
        over = fmaxf(over, top + e.y);
      }
    };
    // whether a reference that goes to n would be large
    auto any_large = [](float n) { return __any_sync(VG_FULL_MASK, fabsf(n) > kLargeScore && n != -VG_INF); };
    // the sums of values so far shrink
    auto shrink = [&](float c) {
#pragma unroll 1
      for (int b = 0; b < D; b += 16) {
        uint32_t v[16];
        tmem_ld8_nowait(pO + b, v);
        tmem_ld8_nowait(pO + b + 8, v + 8);
        tmem_wait_ld16(v);
#pragma unroll
        for (int k = 0; k < 16; ++k) v[k] = __float_as_uint(__uint_as_float(v[k]) * c);
        tmem_st16(pO + b, v);
      }
    };
    // whether the references lag too far behind n and m
    auto lag = [&](float m, float n) { return __any_sync(VG_FULL_MASK, fmaxf(n, m - lift) > nu + kLazy); };
    // takes them there
    auto raise = [&](float m, float n, bool sums) {
      const float c = raise_references(nu, lift, n, m - n, l);
      if (sums) shrink(c);
    };
    // P of 32 tokens from `from` on, into the denominator and binary16 pairs;
    // large: v holds scores less nu
    auto powers = [&](const uint32_t *v, const float4 *tab, uint32_t from, auto large, uint32_t (&p)[16]) {
      const PowerRefs refs(large.value ? 0.0f : nu, lift);
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const float4 e = tab[g];
        const float f = large.value ? 1.0f : fmaxf(f_row * e.x, 1e-37f), ref = refs.exponent(e.y);
        const f32x2 f2 = f2_pack(f, f), ref2 = f2_pack(ref, ref);
        f32x2 sum2[2] = {0, 0};
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int j = 16 * g + 2 * k;
          float2 y = f2_unpack(f2_fma(f2_pack(__uint_as_float(v[j]), __uint_as_float(v[j + 1])), f2, ref2));
          y.x = exp2_approx(y.x);
          y.y = exp2_approx(y.y);
          sum2[k & 1] = f2_add(sum2[k & 1], f2_pack(y.x, y.y));
          p[8 * g + k] = pack_half2(y.x, y.y);
        }
        const float2 sum = f2_unpack(f2_add(sum2[0], sum2[1]));
        l = fmaf(sum.x + sum.y, refs.share(e.z), l);
        if (e.w != 0.0f && from + 16 * g < lim) poison = fmaxf(poison, e.w);
      }
    };
    auto half_done = [&](int h) {
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(pfull + 2 * x + h);
    };
    // A tile with large scores: S is read for the largest, again for what lies
    // over the new nu, and again for P.
    auto large_tile = [&](const float4 *tab, uint32_t t, bool edge, bool sums) {
      float m = -VG_INF, n = -VG_INF, low = 0.0f, over = 0.0f;
#pragma unroll 1
      for (int step = 0; step < 12; ++step) {
        const int c = step & 3;
        uint32_t v[32], p[16];
        tmem_ld32_nowait(pS + c * 32, v);
        tmem_wait_ld32(v);
        if (edge) hide(v, t + c * 32);
        if (step < 4) {
          largest(v, tab + 2 * c, m, n);
          if (step < 3) continue;
          const float was = nu;
          nu = fmaxf(nu, n);
          l *= exp2_approx(was - nu);
          low = over = lift + (was - nu);
          continue;
        }
        subtract(v, tab + 2 * c, over);
        if (step < 7) continue;
        if (step == 7) {
          lift = over;
          if (sums) shrink(exp2_approx(low - over));
          continue;
        }
        powers(v, tab + 2 * c, t + c * 32, std::true_type{}, p);
        tmem_st16(pS + c * 16, p);
        if (c & 1) half_done(c >> 1);
      }
    };
    bool ok = true, large = false;
    auto ready = [&](uint32_t i) {
      ok = __all_sync(VG_FULL_MASK, mbar_wait(tfull + (i & 1), (i >> 1) & 1) && mbar_wait(sfull + x, i & 1));
      tc_fence_after();
      return ok;
    };
    uint32_t i = 0;
    for (; i < my_tiles && ready(i); ++i) {
      const uint32_t t = t0 + i * kTok;
      const float4 *tab = table + (i & 1) * 8;
      const bool edge = t + kTok > warp_lim;
      float m = -VG_INF, n = -VG_INF;
      if constexpr (kTiles == 2) {
        uint32_t v[kTok];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32_nowait(pS + c * 32, v + c * 32);
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_wait_ld32(v + c * 32);
        if (edge) {
#pragma unroll
          for (int c = 0; c < 4; ++c) hide(v + c * 32, t + c * 32);
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) largest(v + c * 32, tab + 2 * c, m, n);
        if (lag(m, n)) {
          if ((large = any_large(n))) break;
          raise(m, n, i != 0);
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t p[16];
          powers(v + c * 32, tab + 2 * c, t + c * 32, std::false_type{}, p);
          tmem_st16(pS + c * 16, p);
          if (c & 1) half_done(c >> 1);
        }
      } else {
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t v[32];
          tmem_ld32_nowait(pS + c * 32, v);
          tmem_wait_ld32(v);
          if (edge) hide(v, t + c * 32);
          largest(v, tab + 2 * c, m, n);
        }
        if (lag(m, n)) {
          if ((large = any_large(n))) break;
          raise(m, n, i != 0);
        }
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t v[32], p[16];
          tmem_ld32_nowait(pS + c * 32, v);
          tmem_wait_ld32(v);
          if (edge) hide(v, t + c * 32);
          powers(v, tab + 2 * c, t + c * 32, std::false_type{}, p);
          tmem_st16(pS + c * 16, p);  // over S of tokens that have been read
          if (c & 1) half_done(c >> 1);
        }
      }
    }
    // From the first tile on that would take a reference there.  (A loop of its
    // own: as a branch of the one above, its code alone takes 1,024 queries over
    // 16,384 tokens from 314 to 336 us.)
    for (; large && i < my_tiles && ready(i); ++i)
      large_tile(table + (i & 1) * 8, t0 + i * kTok, t0 + (i + 1) * kTok > warp_lim, i != 0);
    if (ok && my_tiles) {
      ok = __all_sync(VG_FULL_MASK, mbar_wait_sleep(pvdone + x, (my_tiles - 1) & 1));
      tc_fence_after();
    }
    if (ok) {
      const bool whole = ps.len <= a.chunk;
      const float nan = __int_as_float(0x7fffffff);
      if (poison == 2.0f) l = nan;
      const size_t at = (static_cast<size_t>(unit) * kv.heads + head) * kUnitRows + threadIdx.x;
#pragma unroll 1
      for (int b = 0; b < D / 4; b += 8) {  // dimensions 4 b .. 4 b + 31
        uint32_t v[32] = {};
        if (my_tiles) {
#pragma unroll
          for (int d = 0; d < 4; ++d) tmem_ld8_nowait(pO + d * (D / 4) + b, v + 8 * d);
          tmem_wait_ld32(v);
        }
        if (!valid) continue;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float y[8];
#pragma unroll
          for (int d = 0; d < 8; ++d) y[d] = poison != 0.0f ? nan : __uint_as_float(v[8 * (d & 3) + 2 * k + (d >> 2)]);
          const uint32_t c = 4 * b + 8 * k;
          if (whole) {
            finish_row(a, static_cast<size_t>(ps.row0) + qi, head * a.group + row - qi * a.group, c, ovec, nu, lift,
                       l, y);
          } else {
            float4 *dst = reinterpret_cast<float4 *>(a.part_o + at * D + c);
            dst[0] = make_float4(y[0], y[1], y[2], y[3]);
            dst[1] = make_float4(y[4], y[5], y[6], y[7]);
          }
        }
      }
      if (!whole && valid) a.part_ml[at] = make_float4(nu, lift, l, 0.0f);
    } else {
      give_up(3);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kColumns) : "memory");
  }
}

// ---- weights -------------------------------------------------------------------------

// One CTA per (sequence, head, 128 tokens): the scores of every row block
// again, transposed (tokens in the lanes), and the sum of a token's
// probabilities 2^(x - lse) in a register.
//   warps 0..7  convert the key tile, then, alternating row blocks, one token
//               per thread
//   warp 8      copies query tiles (two in flight), issues K Q^T
template <int D>
constexpr size_t weigh_smem() {
  return 1024 + 3 * ((D + 63) / 64) * kKBlockBytes + 2 * kRows * (8 + 8 + 4) + kTok * 4 + 8 * 4 + 128;
}

template <int D, class P>
__global__ void __launch_bounds__(kThreads, 2) weigh_tile_kernel(const __grid_constant__ AttendArgs a,
                                                                 const __grid_constant__ P plan) {
  extern __shared__ uint8_t weigh_raw[];
  const uint32_t raw = smem_u32(weigh_raw);
  uint8_t *sm = weigh_raw + (((raw + 1023u) & ~1023u) - raw);
  constexpr uint32_t kQBytes = ((D + 63) / 64) * kKBlockBytes;
  uint8_t *sK = sm, *sQ = sm + kQBytes;  // two query tiles
  float4 *row_f = reinterpret_cast<float4 *>(sQ + 2 * kQBytes);      // [2][64] (factor, factor, -lse, -lse) of a row pair
  float4 *row_ref = row_f + 2 * 64;  // [2][64] lse of a row pair: (score, score, rest, rest)
  uint32_t *row_lim = reinterpret_cast<uint32_t *>(row_ref + 2 * 64);  // [2][128]
  float *half = reinterpret_cast<float *>(row_lim + 2 * kRows);      // [128]
  int *row_large = reinterpret_cast<int *>(half + kTok);             // [2][4] whether 32 rows have large scores
  uint64_t *bars = reinterpret_cast<uint64_t *>(row_large + 8);
  uint64_t *kfull = bars, *qfull = bars + 1, *qempty = bars + 3, *sfull = bars + 5, *sempty = bars + 7, *drain = bars + 9;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 10);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = lane_id();

  const KvView &kv = a.kv;
  const uint32_t unit = blockIdx.x, head = blockIdx.y;
  const PlanSeq &ps = plan.s[plan_find(plan, unit)];
  const uint32_t t0 = (unit - ps.unit0) * kTok;
  const uint32_t rows = ps.count * a.group, nrb = (rows + kRows - 1) / kRows;
  // rows of block b, in whole groups of 32: the columns of its products
  auto columns = [&](uint32_t b) { return min(static_cast<uint32_t>(kRows), (rows - b * kRows + 31) / 32 * 32); };
  const size_t r = static_cast<size_t>(ps.seq) * kv.heads + head;
  // the first row block with a row that sees the tile's first token
  uint32_t rb0 = 0;
  if (a.causal && ps.len > t0) {
    const uint32_t after = ps.len - 1 - t0;                    // query qi sees t0 if count - 1 - qi <= after
    if (ps.count - 1 > after) rb0 = (ps.count - 1 - after) * a.group / kRows;
  }

  if (threadIdx.x == 0) {
    mbar_init(kfull, 8);
    for (int i = 0; i < 2; ++i) {
      mbar_init(qfull + i, 1);
      mbar_init(qempty + i, 1);
      mbar_init(sfull + i, 1);
      mbar_init(sempty + i, 4);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_smem();
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(kTmemColumns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  auto give_up = [&](int code) {
    *abort_flag = 1;
    if (a.error) *reinterpret_cast<volatile int *>(a.error) = code;
  };
  chain_wait();  // the query tiles and what the attention left of its rows

  if (warp == 8) {
    if (lane == 0) {
      const uint32_t dK = desc_low(smem_u32(sK)), dQ = desc_low(smem_u32(sQ));
      const uint32_t n = nrb - rb0;
      auto copy = [&](uint32_t i) {  // row block rb0 + i into stage i & 1
        const size_t at = static_cast<size_t>(ps.block0 + rb0 + i) * kv.heads + head;
        mbar_arrive_expect_tx(qfull + (i & 1), kQBytes);
        bulk_copy_g2s(sQ + (i & 1) * kQBytes, a.q_tiles + at * kQBytes, kQBytes, qfull + (i & 1));
      };
      uint32_t copied = 0;
      for (; copied < min(n, 2u); ++copied) copy(copied);
      bool ok = mbar_wait_sleep(kfull, 0);
      uint32_t i = 0;
      for (; ok && i < n; ++i) {
        const uint32_t st = i & 1, ph = (i >> 1) & 1;
        if (*abort_flag || !mbar_wait_sleep(qfull + st, ph) || (i >= 2 && !mbar_wait_sleep(sempty + st, ph ^ 1))) {
          ok = false;
          break;
        }
        tc_fence_after();
        umma_rows(tmem + st * kRows, dK, dQ + st * (kQBytes >> 4), f16_idesc(columns(rb0 + i)), D / 16);
        umma_commit(qempty + st);
        umma_commit(sfull + st);
        if (i + 2 < n) {
          if (!mbar_wait_sleep(qempty + st, ph)) {
            ok = false;
            break;
          }
          copy(copied++);
        }
      }
      if (!ok) {
        give_up(4);
        // copies still in flight land in shared memory: wait for them (bounded)
        for (uint32_t c = copied > 2 ? copied - 2 : 0; c < copied; ++c) mbar_wait(qfull + (c & 1), (c >> 1) & 1);
      }
      umma_commit(drain);
      mbar_wait(drain, 0);
    }
  } else {
    {
      KeyTile<D, 256> key;
      key.load(kv.codes[0] + (r * kv.stride + t0) * D, threadIdx.x);
      key.store(sK, threadIdx.x);
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(kfull);
    }
    const int eg = warp >> 2, wl = threadIdx.x & 127;  // row blocks of this parity; token = TMEM lane
    const uint32_t t = t0 + wl;
    const uint32_t pS = tmem + eg * kRows + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const float ks = t < ps.len ? kv.scales[0][r * (kv.stride >> kv.block_shift) + (t >> kv.block_shift)] : 0.0f;
    const f32x2 ks2 = f2_pack(ks, ks);
    float *my_f = reinterpret_cast<float *>(row_f + eg * 64), *my_ref = reinterpret_cast<float *>(row_ref + eg * 64);
    uint32_t *my_lim = row_lim + eg * kRows;
    float total = 0.0f;
    bool ok = true;
    for (uint32_t i = eg; i < nrb - rb0; i += 2) {
      const uint32_t b = rb0 + i;
      {
        const uint32_t row = b * kRows + wl, qi = row / a.group;
        float2 lse = make_float2(0.0f, VG_INF);  // rows past the end, or that see nothing: probability 0
        uint32_t lim = 0;
        if (row < rows) {
          lim = tokens_seen(ps, qi, a.causal);
          lse = a.lse2[(static_cast<size_t>(ps.row0) + qi) * a.q_heads + head * a.group + row - qi * a.group];
        }
        const float f = a.q_factor[(static_cast<size_t>(ps.block0 + b) * kv.heads + head) * kRows + wl];
        const bool large = __any_sync(VG_FULL_MASK, fabsf(lse.x) > kLargeScore);
        named_sync(1 + eg, 128);  // the previous block's have been read
        my_f[(wl >> 1) * 4 + (wl & 1)] = f;
        my_f[(wl >> 1) * 4 + 2 + (wl & 1)] = -(lse.x + lse.y);
        my_ref[(wl >> 1) * 4 + (wl & 1)] = lse.x;
        my_ref[(wl >> 1) * 4 + 2 + (wl & 1)] = lse.y;
        if (lane == 0) row_large[eg * 4 + (wl >> 5)] = large;
        my_lim[wl] = lim;
        named_sync(1 + eg, 128);
      }
      // rows are in the order of their queries: the first one sees least
      const bool edge = my_lim[0] < t0 + kTok;
      const int4 any = *reinterpret_cast<const int4 *>(row_large + eg * 4);
      const bool large = any.x | any.y | any.z | any.w;
      // after a wait that gave up the loop goes on, without waits, to keep the barriers in step
      if (ok) ok = __all_sync(VG_FULL_MASK, mbar_wait_sleep(sfull + eg, (i >> 1) & 1));
      tc_fence_after();
      f32x2 sum2 = 0;
      const int groups = static_cast<int>(columns(b)) / 32;
#pragma unroll 1
      for (int c = 0; c < groups; ++c) {
        uint32_t v[32];
        tmem_ld32_nowait(pS + c * 32, v);
        tmem_wait_ld32(v);
        if (c + 1 == groups) {  // in registers: the accumulator is free
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(sempty + eg);
        }
        auto add = [&](int k, float2 p) {  // of rows 2 k and 2 k + 1: powers, where they are seen
          p.x = exp2_approx(p.x);
          p.y = exp2_approx(p.y);
          if (edge) {
            if (t >= my_lim[c * 32 + 2 * k]) p.x = 0.0f;
            if (t >= my_lim[c * 32 + 2 * k + 1]) p.y = 0.0f;
          }
          sum2 = f2_add(sum2, f2_pack(p.x, p.y));
        };
        if (large) {
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            const float4 w = reinterpret_cast<const float4 *>(my_f)[c * 16 + k];
            const float4 ref = reinterpret_cast<const float4 *>(my_ref)[c * 16 + k];
            const f32x2 x = f2_mul(f2_pack(__uint_as_float(v[2 * k]), __uint_as_float(v[2 * k + 1])),
                                   f2_mul(f2_pack(w.x, w.y), ks2));
            float2 p = f2_unpack(f2_sub(f2_sub(x, f2_pack(ref.x, ref.y)), f2_pack(ref.z, ref.w)));
            // the product's sum may differ from the attention's in its last bit: not above 1 (and NaN stays)
            p.x = p.x > 0.0f ? 0.0f : p.x;
            p.y = p.y > 0.0f ? 0.0f : p.y;
            add(k, p);
          }
          continue;
        }
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const float4 w = reinterpret_cast<const float4 *>(my_f)[c * 16 + k];
          // the factors first: a product times the largest scales passes f32
          const f32x2 f = f2_mul(f2_pack(w.x, w.y), ks2);
          add(k, f2_unpack(f2_fma(f2_pack(__uint_as_float(v[2 * k]), __uint_as_float(v[2 * k + 1])), f,
                                  f2_pack(w.z, w.w))));
        }
      }
      const float2 sum = f2_unpack(sum2);
      total += sum.x + sum.y;
    }
    if (!ok) give_up(5);
    if (eg) half[wl] = total;
    named_sync(3, 256);
    if (!eg && t < ps.len) kv.weights[r * kv.stride + t] += total + half[wl];
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemColumns) : "memory");
  }
}

// ---- launches ---------------------------------------------------------------------------

// Shared memory that lets at most two CTAs be on an SM, where each holds half of its TMEM.
constexpr size_t kTwoPerSm = 80 * 1024;

template <int D, int kTiles>
cudaError_t tile(const AttendArgs &a, const Plan &plan, cudaStream_t s) {
  const size_t smem = std::max(TileSmem<D, kTiles>::bytes, kTiles == 1 ? kTwoPerSm : size_t(0));
  return with_plan(plan, [&](const auto &p) {
    static std::atomic<uint64_t> allowed{0};
    auto *kern = attend_tile_kernel<D, kTiles, std::decay_t<decltype(p)>>;
    const cudaError_t e = allow_smem(kern, smem, allowed);
    if (e != cudaSuccess) return e;
    return launch_chained(kern, dim3(p.units, a.kv.heads), kTiles == 2 ? 512 : 288, smem, s, a, p,
                          rows_aligned(a.out, 2));
  });
}

template <int D>
cudaError_t weigh(const AttendArgs &a, const Plan &plan, cudaStream_t s) {
  const size_t smem = std::max(weigh_smem<D>(), kTwoPerSm);
  return with_plan(plan, [&](const auto &p) {
    static std::atomic<uint64_t> allowed{0};
    auto *kern = weigh_tile_kernel<D, std::decay_t<decltype(p)>>;
    const cudaError_t e = allow_smem(kern, smem, allowed);
    if (e != cudaSuccess) return e;
    return launch_chained(kern, dim3(p.units, a.kv.heads), kThreads, smem, s, a, p);
  });
}

}  // namespace

size_t query_tile_bytes(uint32_t dim) { return ((dim + 63) / 64) * kKBlockBytes; }

cudaError_t launch_kv_query_tiles(const AttendArgs &a, const Plan &plan, uint32_t blocks, cudaStream_t s) {
  return with_plan(plan, [&](const auto &p) {
    query_tiles_kernel<<<dim3(blocks, a.kv.heads), kImageThreads, 0, s>>>(a, p, rows_aligned(a.q, 2));
    return cudaGetLastError();
  });
}

cudaError_t launch_kv_attend_tiles(const AttendArgs &a, const Plan &plan, uint32_t tiles, cudaStream_t s) {
  if (plan.units == 0) return cudaSuccess;
  switch (a.kv.dim) {
    case 32: return tiles == 1 ? tile<32, 1>(a, plan, s) : tile<32, 2>(a, plan, s);
    case 64: return tiles == 1 ? tile<64, 1>(a, plan, s) : tile<64, 2>(a, plan, s);
    case 96: return tiles == 1 ? tile<96, 1>(a, plan, s) : tile<96, 2>(a, plan, s);
    default: return tiles == 1 ? tile<128, 1>(a, plan, s) : tile<128, 2>(a, plan, s);
  }
}

cudaError_t launch_kv_weigh_tiles(const AttendArgs &a, const Plan &plan, cudaStream_t s) {
  if (plan.units == 0) return cudaSuccess;
  switch (a.kv.dim) {
    case 32: return weigh<32>(a, plan, s);
    case 64: return weigh<64>(a, plan, s);
    case 96: return weigh<96>(a, plan, s);
    default: return weigh<128>(a, plan, s);
  }
}

}  // namespace vg
