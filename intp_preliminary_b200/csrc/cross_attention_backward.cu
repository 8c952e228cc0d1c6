// cross_attention_backward.cu - cross attention gradients on tcgen05 (sm_100a, bf16 / f16).
//
//   P = exp(scale q k^T - lse),  dS = P (dO v^T - delta),  delta = rowsum(dO out)
//   dq = scale dS k,   dk = scale sum_heads dS^T q,   dv = sum_heads P^T dO
//
// Nothing of size M x N is written: two kernels recompute the score tiles.
//   xattn_stats_kernel   lse in log2 units and delta of every query row, rows padded
//                        to whole tiles so that a tile's values are one bulk copy.
//   dq kernel            an item owns 128 query rows of a head and streams 64-key tiles:
//                        X = q k^T and Y = dO v^T into TMEM, dS (16-bit) back over X,
//                        dq += dS k with dS read from TMEM.
//   dk / dv kernel       an item owns 128 keys of a key head and streams 64-query tiles of
//                        all its query heads: X = k q^T, Y = v dO^T, P^T over X and dS^T
//                        over Y, dv += P^T dO and dk += dS^T q.  Grouped heads are summed
//                        in the accumulators, in a fixed order.
// Where one side has too few tiles for the GPU, the streamed axis is split and fp32 parts
// are summed in order (xattn_sum_kernel).  Every output element has one writer
// and no atomics are used, so results repeat bit for bit.
//
// A CTA (persistent over work items) has an MMA warp, a TMA warp and 8 row warps (row thread t
// owns TMEM lane t % 128 and 32 of a tile's 64 columns).  Score buffers are double: the products
// of tile t + 1 run under the row threads' tile t, and the next item's first score product runs
// under this one's epilogue.  A 128 x 64 x 16 product reads 6 KB of shared memory where both
// operands lie there (48 cycles) and 2 KB with the owned operand in TMEM (32 cycles, the
// tensor core's own pace), so the owned rows go to TMEM where it has room: dq, and dk / dv at
// head_dim <= 64 (two accumulators of 128 columns fill it otherwise).
// Recomputing the scores in both kernels costs 7 matrix products where 5 would do; in exchange
// dq needs no cross-CTA sum (fp32 atomics in an order that changes results, or a key-length
// workspace).
// P and dS are rounded to 16 bits as the tensor core's operands; all sums are fp32.  f16 has
// full precision for 30 powers of two only, and P is about 1 / N, so there both are held times
// an exact power of two that the accumulator's store takes out again: P times 2^12, dS times a
// power that brings a bound of it to 2^15 (|dS_ij| <= P (|dO_i| |v_j| + |delta_i|), vectors'
// lengths), one per query row in dq (free: it joins the exponent of P), one per key and item in
// dk / dv (a multiplication a pair).  A state that is hardly read, with a value R times as long as
// the others', takes log2(R) of those bits from dq's other states and none from dk's.  The bound's
// parts come from the statistics kernel, which reads V once for it.  That and the multiplication
// cost f16 5 to 7 % (B4 H16 M2048 N4096: D128 755 to 765 -> 793 to 815 us, D64 514 to 528 -> 543 to
// 578).  delta uses the rounded result, the only one a forward gives: nothing beside the rounding
// of dS over many states (dq 0.0024 for 0.0017 in bf16), a little over few (0.0025 at 50).
#include <cuda.h>
#include <cstdint>
#include "sla_tc_common.cuh"
#include "xattn_common.cuh"
#include "xattn_internal.h"

namespace intp {
namespace {

constexpr int kRows = 128;                 // TMEM lanes: query rows (dq) / keys (dk, dv)
constexpr int kCols = 64;                  // streamed tile: keys (dq) / query rows (dk, dv)
// Columns of a tile per row thread.  8 warps of 32 columns: 716 us for the backward of B4 H16
// M2048 N4096 D128; 16 warps of 16 columns execute a third more instructions: 735 us (one box, in
// turn; the backward takes 726 to 751 us on others).
constexpr int kW = 32;
constexpr int kParts = kCols / kW;         // row threads of a row
constexpr int kRowThreads = kRows * kParts;
constexpr int kRowWarps = kRowThreads / 32;
// The MMA and TMA warps come first, with two idle ones, so that row warp w reaches TMEM lanes 32 (w % 4) ..
constexpr int kMmaWarp = 0, kLoadWarp = 1, kFirstRowWarp = 4;
constexpr int kThreads = kFirstRowWarp * 32 + kRowThreads;
constexpr int kStages = 4;
constexpr uint32_t kTmemCols = 512, kColAcc = 256;
constexpr float kLog2e = 1.4426950408889634f;
// f16: P is held as 2^12 P.  P is at most 1, but for what the scores' own rounding between the
// forward and here makes of it (a score of 2^24 is an even number): 2^16 P may not be reached.
constexpr int32_t kPowP = 12;

// f16: the power of two that brings a bound of |dS| / P to [2^14, 2^15): P up to 2 does not
// overflow, and where it is past 1 by rounding it is the row's only one, whose dP - delta is near
// zero.  0 for no bound (zero, or not finite: then the gradients are not either).
__device__ __forceinline__ int32_t power_for(float bound) {
  const int32_t e = static_cast<int32_t>(__float_as_uint(bound) >> 23) - 127;
  return e == 128 || e == -127 ? 0 : 14 - e;
}
__device__ __forceinline__ float two_to(int32_t e) { return __int_as_float((e + 127) << 23); }
// Of numbers that are not negative; NaN counts as the largest.
__device__ __forceinline__ float max_of(float a, float b) { return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b))); }
__device__ __forceinline__ float warp_max(float v) { return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v))); }

// DP: head_dim rounded up to 64 or 128.  KV: the dk / dv kernel.
template <int DP, bool KV>
struct Shape {
  static constexpr bool kOwnedInTmem = !KV || DP == 64;
  static constexpr int kBlocks = DP / 64;
  static constexpr uint32_t kOwnedBlock = kRows * 128, kRingBlock = kCols * 128;
  static constexpr uint32_t kOwned = kBlocks * kOwnedBlock;   // one owned operand
  static constexpr uint32_t kRing = kBlocks * kRingBlock;     // one streamed operand
  static constexpr uint32_t kStats = 2 * kCols * 4;           // -lse, -delta of 64 query rows
  static constexpr uint32_t ring = kOwnedInTmem ? 0 : 2 * kOwned;
  static constexpr uint32_t stats = ring + kStages * 2 * kRing;
  static constexpr uint32_t bars = stats + kStages * kStats;
  static constexpr uint32_t kColOwned = kColAcc + (KV ? 2 : 1) * DP;   // TMEM: two operands of DP / 2 columns
};

struct alignas(8) Bars {
  uint64_t owned_full, owned_empty;        // the item's own operands
  uint64_t ring_full[kStages], ring_empty[kStages];
  uint64_t clean[kStages];                 // padded key rows of the K tile in a stage zeroed (dq)
  uint64_t s_full[2], ready[2];
  uint64_t acc_full, drain;
  uint32_t tmem_base;
  int32_t abort;
};

struct Args {
  XaBwdParams p;
  MapOrder of0, of1, or0, or1;
  float* stats;                            // [B * H][m_pad / 64][-lse 64 | -delta 64], lse in log2 units
  int32_t m_tiles64;                       // 64-row tiles of a head's queries
  int32_t n_row_tiles, n_split, split_tiles, n_items;
  int32_t k_steps;
  bool wide;                               // gradient rows are 32-byte aligned
  // The kernel before this one writes the statistics.  False for dk / dv after dq, which then reads
  // them without a wait of its own: it starts only once every dq CTA has called allow_next_kernel
  // (or left), dq's threads call that after wait_previous_kernel and a fence, and that wait returns
  // when the statistics' kernel has ended and its writes are in device memory.  The copies (bulk,
  // through L2) see no cache line from before, and the kernel still waits for dq before its end.
  bool after_stats;
};

// One work item: what it owns and what it streams.
struct Work {
  int32_t b, g, h0;          // sequence, key head, first query head (dq: the head itself)
  int32_t row0, own;         // first owned row, owned rows
  int32_t t0, n_t;           // streamed tiles [t0, t0 + n_t)
  int32_t length, split;
};

template <bool KV>
__device__ __forceinline__ Work decode_work(const Args& a, int32_t item) {
  const XaParams& p = a.p.f;
  Work w;
  const int32_t rest = item / a.n_row_tiles;
  w.row0 = (item - rest * a.n_row_tiles) * kRows;
  const int32_t outer = rest / a.n_split, heads = KV ? p.groups : p.heads;
  w.split = rest - outer * a.n_split;
  w.b = outer / heads;
  const int32_t head = outer - w.b * heads;
  w.g = KV ? head : head / p.per_group;
  w.h0 = KV ? head * p.per_group : head;
  w.length = xa_length(p, w.b);
  w.t0 = w.split * a.split_tiles;
  const int32_t extent = KV ? p.states : p.queries;
  w.own = extent - w.row0 < kRows ? extent - w.row0 : kRows;
  const int32_t total = KV ? (w.row0 < w.length ? p.per_group * a.m_tiles64 : 0) : (w.length + kCols - 1) / kCols;
  const int32_t left = total - w.t0;
  w.n_t = left < 0 ? 0 : (left < a.split_tiles ? left : a.split_tiles);
  return w;
}

// ============================================================================ row statistics
// A block takes 64 rows of one head, D / 8 lanes (rounded to a power of two) a row, every
// lane's loads in flight at once.  Rows past M, and rows without states, get -lse = -inf:
// their P is zero.  In f16 it also takes what bounds dS: |dO| of each row, the largest of it and
// of |delta| in the block, and, in blocks behind the rows', |v| of each of 64 states and the largest.

// |v| of 64 states (zero for one that is not visible) and the largest of them.
template <int LPR>
__device__ __forceinline__ void state_norms(const XaBwdParams& bp, int32_t index) {
  constexpr int kPerPass = 256 / LPR, kPasses = kCols / kPerPass;
  __shared__ float warp_top[8];
  const XaParams& p = bp.f;
  const int32_t tiles = (p.states + kCols - 1) / kCols;
  const int32_t bg = index / tiles, n0 = (index - bg * tiles) * kCols;
  const int32_t b = bg / p.groups, g = bg - b * p.groups, length = xa_length(p, b);
  const int sub = threadIdx.x % LPR, r0 = threadIdx.x / LPR;
  const uint16_t* v = static_cast<const uint16_t*>(p.v) + b * p.vs[0] + g * p.vs[1] + sub * 8;
  uint4 x[kPasses];
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int32_t n = n0 + r0 + i * kPerPass;
    x[i] = n < length && sub * 8 < p.head_dim ? __ldg(reinterpret_cast<const uint4*>(v + n * p.vs[2]))
                                              : make_uint4(0u, 0u, 0u, 0u);
  }
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const uint32_t xs[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
    float2 sum = make_float2(0.f, 0.f);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 f = unpack2<false>(xs[e]);
      sum = fma2(f, f, sum);
    }
    float square = sum.x + sum.y;
#pragma unroll
    for (int s = LPR / 2; s > 0; s >>= 1) square += __shfl_xor_sync(0xffffffffu, square, s);
    const float norm = sqrtf(square);
    const int32_t n = n0 + r0 + i * kPerPass;
    if (sub == 0 && n < p.states) bp.v_norm[static_cast<int64_t>(bg) * p.states + n] = norm;
    top = max_of(top, norm);
  }
  top = warp_max(top);
  if ((threadIdx.x & 31) == 0) warp_top[threadIdx.x >> 5] = top;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 8; ++i) top = max_of(top, warp_top[i]);
    bp.v_max[index] = top;
  }
}

template <int LPR, bool BF16>
__global__ void __launch_bounds__(256)
xattn_stats_kernel(const XaBwdParams bp, float* stats, int32_t m_tiles64) {
  constexpr int kPerPass = 256 / LPR, kPasses = kCols / kPerPass;
  __shared__ float row_max[2][kCols];      // f16: |dO| and |delta| of the block's rows
  allow_next_kernel();
  const XaParams& p = bp.f;
  const int32_t row_blocks = p.batch * p.heads * m_tiles64;
  if (!BF16 && blockIdx.x >= row_blocks) {
    state_norms<LPR>(bp, blockIdx.x - row_blocks);
    return;
  }
  const int32_t bh = blockIdx.x / m_tiles64, m0 = (blockIdx.x - bh * m_tiles64) * kCols;
  const int32_t b = bh / p.heads, h = bh - b * p.heads;
  const int sub = threadIdx.x % LPR, r0 = threadIdx.x / LPR;
  const uint16_t* o = static_cast<const uint16_t*>(p.out) + b * p.os[0] + h * p.os[1] + sub * 8;
  const uint16_t* d = static_cast<const uint16_t*>(bp.dout) + b * bp.ds[0] + h * bp.ds[1] + sub * 8;
  uint4 x[kPasses], y[kPasses];
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int32_t m = m0 + r0 + i * kPerPass;
    const bool in = m < p.queries && sub * 8 < p.head_dim;
    x[i] = in ? __ldg(reinterpret_cast<const uint4*>(o + m * p.os[2])) : make_uint4(0u, 0u, 0u, 0u);
    y[i] = in ? __ldg(reinterpret_cast<const uint4*>(d + m * bp.ds[2])) : make_uint4(0u, 0u, 0u, 0u);
  }
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const uint32_t xs[4] = {x[i].x, x[i].y, x[i].z, x[i].w}, ys[4] = {y[i].x, y[i].y, y[i].z, y[i].w};
    float2 sum = make_float2(0.f, 0.f), squares = make_float2(0.f, 0.f);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 go = unpack2<BF16>(ys[e]);
      sum = fma2(unpack2<BF16>(xs[e]), go, sum);
      if (!BF16) squares = fma2(go, go, squares);
    }
    float delta = sum.x + sum.y, square = squares.x + squares.y;
#pragma unroll
    for (int s = LPR / 2; s > 0; s >>= 1) {
      delta += __shfl_xor_sync(0xffffffffu, delta, s);
      if (!BF16) square += __shfl_xor_sync(0xffffffffu, square, s);
    }
    if (sub == 0) {
      const int32_t r = r0 + i * kPerPass, m = m0 + r;
      const float l = m < p.queries ? p.lse[static_cast<int64_t>(bh) * p.queries + m] : -INFINITY;
      float* dst = stats + static_cast<int64_t>(blockIdx.x) * (2 * kCols) + r;
      dst[0] = l == -INFINITY ? -INFINITY : BF16 ? -l * kLog2e : fmaf(-l, kLog2e, static_cast<float>(kPowP));
      dst[kCols] = -delta;
      if (!BF16) {
        const float norm = sqrtf(square);
        bp.row_norm[static_cast<int64_t>(blockIdx.x) * kCols + r] = norm;
        row_max[0][r] = norm;
        row_max[1][r] = fabsf(delta);
      }
    }
  }
  if (!BF16) {
    __syncthreads();
    if (threadIdx.x < 64) {
      const int which = threadIdx.x >> 5, lane = threadIdx.x & 31;
      const float top = warp_max(max_of(row_max[which][lane], row_max[which][lane + 32]));
      if (lane == 0) bp.tile_max[static_cast<int64_t>(blockIdx.x) * 2 + which] = top;
    }
  }
}

// ============================================================================ roles
__device__ __forceinline__ void init_bars(Bars* bars, uint32_t owned_arrivals) {
  mbar_init(&bars->owned_full, owned_arrivals);
  mbar_init(&bars->owned_empty, 1);
  for (int s = 0; s < kStages; ++s) {
    mbar_init(&bars->ring_full[s], 1);
    mbar_init(&bars->ring_empty[s], 1);
    mbar_init(&bars->clean[s], 1);
  }
  for (int s = 0; s < 2; ++s) {
    mbar_init(&bars->s_full[s], 1);
    mbar_init(&bars->ready[s], kRowWarps);
  }
  mbar_init(&bars->acc_full, 1);
  mbar_init(&bars->drain, 1);
  bars->abort = 0;
  mbar_fence_init();
}

__device__ __forceinline__ void tma_rows(uint8_t* dst, const CUtensorMap* tm, uint64_t* bar, const MapOrder& o, int x,
                                         int32_t row, int32_t head, int32_t b) {
  tma_load_4d(dst, tm, bar, x, map_coord(o, 1, row, head, b), map_coord(o, 2, row, head, b),
              map_coord(o, 3, row, head, b));
}

// TMEM column of the 16-bit operand of depth step kk: each row thread packs its kW columns into
// the first half of them.
__device__ __forceinline__ constexpr uint32_t operand_col(int kk) {
  return static_cast<uint32_t>(kk * 16 / kW * kW + kk * 16 % kW / 2);
}

// dq: a padded key tile of a sequence (rows past the tensor's end arrive as zeros by themselves).
__device__ __forceinline__ bool needs_cleaning(const XaParams& p, const Work& w, int32_t i) {
  return w.length < p.states && w.length - (w.t0 + i) * kCols < kCols;
}

// Streamed tile t of an item: key tile t (dq), or query tile t % m_tiles64 of query head h0 + t / m_tiles64.
template <int DP, bool KV>
__device__ __forceinline__ void load_role(const CUtensorMap* f0, const CUtensorMap* f1, const CUtensorMap* r0,
                                          const CUtensorMap* r1, const Args& a, Bars* bars, uint8_t* smem, int lane) {
  using L = Shape<DP, KV>;
  const XaParams& p = a.p.f;
  volatile int32_t* abort_flag = &bars->abort;
  auto wait = [&](uint64_t* bar, uint32_t phase) -> bool {
    return warp_wait(bar, phase, abort_flag, p.status, kDevTimeoutProducer, p.wait_ns);
  };
  if (lane == 0) {
    if (!L::kOwnedInTmem) {
      tma_prefetch_desc(f0);
      tma_prefetch_desc(f1);
    }
    tma_prefetch_desc(r0);
    tma_prefetch_desc(r1);
  }
  uint32_t tile = 0, items = 0;            // loaded by this CTA
  bool ok = true;
  if (KV && a.after_stats) wait_previous_kernel();
  for (int32_t item = blockIdx.x; item < a.n_items && ok; item += gridDim.x) {
    const Work wk = decode_work<KV>(a, item);
    if (wk.n_t == 0) continue;
    if (!L::kOwnedInTmem) {
      if (items > 0 && !wait(&bars->owned_empty, items - 1)) break;
      if (lane == 0) {
        mbar_arrive_expect_tx(&bars->owned_full, 2 * L::kOwned);
#pragma unroll
        for (int blk = 0; blk < L::kBlocks; ++blk) {
          tma_rows(smem + blk * L::kOwnedBlock, f0, &bars->owned_full, a.of0, blk * 64, wk.row0, wk.g, wk.b);
          tma_rows(smem + L::kOwned + blk * L::kOwnedBlock, f1, &bars->owned_full, a.of1, blk * 64, wk.row0, wk.g, wk.b);
        }
      }
      __syncwarp();
      ++items;
    }
    for (int32_t i = 0; i < wk.n_t; ++i) {
      const uint32_t s = tile % kStages;
      if (tile >= kStages && !wait(&bars->ring_empty[s], tile / kStages - 1)) {
        ok = false;
        break;
      }
      uint8_t* r0_s = smem + L::ring + s * 2 * L::kRing;
      uint8_t* r1_s = r0_s + L::kRing;
      const int32_t t = wk.t0 + i;
      const int32_t hq = KV ? t / a.m_tiles64 : 0;
      const int32_t row = (KV ? t - hq * a.m_tiles64 : t) * kCols, head = KV ? wk.h0 + hq : wk.g;
      if (lane == 0) {
        mbar_arrive_expect_tx(&bars->ring_full[s], 2 * L::kRing + (KV ? L::kStats : 0));
#pragma unroll
        for (int blk = 0; blk < L::kBlocks; ++blk) {
          tma_rows(r0_s + blk * L::kRingBlock, r0, &bars->ring_full[s], a.or0, blk * 64, row, head, wk.b);
          tma_rows(r1_s + blk * L::kRingBlock, r1, &bars->ring_full[s], a.or1, blk * 64, row, head, wk.b);
        }
        if (KV)
          bulk_load(smem + L::stats + s * L::kStats,
                    a.stats + ((static_cast<int64_t>(wk.b) * p.heads + head) * a.m_tiles64 + row / kCols) * (2 * kCols),
                    L::kStats, &bars->ring_full[s]);
      }
      __syncwarp();
      ++tile;
      if (!KV && needs_cleaning(p, wk, i)) {
        // dS is zero for padded keys, but 0 * NaN is not: their K rows become zeros.
        if (!wait(&bars->ring_full[s], (tile - 1) / kStages)) {
          ok = false;
          break;
        }
        for (int c = (wk.length - row) * 8 + lane; c < kCols * 8; c += 32)
#pragma unroll
          for (int blk = 0; blk < L::kBlocks; ++blk)
            reinterpret_cast<uint4*>(r0_s + blk * L::kRingBlock)[c] = make_uint4(0u, 0u, 0u, 0u);
        fence_proxy_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->clean[s]);
      }
    }
  }
  // Every issued copy has landed before the CTA exits.
  volatile int32_t no_abort = 0;
  if (!L::kOwnedInTmem && items > 0)
    mbar_wait(&bars->owned_full, (items - 1) & 1, &no_abort, p.status, kDevTimeoutDrain);
  for (uint32_t s = 0; s < kStages; ++s) {
    const uint32_t cnt = tile > s ? (tile - s + kStages - 1) / kStages : 0;
    if (cnt > 0) mbar_wait(&bars->ring_full[s], (cnt - 1) & 1, &no_abort, p.status, kDevTimeoutDrain);
  }
}

// Tile i: X = F0 R0^T, Y = F1 R1^T (F0, F1 owned, R0, R1 streamed) into the buffer of its parity;
// once the row threads have written a tile's operands, dq: acc0 += X R0;  dk, dv: acc1 += X R1,
// acc0 += Y R0.  A buffer is overwritten by products that were issued after those that read it,
// and products execute in issue order.
template <int DP, bool BF16, bool KV>
__device__ __forceinline__ void mma_role(const Args& a, Bars* bars, uint8_t* smem, uint32_t tmem) {
  using L = Shape<DP, KV>;
  const XaParams& p = a.p.f;
  volatile int32_t* abort_flag = &bars->abort;
  const uint32_t leader = elect_one();
  auto wait = [&](uint64_t* bar, uint32_t phase) -> bool {
    return warp_wait(bar, phase, abort_flag, p.status, kDevTimeoutMma, p.wait_ns);
  };
  const uint32_t idesc_s = idesc_f16(BF16, false, kRows, kCols);
  const uint32_t idesc_acc = idesc_f16(BF16, true, kRows, a.k_steps * 16);
  const uint64_t f0 = smem_desc_sw128(smem_u32(smem), 16, 1024);
  const uint64_t f1 = smem_desc_sw128(smem_u32(smem + (L::kOwnedInTmem ? 0 : L::kOwned)), 16, 1024);
  // Streamed operands: K-major for the scores; MN-major for the sums (depth = the tile's
  // 64 rows, N = head_dim in 64-column blocks).
  const uint64_t r_score = smem_desc_sw128(smem_u32(smem + L::ring), 16, 1024);
  const uint64_t r_acc = smem_desc_sw128(smem_u32(smem + L::ring), L::kRingBlock, 1024);
  uint32_t tile = 0, items = 0;            // tiles summed, items begun
  uint32_t clean_phase = 0;                // bit s: parity of stage s's next cleaned tile
  bool ok = true, issued = false;
  // The streamed tile `t` (the item's i-th) has arrived.
  auto arrived = [&](const Work& wk, uint32_t t, int32_t i) {
    const uint32_t s = t % kStages;
    ok = wait(&bars->ring_full[s], t / kStages);
    if (ok && !KV && needs_cleaning(p, wk, i)) {
      ok = wait(&bars->clean[s], clean_phase >> s);
      clean_phase ^= 1u << s;
    }
  };
  auto score = [&](uint32_t t) {
    const uint32_t st = t & 1, s = t % kStages;
    tc_fence_after();
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const uint64_t r = r_score + ((s * 2 * L::kRing + y * L::kRing) >> 4);
      const uint32_t d = tmem + st * 128 + y * 64;
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk) {
        if (kk >= a.k_steps) continue;
        const uint64_t rb = r + (((kk >> 2) * L::kRingBlock + (kk & 3) * 32) >> 4);
        if (L::kOwnedInTmem)
          mma_ts_warp(leader, d, tmem + L::kColOwned + y * (DP / 2) + kk * 8, rb, idesc_s, kk > 0 ? 1u : 0u);
        else
          mma_ss_warp(leader, d, (y ? f1 : f0) + (((kk >> 2) * L::kOwnedBlock + (kk & 3) * 32) >> 4), rb, idesc_s,
                      kk > 0 ? 1u : 0u);
      }
    }
    mma_commit_warp(leader, &bars->s_full[st]);
    issued = true;
  };
  for (int32_t item = blockIdx.x; item < a.n_items && ok; item += gridDim.x) {
    const Work wk = decode_work<KV>(a, item);
    if (wk.n_t == 0) continue;
    arrived(wk, tile, 0);
    if (ok) ok = wait(&bars->owned_full, items);
    if (!ok) break;
    ++items;
    score(tile);
    if (wk.n_t > 1) arrived(wk, tile + 1, 1);
    for (int32_t i = 0; i < wk.n_t && ok; ++i, ++tile) {
      if (i + 1 < wk.n_t)
        score(tile + 1);
      else
        mma_commit_warp(leader, &bars->owned_empty);
      const uint32_t st = tile & 1, s = tile % kStages;
      // A wait that is already over costs 60 cycles and more.  The next tile's goes under the
      // sums, or, where those are short, before the row threads are waited for.
      if (DP == 64 && i + 2 < wk.n_t) arrived(wk, tile + 2, i + 2);
      if (ok) ok = wait(&bars->ready[st], tile >> 1);
      if (!ok) break;
      tc_fence_after();
      const uint64_t r0 = r_acc + ((s * 2 * L::kRing) >> 4), r1 = r0 + (L::kRing >> 4);
      const uint32_t x = tmem + st * 128, y = x + 64;
#pragma unroll
      for (int kk = 0; kk < kCols / 16; ++kk)
        mma_ts_warp(leader, tmem + kColAcc + (KV ? DP : 0), x + operand_col(kk), (KV ? r1 : r0) + ((kk * 2048) >> 4), idesc_acc,
                    (i > 0 || kk > 0) ? 1u : 0u);
      if (KV) {
#pragma unroll
        for (int kk = 0; kk < kCols / 16; ++kk)
          mma_ts_warp(leader, tmem + kColAcc, y + operand_col(kk), r0 + ((kk * 2048) >> 4), idesc_acc,
                      (i > 0 || kk > 0) ? 1u : 0u);
      }
      mma_commit_warp(leader, &bars->ring_empty[s]);
      if (DP != 64 && i + 2 < wk.n_t) arrived(wk, tile + 2, i + 2);
    }
    if (ok) mma_commit_warp(leader, &bars->acc_full);
  }
  if (issued) {
    volatile int32_t no_abort = 0;
    mma_commit_warp(leader, &bars->drain);
    mbar_wait(&bars->drain, 0, &no_abort, p.status, kDevTimeoutDrain);
  }
}

// The row threads' owned operands on their way to TMEM: this thread's quarter of its row of F0 and F1.
template <int DP>
struct OwnedRow {
  uint4 f[2][DP / (8 * kParts)];
};

template <int DP>
__device__ __forceinline__ void fetch_owned(OwnedRow<DP>& o, const uint16_t* f0, const uint16_t* f1, int c0, int32_t head_dim) {
#pragma unroll
  for (int y = 0; y < 2; ++y) {
    const uint16_t* src = y ? f1 : f0;
#pragma unroll
    for (int c = 0; c < DP / (8 * kParts); ++c) {
      o.f[y][c] = make_uint4(0u, 0u, 0u, 0u);
      if (src != nullptr && c0 + c * 8 < head_dim) o.f[y][c] = __ldg(reinterpret_cast<const uint4*>(src + c0 + c * 8));
    }
  }
}

template <int DP>
__device__ __forceinline__ void store_owned(const OwnedRow<DP>& o, uint32_t taddr) {
  constexpr int kWords = DP / (2 * kParts);   // 8, 16 or 32
#pragma unroll
  for (int y = 0; y < 2; ++y) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(o.f[y]);
    if (kWords == 8) {
      tmem_st8(taddr + y * (DP / 2), *reinterpret_cast<const uint32_t(*)[8]>(w));
    } else {
#pragma unroll
      for (int c = 0; c < kWords; c += 16)
        tmem_st16(taddr + y * (DP / 2) + c, *reinterpret_cast<const uint32_t(*)[16]>(w + c));
    }
  }
  tmem_wait_st();
  tc_fence_before();
}

// This thread's columns of X and Y.
__device__ __forceinline__ void load_scores(uint32_t x, uint32_t (&xr)[kW], uint32_t (&yr)[kW]) {
#pragma unroll
  for (int c = 0; c < kW; c += 16) {
    tmem_ld16(x + c, *reinterpret_cast<uint32_t(*)[16]>(xr + c));
    tmem_ld16(x + 64 + c, *reinterpret_cast<uint32_t(*)[16]>(yr + c));
  }
  tmem_wait_ld();
#pragma unroll
  for (int c = 0; c < kW; c += 16) {
    reg_fence16(*reinterpret_cast<uint32_t(*)[16]>(xr + c));
    reg_fence16(*reinterpret_cast<uint32_t(*)[16]>(yr + c));
  }
}

__device__ __forceinline__ void store_operand(uint32_t taddr, const uint32_t (&w)[kW / 2]) {
  if (kW == 16)
    tmem_st8(taddr, *reinterpret_cast<const uint32_t(*)[8]>(w));
  else
    tmem_st16(taddr, *reinterpret_cast<const uint32_t(*)[16]>(w));
}

// Columns [c0, c0 + DP / kParts) of an accumulator row, scaled, to a 16-bit or (split) fp32 row.
template <int DP, bool BF16>
__device__ __forceinline__ void store_row(uint32_t taddr, int c0, float f, bool write, bool zero, uint16_t* dst,
                                          float* part, bool wide, int32_t head_dim) {
#pragma unroll
  for (int c = 0; c < DP / kParts; c += 16) {
    uint32_t r[16];
    tmem_ld16(taddr + c0 + c, r);
    tmem_wait_ld();
    reg_fence16(r);
    float v[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = zero ? 0.f : __uint_as_float(r[e]) * f;
    if (write) store16<BF16>(v, dst, part, wide, c0 + c, head_dim);
    __syncwarp();
  }
}

// An item without streamed tiles: zeros for its rows.
__device__ __forceinline__ void store_zero_rows(int tid, int32_t rows, uint16_t* dst, float* part, int32_t head_dim) {
  const int64_t chunks = static_cast<int64_t>(rows) * head_dim / 8;
  for (int64_t i = tid; i < chunks; i += kRowThreads) {
    if (part != nullptr) {
      reinterpret_cast<float4*>(part)[2 * i] = make_float4(0.f, 0.f, 0.f, 0.f);
      reinterpret_cast<float4*>(part)[2 * i + 1] = make_float4(0.f, 0.f, 0.f, 0.f);
    } else {
      reinterpret_cast<uint4*>(dst)[i] = make_uint4(0u, 0u, 0u, 0u);
    }
  }
}

// The dq (KV false) and the dk / dv kernel.  Tensor maps f0, f1 of the owned operands (dk / dv
// at head_dim > 64 only), r0, r1 of the streamed ones.
template <int DP, bool BF16, bool KV>
__global__ void __launch_bounds__(kThreads, 1)
xattn_grad_kernel(const __grid_constant__ CUtensorMap tm_f0, const __grid_constant__ CUtensorMap tm_f1,
                  const __grid_constant__ CUtensorMap tm_r0, const __grid_constant__ CUtensorMap tm_r1, const Args a) {
  using L = Shape<DP, KV>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  Bars* bars = reinterpret_cast<Bars*>(smem + L::bars);
  const XaParams& p = a.p.f;
  // read from lane 0: the compiler then knows the roles' values to be uniform
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  volatile int32_t* abort_flag = &bars->abort;

  if (threadIdx.x == 0) init_bars(bars, L::kOwnedInTmem ? kRowWarps : 1);
  if (warp == kMmaWarp) {
    tmem_alloc(&bars->tmem_base, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, bars->tmem_base, 0);

  if (warp == kLoadWarp) {
    load_role<DP, KV>(&tm_f0, &tm_f1, &tm_r0, &tm_r1, a, bars, smem, lane);
  } else if (warp == kMmaWarp) {
    mma_role<DP, BF16, KV>(a, bars, smem, tmem);
  } else if (warp >= kFirstRowWarp) {
    const int tid = threadIdx.x - kFirstRowWarp * 32, row = tid & (kRows - 1), wg = tid >> 7;
    const uint32_t lane_base = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const float2 scale2 = make_float2(p.scale * kLog2e, p.scale * kLog2e);
    const int64_t n_states = static_cast<int64_t>(p.batch) * p.groups * p.states;
    auto wait = [&](uint64_t* bar, uint32_t phase) -> bool {
      return warp_wait(bar, phase, abort_flag, p.status, kDevTimeoutSoftmax, p.wait_ns);
    };
    // The next item with tiles, its owned row and (dq) the row's statistics, fetched one item ahead.
    OwnedRow<DP> owned;
    float nlse = -INFINITY, ndelta = 0.f, next_nlse = -INFINITY, next_ndelta = 0.f;
    // f16: the bound of dS as fetched (dq: |dO| of the row, this lane's part of the largest |v|;
    // dk, dv: this lane's part of the largest |dO| and |delta|, |v| of the key), and what it gives at
    // the hand-over: the factor that takes dS's power of two out of an accumulator again and (dk,
    // dv) the one from 2^12 P to the factor of dS.
    float go_part = 0.f, delta_part = 0.f, v_part = 0.f, undo = p.scale, lift = 1.f;
    auto fetch = [&](int32_t from) -> bool {
      for (int32_t i = from; i < a.n_items; i += gridDim.x) {
        const Work w = decode_work<KV>(a, i);
        if (w.n_t == 0) continue;
        if (L::kOwnedInTmem) {
          const uint16_t *f0 = nullptr, *f1 = nullptr;
          if (row < w.own) {
            const int64_t r = w.row0 + row;
            f0 = KV ? static_cast<const uint16_t*>(p.k) + w.b * p.ks[0] + w.g * p.ks[1] + r * p.ks[2]
                    : static_cast<const uint16_t*>(p.q) + w.b * p.qs[0] + w.h0 * p.qs[1] + r * p.qs[2];
            f1 = KV ? static_cast<const uint16_t*>(p.v) + w.b * p.vs[0] + w.g * p.vs[1] + r * p.vs[2]
                    : static_cast<const uint16_t*>(a.p.dout) + w.b * a.p.ds[0] + w.h0 * a.p.ds[1] + r * a.p.ds[2];
          }
          fetch_owned<DP>(owned, f0, f1, wg * (DP / kParts), p.head_dim);
        }
        if (!KV) {
          next_nlse = -INFINITY;
          next_ndelta = 0.f;
          if (row < w.own) {
            const int32_t m = w.row0 + row;
            const float* st = a.stats + (static_cast<int64_t>(w.b * p.heads + w.h0) * a.m_tiles64 + m / kCols) * (2 * kCols) +
                              m % kCols;
            // not __ldg: the kernel that writes them may still run when this one starts
            next_nlse = __ldcg(st);
            next_ndelta = __ldcg(st + kCols);
          }
          if (!BF16) {
            go_part = row < w.own ? __ldcg(a.p.row_norm + static_cast<int64_t>(w.b * p.heads + w.h0) * a.m_tiles64 * kCols +
                                           w.row0 + row)
                                  : 0.f;
            const int32_t t1 = (w.length + kCols - 1) / kCols;
            const float* src = a.p.v_max + static_cast<int64_t>(w.b * p.groups + w.g) * ((p.states + kCols - 1) / kCols);
            v_part = lane < t1 ? __ldcg(src + lane) : 0.f;
            for (int32_t t = lane + 32; t < t1; t += 32) v_part = max_of(v_part, __ldcg(src + t));
          }
        } else if (!BF16) {
          const float2* tops = reinterpret_cast<const float2*>(a.p.tile_max) +
                               (static_cast<int64_t>(w.b) * p.heads + w.h0) * a.m_tiles64 + w.t0;
          const float2 top = lane < w.n_t ? __ldcg(tops + lane) : make_float2(0.f, 0.f);
          go_part = top.x;
          delta_part = top.y;
          for (int32_t t = lane + 32; t < w.n_t; t += 32) {
            const float2 more_top = __ldcg(tops + t);
            go_part = max_of(go_part, more_top.x);
            delta_part = max_of(delta_part, more_top.y);
          }
          v_part = row < w.own ? __ldcg(a.p.v_norm + static_cast<int64_t>(w.b * p.groups + w.g) * p.states + w.row0 + row)
                               : 0.f;
        }
        return true;
      }
      return false;
    };
    auto hand_over = [&] {
      if (L::kOwnedInTmem) {
        store_owned<DP>(owned, lane_base + L::kColOwned + wg * (DP / (2 * kParts)));
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->owned_full);
      }
      nlse = next_nlse;
      ndelta = next_ndelta;
      if (!BF16) {
        const int32_t e = power_for(KV ? fmaf(warp_max(go_part), v_part, warp_max(delta_part))
                                       : fmaf(go_part, warp_max(v_part), fabsf(ndelta)));
        undo = p.scale * two_to(-e);
        if (KV)
          lift = two_to(e - kPowP);
        else
          nlse += static_cast<float>(e - kPowP);
      }
    };
    uint32_t tile = 0, items = 0;
    bool ok = true;
    if (!KV) {
      wait_previous_kernel();                  // for the statistics
      __threadfence();                         // and for whoever starts after this thread (after_stats)
    }
    // The dk / dv kernel after dq needs the statistics too, and nothing of dq's.
    allow_next_kernel();
    if (KV && !BF16 && a.after_stats) wait_previous_kernel();  // these warps read the bound's parts
    if (fetch(blockIdx.x)) hand_over();
    for (int32_t item = blockIdx.x; item < a.n_items && ok; item += gridDim.x) {
      const Work wk = decode_work<KV>(a, item);
      const int64_t outer = KV ? static_cast<int64_t>(wk.b) * p.groups + wk.g : static_cast<int64_t>(wk.b) * p.heads + wk.h0;
      const int64_t lin0 = outer * (KV ? p.states : p.queries) + wk.row0;
      const int64_t at = (wk.split * (KV ? n_states : p.rows_total) + lin0) * p.head_dim;
      void* const dst[2] = {KV ? a.p.dk : a.p.dq, KV ? a.p.dv : nullptr};
      float* const parts[2] = {KV ? a.p.dk_part : a.p.dq_part, KV ? a.p.dv_part : nullptr};
      if (wk.n_t == 0) {
#pragma unroll
        for (int y = 0; y < (KV ? 2 : 1); ++y)
          if (dst[y] != nullptr)
            store_zero_rows(tid, wk.own, static_cast<uint16_t*>(dst[y]) + lin0 * p.head_dim,
                            parts[y] == nullptr ? nullptr : parts[y] + at, p.head_dim);
        continue;
      }
      const bool more = fetch(item + gridDim.x);
      const float2 nlse2 = make_float2(nlse, nlse), ndelta2 = make_float2(ndelta, ndelta);
      // the item's own: the hand-over of the next one comes before this one's store
      const float2 lift2 = make_float2(lift, lift);
      const float item_undo = undo;
      for (int32_t i = 0; i < wk.n_t; ++i, ++tile) {
        const uint32_t st = tile & 1, s = tile % kStages;
        // The statistics came with the tile that the finished products have read.
        if ((KV && !wait(&bars->ring_full[s], tile / kStages)) || !wait(&bars->s_full[st], tile >> 1)) {
          ok = false;
          break;
        }
        tc_fence_after();
        uint32_t xr[kW], yr[kW], pw[kW / 2], dw[kW / 2];
        const uint32_t x = lane_base + st * 128 + wg * kW;
        load_scores(x, xr, yr);
        const float4* lse4 = reinterpret_cast<const float4*>(smem + L::stats + s * L::kStats) + wg * (kW / 4);
        const float4* delta4 = lse4 + kCols / 4;
#pragma unroll
        for (int e = 0; e < kW; e += 4) {
          // dk, dv: a query's statistics are a column's; dq: the thread's own row's
          float2 nl[2] = {nlse2, nlse2}, nd[2] = {ndelta2, ndelta2};
          if (KV) {
            const float4 l = lse4[e / 4], d = delta4[e / 4];
            nl[0] = make_float2(l.x, l.y);
            nl[1] = make_float2(l.z, l.w);
            nd[0] = make_float2(d.x, d.y);
            nd[1] = make_float2(d.z, d.w);
          }
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int c = e + 2 * u;
            const float2 t = fma2(make_float2(__uint_as_float(xr[c]), __uint_as_float(xr[c + 1])), scale2, nl[u]);
            const float2 pr = make_float2(fast_exp2(t.x), fast_exp2(t.y));
            const float2 g = mul2(KV && !BF16 ? mul2(pr, lift2) : pr, add2(make_float2(__uint_as_float(yr[c]), __uint_as_float(yr[c + 1])), nd[u]));
            if (KV) pw[c / 2] = pack2<BF16>(pr.x, pr.y);
            dw[c / 2] = pack2<BF16>(g.x, g.y);
          }
        }
        if (!KV) {
          const int32_t left = wk.length - (wk.t0 + i) * kCols - wg * kW;  // of this thread's columns
          if (left < kW) {
#pragma unroll
            for (int c = 0; c < kW / 2; ++c) {
              if (2 * c >= left) dw[c] = 0u;
              else if (2 * c + 1 >= left) dw[c] &= 0xffffu;
            }
          }
        }
        if (KV) store_operand(x, pw);          // P^T over the read X columns
        store_operand(KV ? x + 64 : x, dw);    // dS (dk, dv: its transpose over Y)
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->ready[st]);
      }
      if (!ok) break;
      if (more) hand_over();                   // the item's last score product is done
      if (!wait(&bars->acc_full, items)) {
        ok = false;
        break;
      }
      ++items;
      tc_fence_after();
      // A padded key's rows of the accumulators hold whatever its states gave.
      const bool zero = KV && wk.row0 + row >= wk.length;
      const int64_t off = static_cast<int64_t>(row) * p.head_dim;
#pragma unroll
      for (int y = 0; y < (KV ? 2 : 1); ++y)
        store_row<DP, BF16>(lane_base + kColAcc + y * DP, wg * (DP / kParts),
                            y == 0 ? (BF16 ? p.scale : item_undo) : (BF16 ? 1.f : two_to(-kPowP)),
                            row < wk.own && dst[y] != nullptr, zero,
                            static_cast<uint16_t*>(dst[y]) + lin0 * p.head_dim + off,
                            parts[y] == nullptr ? nullptr : parts[y] + at + off, a.wide, p.head_dim);
      tc_fence_before();
    }
  }
  wait_previous_kernel();
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// ============================================================================ split sums
// dst = round(sum_s part[s]), parts in order; 4 values per thread, up to two sums (blockIdx.y).
template <bool BF16>
__global__ void __launch_bounds__(128)
xattn_sum_kernel(const float* part0, uint16_t* dst0, const float* part1, uint16_t* dst1, int64_t n, int32_t n_split) {
  wait_previous_kernel();
  const float* part = blockIdx.y ? part1 : part0;
  uint16_t* dst = blockIdx.y ? dst1 : dst0;
  const int64_t i = (static_cast<int64_t>(blockIdx.x) * 128 + threadIdx.x) * 4;
  if (i >= n) return;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
  for (int s = 0; s < n_split; ++s) {
    const float4 x = __ldcs(reinterpret_cast<const float4*>(part + s * n + i));
    a = make_float4(a.x + x.x, a.y + x.y, a.z + x.z, a.w + x.w);
  }
  *reinterpret_cast<uint2*>(dst + i) = make_uint2(pack2<BF16>(a.x, a.y), pack2<BF16>(a.z, a.w));
}

// One sum, or two of equal size (the second null without).
template <bool BF16>
int32_t launch_sum(const float* part0, void* dst0, const float* part1, void* dst1, int64_t n, int32_t n_split,
                   cudaStream_t stream) {
  const int64_t grid = (n / 4 + 127) / 128;
  if (grid > INT32_MAX) return 8;
  return launch_kernel(xattn_sum_kernel<BF16>, dim3(static_cast<unsigned>(grid), dst1 != nullptr ? 2 : 1), 128, 0, stream,
                       true, part0, static_cast<uint16_t*>(dst0), part1, static_cast<uint16_t*>(dst1), n, n_split)
             ? 0
             : 6;
}

template <int DP, bool BF16, bool KV>
int32_t launch_grad(const CUtensorMap& f0, const CUtensorMap& f1, const CUtensorMap& r0, const CUtensorMap& r1, Args a,
                    int sm_count, cudaStream_t stream) {
  constexpr int smem = Shape<DP, KV>::bars + sizeof(Bars) + 1024;
  static_assert(smem <= 227 * 1024, "shared memory of a CTA");
  static_assert(Shape<DP, KV>::kColOwned + (Shape<DP, KV>::kOwnedInTmem ? DP : 0) <= kTmemCols, "tensor memory");
  const XaParams& p = a.p.f;
  const int64_t outer = static_cast<int64_t>(p.batch) * (KV ? p.groups : p.heads);
  a.n_row_tiles = ((KV ? p.states : p.queries) + kRows - 1) / kRows;
  a.n_split = KV ? a.p.kv_split : a.p.dq_split;
  a.split_tiles = KV ? a.p.kv_split_tiles : a.p.dq_split_tiles;
  const int64_t items = outer * a.n_row_tiles * a.n_split;
  if (items > (1 << 30)) return 8;
  a.n_items = static_cast<int32_t>(items);
  auto kernel = xattn_grad_kernel<DP, BF16, KV>;
  static std::atomic<uint64_t> done{0};
  if (!allow_smem(kernel, smem, done)) return 6;
  // one CTA per SM: it holds all of the SM's tensor memory
  const unsigned grid = static_cast<unsigned>(items < sm_count ? items : sm_count);
  return launch_kernel(kernel, dim3(grid), kThreads, smem, stream, true, f0, f1, r0, r1, a) ? 0 : 6;
}

template <int DP, bool BF16>
int32_t launch_typed(const XaBwdParams& bp, cudaStream_t stream, int sm_count) {
  const XaParams& p = bp.f;
  Args a;
  a.p = bp;
  a.stats = bp.delta;
  a.m_tiles64 = (p.queries + kCols - 1) / kCols;
  a.k_steps = (p.head_dim + 15) / 16;
  a.wide = p.head_dim % 16 == 0;
  for (const void* g : {bp.dq, bp.dk, bp.dv}) a.wide = a.wide && reinterpret_cast<uintptr_t>(g) % 32 == 0;

  const int64_t state_blocks = BF16 ? 0 : static_cast<int64_t>(p.batch) * p.groups * ((p.states + kCols - 1) / kCols);
  const int64_t stat_blocks = static_cast<int64_t>(p.batch) * p.heads * a.m_tiles64 + state_blocks;
  if (stat_blocks > INT32_MAX) return 8;
  xattn_stats_kernel<DP / 8, BF16><<<static_cast<unsigned>(stat_blocks), 256, 0, stream>>>(bp, bp.delta, a.m_tiles64);
  if (cudaGetLastError() != cudaSuccess) return 6;

  SlaParams tq{}, tk{};
  tq.batch = tk.batch = p.batch;
  tq.head_dim = tk.head_dim = p.head_dim;
  tq.dtype = tk.dtype = p.dtype;
  tq.heads = p.heads;
  tq.seq = p.queries;
  tk.heads = p.groups;
  tk.seq = p.states;
  const int64_t qs[4] = {p.qs[0], p.qs[1], p.qs[2], 1}, ds[4] = {bp.ds[0], bp.ds[1], bp.ds[2], 1};
  const int64_t ks[4] = {p.ks[0], p.ks[1], p.ks[2], 1}, vs[4] = {p.vs[0], p.vs[1], p.vs[2], 1};
  if (bp.dq != nullptr) {
    CUtensorMap r0, r1;
    if (!make_map(&r0, &a.or0, p.k, ks, tk, kCols) || !make_map(&r1, &a.or1, p.v, vs, tk, kCols)) return 4;
    static_assert(Shape<DP, false>::kOwnedInTmem, "no maps of q and dO");
    a.after_stats = true;
    const int32_t st = launch_grad<DP, BF16, false>(r0, r1, r0, r1, a, sm_count, stream);
    if (st) return st;
  }
  if (bp.dk != nullptr || bp.dv != nullptr) {
    CUtensorMap f0, f1, r0, r1;
    if (!make_map(&r0, &a.or0, p.q, qs, tq, kCols) || !make_map(&r1, &a.or1, bp.dout, ds, tq, kCols)) return 4;
    f0 = r0;
    f1 = r1;
    if (!Shape<DP, true>::kOwnedInTmem &&
        (!make_map(&f0, &a.of0, p.k, ks, tk, kRows) || !make_map(&f1, &a.of1, p.v, vs, tk, kRows)))
      return 4;
    a.after_stats = bp.dq == nullptr;
    const int32_t st = launch_grad<DP, BF16, true>(f0, f1, r0, r1, a, sm_count, stream);
    if (st) return st;
  }
  if (bp.dq != nullptr && bp.dq_part != nullptr) {
    const int32_t st = launch_sum<BF16>(bp.dq_part, bp.dq, nullptr, nullptr, p.rows_total * p.head_dim, bp.dq_split, stream);
    if (st) return st;
  }
  if ((bp.dk != nullptr || bp.dv != nullptr) && bp.dk_part != nullptr) {
    const int64_t n = static_cast<int64_t>(p.batch) * p.groups * p.states * p.head_dim;
    const int32_t st = bp.dk != nullptr
                           ? launch_sum<BF16>(bp.dk_part, bp.dk, bp.dv_part, bp.dv, n, bp.kv_split, stream)
                           : launch_sum<BF16>(bp.dv_part, bp.dv, nullptr, nullptr, n, bp.kv_split, stream);
    if (st) return st;
  }
  return 0;
}

}  // namespace

int32_t launch_xattn_backward(const XaBwdParams& bp, cudaStream_t stream, int sm_count) {
  if (bp.f.head_dim <= 64)
    return bp.f.dtype == 2 ? launch_typed<64, true>(bp, stream, sm_count) : launch_typed<64, false>(bp, stream, sm_count);
  return bp.f.dtype == 2 ? launch_typed<128, true>(bp, stream, sm_count) : launch_typed<128, false>(bp, stream, sm_count);
}

}  // namespace intp
