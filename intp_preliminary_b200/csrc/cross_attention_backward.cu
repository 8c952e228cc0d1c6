// cross_attention_backward.cu - cross attention gradients on tcgen05 (sm_100a, bf16 / f16).
//
//   P = exp(scale q k^T - lse),  dS = P (dO v^T - delta),  delta = rowsum(dO out)
//   dq = scale dS k,   dk = scale sum_heads dS^T q,   dv = sum_heads P^T dO
//
// Nothing of size M x N is written: two kernels recompute the score tiles.
//   xattn_stats_kernel   lse in log2 units and delta of every query row, rows padded
//                        to whole tiles so that a tile's values are one bulk copy.
//   xattn_dq_kernel      a CTA owns 128 query rows of a head and streams 64-key tiles:
//                        X = q k^T and Y = dO v^T into TMEM, dS (16-bit) back over X,
//                        dq += dS k with dS read from TMEM.
//   xattn_dkv_kernel     a CTA owns 128 keys of a key head and streams 64-query tiles of
//                        all its query heads: X = k q^T, Y = v dO^T, P^T over X and dS^T
//                        over Y, dv += P^T dO and dk += dS^T q.  Grouped heads are summed
//                        in the accumulators, in a fixed order.
// Where one side has too few tiles for the GPU, the streamed axis is split and fp32
// parts are summed in order (xattn_sum_kernel).  Every output element has one writer
// and no atomics are used, so results repeat bit for bit.
//
// A CTA: 16 row warps (thread t owns TMEM lane t % 128 and 16 of a tile's 64 columns),
// a TMA warp and an MMA warp.  Score buffers are double: the products of tile t + 1 run
// under the row threads' tile t.  Recomputing the scores in both kernels costs 7 matrix
// products where 5 would do; in exchange dq needs no cross-CTA sum (fp32 atomics in an
// order that changes results, or a key-length workspace).
// P and dS are rounded to 16 bits as the tensor core's operands; all sums are fp32.
#include <cuda.h>
#include <cstdint>
#include "sla_tc_common.cuh"
#include "xattn_common.cuh"
#include "xattn_internal.h"

namespace intp {
namespace {

constexpr int kRows = 128;                 // TMEM lanes: query rows (dq) / keys (dk, dv)
constexpr int kCols = 64;                  // streamed tile: keys (dq) / query rows (dk, dv)
constexpr int kW = 16;                     // columns of a tile per row thread
constexpr int kRowThreads = kRows * kCols / kW;  // 512
constexpr int kRowWarps = kRowThreads / 32;
constexpr int kLoadWarp = kRowWarps, kMmaWarp = kRowWarps + 1;
constexpr int kThreads = kRowThreads + 64;
constexpr int kStages = 4;
constexpr uint32_t kTmemCols = 512, kColAcc = 256;
constexpr float kLog2e = 1.4426950408889634f;

template <int DP>
struct Shape {
  static constexpr int kBlocks = DP / 64;
  static constexpr uint32_t kFixedBlock = kRows * 128, kRingBlock = kCols * 128;
  static constexpr uint32_t kFixed = kBlocks * kFixedBlock;   // one resident operand
  static constexpr uint32_t kRing = kBlocks * kRingBlock;     // one streamed operand
  static constexpr uint32_t kStats = 2 * kCols * 4;           // lse, delta of 64 query rows
  static constexpr uint32_t fixed0 = 0, fixed1 = kFixed, ring = 2 * kFixed;
  static constexpr uint32_t stats = ring + kStages * 2 * kRing;
  static constexpr uint32_t bars = stats + kStages * kStats;
};

struct alignas(8) Bars {
  uint64_t fixed_full;
  uint64_t ring_full[kStages], ring_empty[kStages];
  uint64_t clean;                          // padded key rows of a K tile zeroed (dq)
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
  int32_t n_row_tiles, n_split, split_tiles;
  int32_t k_steps;
};

// What a CTA streams and owns.
struct Work {
  int32_t b, g, h0;          // sequence, key head, first query head (dq: the head itself)
  int32_t row0;              // first owned row
  int32_t t0, n_t;           // streamed tiles [t0, t0 + n_t)
  int32_t length, split;
};

// ============================================================================ row statistics
// 8 lanes per query row.  Rows past M, and rows without states, get lse = +inf: their P is zero.
template <bool BF16>
__global__ void __launch_bounds__(256)
xattn_stats_kernel(const XaBwdParams bp, float* stats, int32_t m_tiles64) {
  const XaParams& p = bp.f;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 32 + (threadIdx.x >> 3);
  const int sub = threadIdx.x & 7;
  const int64_t m_pad = static_cast<int64_t>(m_tiles64) * kCols;
  const int64_t bh = row / m_pad;
  const int32_t m = static_cast<int32_t>(row - bh * m_pad);
  float delta = 0.f, lse = INFINITY;
  if (bh < static_cast<int64_t>(p.batch) * p.heads && m < p.queries) {
    const int32_t b = static_cast<int32_t>(bh / p.heads), h = static_cast<int32_t>(bh - static_cast<int64_t>(b) * p.heads);
    const uint4* o = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.out) + b * p.os[0] + h * p.os[1] +
                                                    m * p.os[2]);
    const uint4* d = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(bp.dout) + b * bp.ds[0] +
                                                    h * bp.ds[1] + m * bp.ds[2]);
    for (int c = sub; c * 8 < p.head_dim; c += 8) {
      const uint4 x = __ldg(o + c), y = __ldg(d + c);
      const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 u = unpack2<BF16>(xs[e]), v = unpack2<BF16>(ys[e]);
        delta = fmaf(u.x, v.x, delta);
        delta = fmaf(u.y, v.y, delta);
      }
    }
    const float l = p.lse[bh * p.queries + m];
    lse = l == -INFINITY ? INFINITY : l * kLog2e;
  }
#pragma unroll
  for (int s = 4; s > 0; s >>= 1) delta += __shfl_xor_sync(0xffffffffu, delta, s);
  if (sub == 0 && bh < static_cast<int64_t>(p.batch) * p.heads) {
    float* dst = stats + (bh * m_tiles64 + m / kCols) * (2 * kCols) + m % kCols;
    dst[0] = -lse;
    dst[kCols] = -delta;
  }
}

// ============================================================================ shared roles
__device__ __forceinline__ void init_bars(Bars* bars) {
  mbar_init(&bars->fixed_full, 1);
  for (int s = 0; s < kStages; ++s) {
    mbar_init(&bars->ring_full[s], 1);
    mbar_init(&bars->ring_empty[s], 1);
  }
  mbar_init(&bars->clean, 1);
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

// Streamed tile t of the CTA: key tile t (dq), or query tile t % m_tiles64 of query head h0 + t / m_tiles64.
template <int DP, bool KV>
__device__ __forceinline__ void load_role(const CUtensorMap* f0, const CUtensorMap* f1, const CUtensorMap* r0,
                                          const CUtensorMap* r1, const Args& a, const Work& wk, Bars* bars,
                                          uint8_t* smem, int lane) {
  using L = Shape<DP>;
  const XaParams& p = a.p.f;
  volatile int32_t* abort_flag = &bars->abort;
  const int32_t fixed_head = KV ? wk.g : wk.h0;
  if (lane == 0) {
    tma_prefetch_desc(f0);
    tma_prefetch_desc(f1);
    tma_prefetch_desc(r0);
    tma_prefetch_desc(r1);
    mbar_arrive_expect_tx(&bars->fixed_full, 2 * L::kFixed);
#pragma unroll
    for (int blk = 0; blk < L::kBlocks; ++blk) {
      tma_rows(smem + L::fixed0 + blk * L::kFixedBlock, f0, &bars->fixed_full, a.of0, blk * 64, wk.row0, fixed_head, wk.b);
      tma_rows(smem + L::fixed1 + blk * L::kFixedBlock, f1, &bars->fixed_full, a.of1, blk * 64, wk.row0, fixed_head, wk.b);
    }
  }
  int32_t loaded = 0;
  for (int32_t i = 0; i < wk.n_t; ++i) {
    const int s = i % kStages;
    if (i >= kStages && !warp_wait(&bars->ring_empty[s], i / kStages - 1, abort_flag, p.status, kDevTimeoutProducer,
                                   p.wait_ns))
      break;
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
    ++loaded;
    const int32_t valid = wk.length - row;
    if (!KV && valid < kCols && wk.length < p.states) {
      // dS is zero for padded keys, but 0 * NaN is not: their K rows become zeros.
      if (!warp_wait(&bars->ring_full[s], i / kStages, abort_flag, p.status, kDevTimeoutProducer, p.wait_ns)) break;
      for (int c = valid * 8 + lane; c < kCols * 8; c += 32)
#pragma unroll
        for (int blk = 0; blk < L::kBlocks; ++blk)
          reinterpret_cast<uint4*>(r0_s + blk * L::kRingBlock)[c] = make_uint4(0u, 0u, 0u, 0u);
      fence_proxy_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->clean);
    }
  }
  // Every issued copy has landed before the CTA exits.
  volatile int32_t no_abort = 0;
  mbar_wait(&bars->fixed_full, 0, &no_abort, p.status, kDevTimeoutDrain);
  for (int s = 0; s < kStages; ++s) {
    const int32_t cnt = loaded > s ? (loaded - s + kStages - 1) / kStages : 0;
    if (cnt > 0) mbar_wait(&bars->ring_full[s], (cnt - 1) & 1, &no_abort, p.status, kDevTimeoutDrain);
  }
}

// Tile i: X = F0 R0^T, Y = F1 R1^T into buffer i & 1; then, once the row threads have
// written tile i - 1's operands, dq: acc0 += X R0;  dk, dv: acc1 += X R1, acc0 += Y R0.
template <int DP, bool BF16, bool KV>
__device__ __forceinline__ void mma_role(const Args& a, const Work& wk, Bars* bars, uint8_t* smem, uint32_t tmem) {
  using L = Shape<DP>;
  const XaParams& p = a.p.f;
  volatile int32_t* abort_flag = &bars->abort;
  const uint32_t leader = elect_one();
  auto wait = [&](uint64_t* bar, uint32_t phase) -> bool {
    return warp_wait(bar, phase, abort_flag, p.status, kDevTimeoutMma, p.wait_ns);
  };
  const uint32_t idesc_s = idesc_f16(BF16, false, kRows, kCols);
  const uint32_t idesc_acc = idesc_f16(BF16, true, kRows, a.k_steps * 16);
  const uint64_t f0 = smem_desc_sw128(smem_u32(smem + L::fixed0), 16, 1024);
  const uint64_t f1 = smem_desc_sw128(smem_u32(smem + L::fixed1), 16, 1024);
  // Streamed operands: K-major for the scores; MN-major for the sums (depth = the tile's
  // 64 rows, N = head_dim in 64-column blocks).
  const uint64_t r_score = smem_desc_sw128(smem_u32(smem + L::ring), 16, 1024);
  const uint64_t r_acc = smem_desc_sw128(smem_u32(smem + L::ring), L::kRingBlock, 1024);
  bool issued = false;
  auto acc = [&](int32_t i) -> bool {
    const uint32_t st = i & 1, s = i % kStages;
    if (!wait(&bars->ready[st], i >> 1)) return false;
    tc_fence_after();
    const uint64_t r0 = r_acc + ((s * 2 * L::kRing) >> 4), r1 = r0 + (L::kRing >> 4);
    const uint32_t x = tmem + st * 128, y = x + 64;
#pragma unroll
    for (int kk = 0; kk < kCols / 16; ++kk)
      mma_ts_warp(leader, tmem + kColAcc + (KV ? DP : 0), x + kk * kW, (KV ? r1 : r0) + ((kk * 2048) >> 4), idesc_acc,
                  (i > 0 || kk > 0) ? 1u : 0u);
    if (KV) {
#pragma unroll
      for (int kk = 0; kk < kCols / 16; ++kk)
        mma_ts_warp(leader, tmem + kColAcc, y + kk * kW, r0 + ((kk * 2048) >> 4), idesc_acc,
                    (i > 0 || kk > 0) ? 1u : 0u);
    }
    mma_commit_warp(leader, &bars->ring_empty[s]);
    return true;
  };
  bool ok = wait(&bars->fixed_full, 0);
  for (int32_t i = 0; i < wk.n_t && ok; ++i) {
    const uint32_t st = i & 1, s = i % kStages;
    ok = wait(&bars->ring_full[s], i / kStages);
    if (ok && !KV && wk.length - (wk.t0 + i) * kCols < kCols && wk.length < p.states) ok = wait(&bars->clean, 0);
    if (!ok) break;
    // Buffer st was read by tile i - 2's sums, issued before: products execute in issue order.
    tc_fence_after();
    const uint64_t r0 = r_score + ((s * 2 * L::kRing) >> 4), r1 = r0 + (L::kRing >> 4);
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk)
      if (kk < a.k_steps)
        mma_ss_warp(leader, tmem + st * 128, f0 + (((kk >> 2) * L::kFixedBlock + (kk & 3) * 32) >> 4),
                    r0 + (((kk >> 2) * L::kRingBlock + (kk & 3) * 32) >> 4), idesc_s, kk > 0 ? 1u : 0u);
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk)
      if (kk < a.k_steps)
        mma_ss_warp(leader, tmem + st * 128 + 64, f1 + (((kk >> 2) * L::kFixedBlock + (kk & 3) * 32) >> 4),
                    r1 + (((kk >> 2) * L::kRingBlock + (kk & 3) * 32) >> 4), idesc_s, kk > 0 ? 1u : 0u);
    mma_commit_warp(leader, &bars->s_full[st]);
    issued = true;
    if (i >= 1) ok = acc(i - 1);
  }
  if (ok && acc(wk.n_t - 1)) mma_commit_warp(leader, &bars->acc_full);
  if (issued) {
    volatile int32_t no_abort = 0;
    mma_commit_warp(leader, &bars->drain);
    mbar_wait(&bars->drain, 0, &no_abort, p.status, kDevTimeoutDrain);
  }
}

// This thread's 16 columns of X and Y.
__device__ __forceinline__ void load_scores(uint32_t x, uint32_t (&xr)[kW], uint32_t (&yr)[kW]) {
  tmem_ld16(x, xr);
  tmem_ld16(x + 64, yr);
  tmem_wait_ld();
  reg_fence16(xr);
  reg_fence16(yr);
}

// Columns [c0, c0 + DP / 4) of an accumulator row, scaled, to a 16-bit or (split) fp32 row.
template <int DP, bool BF16>
__device__ __forceinline__ void store_row(uint32_t taddr, int c0, float f, bool write, bool zero, uint16_t* dst,
                                          float* part, int32_t head_dim) {
#pragma unroll
  for (int c = 0; c < DP / 4; c += 16) {
    uint32_t r[16];
    tmem_ld16(taddr + c0 + c, r);
    tmem_wait_ld();
    reg_fence16(r);
    float v[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = zero ? 0.f : __uint_as_float(r[e]) * f;
    if (write) {
#pragma unroll
      for (int e = 0; e < 16; e += 8) {
        if (c0 + c + e >= head_dim) break;
        if (part != nullptr) {
          reinterpret_cast<float4*>(part + c0 + c + e)[0] = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
          reinterpret_cast<float4*>(part + c0 + c + e)[1] = make_float4(v[e + 4], v[e + 5], v[e + 6], v[e + 7]);
        } else {
          *reinterpret_cast<uint4*>(dst + c0 + c + e) =
              make_uint4(pack2<BF16>(v[e], v[e + 1]), pack2<BF16>(v[e + 2], v[e + 3]), pack2<BF16>(v[e + 4], v[e + 5]),
                         pack2<BF16>(v[e + 6], v[e + 7]));
        }
      }
    }
    __syncwarp();
  }
}

// A CTA without streamed tiles: zeros for its rows.
__device__ __forceinline__ void store_zero_rows(int32_t rows, uint16_t* dst, float* part, int32_t head_dim) {
  const int64_t chunks = static_cast<int64_t>(rows) * head_dim / 8;
  for (int64_t i = threadIdx.x; i < chunks; i += blockDim.x) {
    if (part != nullptr) {
      reinterpret_cast<float4*>(part)[2 * i] = make_float4(0.f, 0.f, 0.f, 0.f);
      reinterpret_cast<float4*>(part)[2 * i + 1] = make_float4(0.f, 0.f, 0.f, 0.f);
    } else {
      reinterpret_cast<uint4*>(dst)[i] = make_uint4(0u, 0u, 0u, 0u);
    }
  }
}

// ============================================================================ dq
template <int DP, bool BF16>
__global__ void __launch_bounds__(kThreads, 1)
xattn_dq_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_do,
                const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const Args a) {
  using L = Shape<DP>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  Bars* bars = reinterpret_cast<Bars*>(smem + L::bars);
  const XaParams& p = a.p.f;
  // read from lane 0: the compiler then knows the roles' values to be uniform
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  volatile int32_t* abort_flag = &bars->abort;

  Work wk;
  const int32_t rest = blockIdx.x / a.n_row_tiles;
  wk.row0 = (blockIdx.x - rest * a.n_row_tiles) * kRows;
  const int32_t bh = rest / a.n_split;
  wk.split = rest - bh * a.n_split;
  wk.b = bh / p.heads;
  wk.h0 = bh - wk.b * p.heads;
  wk.g = wk.h0 / p.per_group;
  wk.length = xa_length(p, wk.b);
  wk.t0 = wk.split * a.split_tiles;
  const int32_t tiles = (wk.length + kCols - 1) / kCols - wk.t0;
  wk.n_t = tiles < 0 ? 0 : (tiles < a.split_tiles ? tiles : a.split_tiles);

  const int32_t own = p.queries - wk.row0 < kRows ? p.queries - wk.row0 : kRows;
  const int64_t lin0 = static_cast<int64_t>(bh) * p.queries + wk.row0;
  uint16_t* out = static_cast<uint16_t*>(a.p.dq) + lin0 * p.head_dim;
  float* part = a.p.dq_part == nullptr ? nullptr
                                       : a.p.dq_part + (wk.split * p.rows_total + lin0) * p.head_dim;
  if (wk.n_t == 0) {
    store_zero_rows(own, out, part, p.head_dim);
    return;
  }

  if (threadIdx.x == 0) init_bars(bars);
  if (warp == kMmaWarp) {
    tmem_alloc(&bars->tmem_base, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, bars->tmem_base, 0);

  if (warp == kLoadWarp) {
    load_role<DP, false>(&tm_q, &tm_do, &tm_k, &tm_v, a, wk, bars, smem, lane);
  } else if (warp == kMmaWarp) {
    mma_role<DP, BF16, false>(a, wk, bars, smem, tmem);
  } else {
    const int row = threadIdx.x & (kRows - 1), wg = threadIdx.x >> 7;
    const uint32_t lane_base = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const float scale_log2 = p.scale * kLog2e;
    float nlse = -INFINITY, ndelta = 0.f;
    if (row < own) {
      const int32_t m = wk.row0 + row;
      const float* st = a.stats + (static_cast<int64_t>(bh) * a.m_tiles64 + m / kCols) * (2 * kCols) + m % kCols;
      nlse = __ldg(st);
      ndelta = __ldg(st + kCols);
    }
    const float2 scale2 = make_float2(scale_log2, scale_log2), nlse2 = make_float2(nlse, nlse),
                 ndelta2 = make_float2(ndelta, ndelta);
    auto wait = [&](uint64_t* bar, uint32_t phase) -> bool {
      return warp_wait(bar, phase, abort_flag, p.status, kDevTimeoutSoftmax, p.wait_ns);
    };
    bool ok = true;
    for (int32_t i = 0; i < wk.n_t; ++i) {
      const int st = i & 1;
      if (!wait(&bars->s_full[st], i >> 1)) {
        ok = false;
        break;
      }
      tc_fence_after();
      uint32_t xr[kW], yr[kW], dw[kW / 2];
      const uint32_t x = lane_base + st * 128 + wg * kW;
      load_scores(x, xr, yr);
      const int32_t left = wk.length - (wk.t0 + i) * kCols - wg * kW;  // of this thread's columns
#pragma unroll
      for (int e = 0; e < kW; e += 2) {
        const float2 t = fma2(make_float2(__uint_as_float(xr[e]), __uint_as_float(xr[e + 1])), scale2, nlse2);
        float2 d = add2(make_float2(__uint_as_float(yr[e]), __uint_as_float(yr[e + 1])), ndelta2);
        d = mul2(make_float2(fast_exp2(t.x), fast_exp2(t.y)), d);
        if (e >= left) d.x = 0.f;
        if (e + 1 >= left) d.y = 0.f;
        dw[e / 2] = pack2<BF16>(d.x, d.y);
      }
      tmem_st8(x, dw);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->ready[st]);
    }
    if (ok && wait(&bars->acc_full, 0)) {
      tc_fence_after();
      store_row<DP, BF16>(lane_base + kColAcc, wg * (DP / 4), p.scale, row < own, false,
                          out + static_cast<int64_t>(row) * p.head_dim,
                          part == nullptr ? nullptr : part + static_cast<int64_t>(row) * p.head_dim, p.head_dim);
      tc_fence_before();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// ============================================================================ dk, dv
template <int DP, bool BF16>
__global__ void __launch_bounds__(kThreads, 1)
xattn_dkv_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                 const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_do, const Args a) {
  using L = Shape<DP>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  Bars* bars = reinterpret_cast<Bars*>(smem + L::bars);
  const XaParams& p = a.p.f;
  // read from lane 0: the compiler then knows the roles' values to be uniform
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  volatile int32_t* abort_flag = &bars->abort;

  Work wk;
  const int32_t rest = blockIdx.x / a.n_row_tiles;
  wk.row0 = (blockIdx.x - rest * a.n_row_tiles) * kRows;
  const int32_t bg = rest / a.n_split;
  wk.split = rest - bg * a.n_split;
  wk.b = bg / p.groups;
  wk.g = bg - wk.b * p.groups;
  wk.h0 = wk.g * p.per_group;
  wk.length = xa_length(p, wk.b);
  wk.t0 = wk.split * a.split_tiles;
  const int32_t tiles = p.per_group * a.m_tiles64 - wk.t0;
  wk.n_t = tiles < 0 || wk.row0 >= wk.length ? 0 : (tiles < a.split_tiles ? tiles : a.split_tiles);

  const int32_t own = p.states - wk.row0 < kRows ? p.states - wk.row0 : kRows;
  const int64_t n_states = static_cast<int64_t>(p.batch) * p.groups * p.states;
  const int64_t lin0 = static_cast<int64_t>(bg) * p.states + wk.row0;
  uint16_t* dk = static_cast<uint16_t*>(a.p.dk) + lin0 * p.head_dim;
  uint16_t* dv = static_cast<uint16_t*>(a.p.dv) + lin0 * p.head_dim;
  const int64_t at = (wk.split * n_states + lin0) * p.head_dim;
  float* dk_part = a.p.dk_part == nullptr ? nullptr : a.p.dk_part + at;
  float* dv_part = a.p.dv_part == nullptr ? nullptr : a.p.dv_part + at;
  if (wk.n_t == 0) {
    if (a.p.dk != nullptr) store_zero_rows(own, dk, dk_part, p.head_dim);
    if (a.p.dv != nullptr) store_zero_rows(own, dv, dv_part, p.head_dim);
    return;
  }

  if (threadIdx.x == 0) init_bars(bars);
  if (warp == kMmaWarp) {
    tmem_alloc(&bars->tmem_base, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, bars->tmem_base, 0);

  if (warp == kLoadWarp) {
    load_role<DP, true>(&tm_k, &tm_v, &tm_q, &tm_do, a, wk, bars, smem, lane);
  } else if (warp == kMmaWarp) {
    mma_role<DP, BF16, true>(a, wk, bars, smem, tmem);
  } else {
    const int row = threadIdx.x & (kRows - 1), wg = threadIdx.x >> 7;
    const uint32_t lane_base = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const float2 scale2 = make_float2(p.scale * kLog2e, p.scale * kLog2e);
    auto wait = [&](uint64_t* bar, uint32_t phase) -> bool {
      return warp_wait(bar, phase, abort_flag, p.status, kDevTimeoutSoftmax, p.wait_ns);
    };
    bool ok = true;
    for (int32_t i = 0; i < wk.n_t; ++i) {
      const int st = i & 1, s = i % kStages;
      // The statistics came with the tile that the finished products have read.
      if (!wait(&bars->ring_full[s], i / kStages) || !wait(&bars->s_full[st], i >> 1)) {
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
        const float4 l = lse4[e / 4], d = delta4[e / 4];
        // the statistics come negated
        const float2 nl[2] = {make_float2(l.x, l.y), make_float2(l.z, l.w)};
        const float2 nd[2] = {make_float2(d.x, d.y), make_float2(d.z, d.w)};
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int c = e + 2 * u;
          const float2 t = fma2(make_float2(__uint_as_float(xr[c]), __uint_as_float(xr[c + 1])), scale2, nl[u]);
          const float2 pr = make_float2(fast_exp2(t.x), fast_exp2(t.y));
          const float2 g = mul2(pr, add2(make_float2(__uint_as_float(yr[c]), __uint_as_float(yr[c + 1])), nd[u]));
          pw[c / 2] = pack2<BF16>(pr.x, pr.y);
          dw[c / 2] = pack2<BF16>(g.x, g.y);
        }
      }
      tmem_st8(x, pw);
      tmem_st8(x + 64, dw);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->ready[st]);
    }
    if (ok && wait(&bars->acc_full, 0)) {
      tc_fence_after();
      // A padded key's row of the accumulators holds whatever its states gave.
      const bool zero = wk.row0 + row >= wk.length;
      const int64_t off = static_cast<int64_t>(row) * p.head_dim;
      store_row<DP, BF16>(lane_base + kColAcc, wg * (DP / 4), p.scale, row < own && a.p.dk != nullptr, zero, dk + off,
                          dk_part == nullptr ? nullptr : dk_part + off, p.head_dim);
      store_row<DP, BF16>(lane_base + kColAcc + DP, wg * (DP / 4), 1.f, row < own && a.p.dv != nullptr, zero, dv + off,
                          dv_part == nullptr ? nullptr : dv_part + off, p.head_dim);
      tc_fence_before();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// ============================================================================ split sums
// dst = round(sum_s part[s]), parts in order; 8 values per thread.
template <bool BF16>
__global__ void __launch_bounds__(256)
xattn_sum_kernel(const float* part, uint16_t* dst, int64_t n, int32_t n_split) {
  const int64_t i = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 8;
  if (i >= n) return;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
#pragma unroll 4
  for (int s = 0; s < n_split; ++s) {
    const float4 x = *reinterpret_cast<const float4*>(part + s * n + i);
    const float4 y = *reinterpret_cast<const float4*>(part + s * n + i + 4);
    a = make_float4(a.x + x.x, a.y + x.y, a.z + x.z, a.w + x.w);
    b = make_float4(b.x + y.x, b.y + y.y, b.z + y.z, b.w + y.w);
  }
  *reinterpret_cast<uint4*>(dst + i) =
      make_uint4(pack2<BF16>(a.x, a.y), pack2<BF16>(a.z, a.w), pack2<BF16>(b.x, b.y), pack2<BF16>(b.z, b.w));
}

template <bool BF16>
int32_t launch_sum(const float* part, void* dst, int64_t n, int32_t n_split, cudaStream_t stream) {
  const int64_t grid = (n / 8 + 255) / 256;
  if (grid > INT32_MAX) return 8;
  xattn_sum_kernel<BF16><<<static_cast<unsigned>(grid), 256, 0, stream>>>(part, static_cast<uint16_t*>(dst), n, n_split);
  return cudaGetLastError() == cudaSuccess ? 0 : 6;
}

template <int DP, bool BF16>
int32_t launch_typed(const XaBwdParams& bp, cudaStream_t stream) {
  using L = Shape<DP>;
  const XaParams& p = bp.f;
  constexpr int smem = L::bars + sizeof(Bars) + 1024;
  static_assert(smem <= 227 * 1024, "shared memory of a CTA");
  Args a;
  a.p = bp;
  a.stats = bp.delta;
  a.m_tiles64 = (p.queries + kCols - 1) / kCols;
  a.k_steps = (p.head_dim + 15) / 16;

  const int64_t stat_rows = static_cast<int64_t>(p.batch) * p.heads * a.m_tiles64 * kCols;
  xattn_stats_kernel<BF16><<<static_cast<unsigned>(stat_rows / 32), 256, 0, stream>>>(bp, bp.delta, a.m_tiles64);
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
  CUtensorMap f0, f1, r0, r1;
  if (bp.dq != nullptr) {
    if (!make_map(&f0, &a.of0, p.q, qs, tq, kRows) || !make_map(&f1, &a.of1, bp.dout, ds, tq, kRows) ||
        !make_map(&r0, &a.or0, p.k, ks, tk, kCols) || !make_map(&r1, &a.or1, p.v, vs, tk, kCols))
      return 4;
    a.n_row_tiles = (p.queries + kRows - 1) / kRows;
    a.n_split = bp.dq_split;
    a.split_tiles = bp.dq_split_tiles;
    const int64_t grid = static_cast<int64_t>(p.batch) * p.heads * a.n_row_tiles * a.n_split;
    if (grid > INT32_MAX) return 8;
    auto kernel = xattn_dq_kernel<DP, BF16>;
    static std::atomic<uint64_t> done{0};
    if (!allow_smem(kernel, smem, done)) return 6;
    kernel<<<static_cast<unsigned>(grid), kThreads, smem, stream>>>(f0, f1, r0, r1, a);
    if (cudaGetLastError() != cudaSuccess) return 6;
    if (bp.dq_part != nullptr) {
      const int32_t st = launch_sum<BF16>(bp.dq_part, bp.dq, p.rows_total * p.head_dim, a.n_split, stream);
      if (st) return st;
    }
  }
  if (bp.dk != nullptr || bp.dv != nullptr) {
    if (!make_map(&f0, &a.of0, p.k, ks, tk, kRows) || !make_map(&f1, &a.of1, p.v, vs, tk, kRows) ||
        !make_map(&r0, &a.or0, p.q, qs, tq, kCols) || !make_map(&r1, &a.or1, bp.dout, ds, tq, kCols))
      return 4;
    a.n_row_tiles = (p.states + kRows - 1) / kRows;
    a.n_split = bp.kv_split;
    a.split_tiles = bp.kv_split_tiles;
    const int64_t grid = static_cast<int64_t>(p.batch) * p.groups * a.n_row_tiles * a.n_split;
    if (grid > INT32_MAX) return 8;
    auto kernel = xattn_dkv_kernel<DP, BF16>;
    static std::atomic<uint64_t> done{0};
    if (!allow_smem(kernel, smem, done)) return 6;
    kernel<<<static_cast<unsigned>(grid), kThreads, smem, stream>>>(f0, f1, r0, r1, a);
    if (cudaGetLastError() != cudaSuccess) return 6;
    const int64_t n = static_cast<int64_t>(p.batch) * p.groups * p.states * p.head_dim;
    if (bp.dk_part != nullptr && bp.dk != nullptr) {
      const int32_t st = launch_sum<BF16>(bp.dk_part, bp.dk, n, a.n_split, stream);
      if (st) return st;
    }
    if (bp.dv_part != nullptr && bp.dv != nullptr) {
      const int32_t st = launch_sum<BF16>(bp.dv_part, bp.dv, n, a.n_split, stream);
      if (st) return st;
    }
  }
  return 0;
}

}  // namespace

int32_t launch_xattn_backward(const XaBwdParams& bp, cudaStream_t stream) {
  if (bp.f.head_dim <= 64)
    return bp.f.dtype == 2 ? launch_typed<64, true>(bp, stream) : launch_typed<64, false>(bp, stream);
  return bp.f.dtype == 2 ? launch_typed<128, true>(bp, stream) : launch_typed<128, false>(bp, stream);
}

}  // namespace intp
