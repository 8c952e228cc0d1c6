// cross_attention_tiles.cu - cross attention forward on tcgen05 (sm_100a, bf16 / f16).
//
//   S = scale q k^T,  P = exp(S - rowmax),  out = (P v) / rowsum(P)
//
// in one pass over the states with the running maximum and sum of a softmax.
// A work item is 256 rows of an instance (xattn_internal.h: all rows that read
// the same states, so the query heads of a key head, or a whole batch's rows on
// a shared prefix, share every key / value tile) and a range of 128-key tiles.
//
// CTA (384 threads, one per SM, persistent over work items):
//   warps 0-3, 4-7  two softmax warpgroups; thread t owns row t % 128 of its
//                   128 rows (TMEM lane).  It copies its query row into the
//                   swizzled operand tile itself (rows of an instance have no
//                   single stride that a tensor map could hold), reads S from
//                   TMEM, keeps the running maximum and the fp32 row sum, and
//                   writes P (16-bit) to TMEM.  O is rescaled there only when the
//                   maximum grew by more than 2^8.
//   warp 8          TMA producer of K and V tiles through one ring; it zeroes the
//                   V rows of a tile past the sequence's length, since 0 * NaN of
//                   a padded state would reach the output through the product.
//   warp 9          issues S = q k^T and O += P v for both warpgroups in turn,
//                   so one's products run under the other's softmax.
//
// P is rounded to 16 bits because the tensor core takes no wider operand of this
// rate (two parts of it, as the few-rows kernel multiplies, would be half as many products
// again): 1.4 times the error of a 32-bit computation rounded once, 0.0024 for 0.0017 in
// bf16.  S, the softmax statistics and O stay in fp32.  Every mbarrier wait is
// bounded (sm100_ptx.cuh); on expiry the CTA unwinds and reports.
//
// Bound by the chain scores -> exponentials -> product of each warpgroup, which the
// other one's products fill: at B4 H16 M2048 N4096 D128 226 to 228 us in bf16, 1.21 PFLOP/s.
// The tensor pipe is busy 64 % of the time at B1 (32 % where one lane of a divergent branch
// issued the products).  Two threads per row (16 softmax warps) measured 249 us: the
// instructions of four warps a scheduler cost more than the shorter chain gives.
#include <cuda.h>
#include <cstdint>
#include "sla_tc_common.cuh"
#include "xattn_common.cuh"
#include "xattn_internal.h"

namespace intp {
namespace {

constexpr int BM = 128;                    // rows of a warpgroup
constexpr int BN = kXaTileKeys;            // keys of a tile
constexpr int kGroups = 2;                 // softmax warpgroups
constexpr int kThreads = kGroups * 128 + 128;
// A softmax thread holds its row's 128 scores: its warpgroups take registers that the
// third one (load and MMA warps, two idle) gives up; 2 x 224 + 56 = 3 x 168, the launch's share.
constexpr int kSoftmaxRegs = 224, kOtherRegs = 56;
constexpr int kLoadWarp = kGroups * 4, kMmaWarp = kLoadWarp + 1;
constexpr uint32_t kBlockBytes = 128 * 128;  // 128 rows of 64 16-bit columns
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kRescaleThreshold = 8.0f;  // log2 units: P stays below 2^8
constexpr uint32_t kTmemCols = 512;

template <int DP>
struct Shape {
  static constexpr int kBlocks = DP / 64;
  static constexpr uint32_t kTileBytes = kBlocks * kBlockBytes;  // a Q, K or V tile
  static constexpr int kStages = DP == 128 ? 4 : 8;
  // TMEM: S0, S1, then O0, O1.  At head_dim <= 64 P has columns of its own, so the next S is
  // formed while the exponentials of this one are taken; at 128 the columns are all in use
  // and P lies over the S it came from.
  static constexpr bool kOwnP = DP == 64;
  static constexpr uint32_t kColO = kGroups * BN;
  static constexpr uint32_t kColP = kOwnP ? kColO + kGroups * DP : 0;
  static constexpr uint32_t kStrideP = kOwnP ? BN / 2 : BN;
  static constexpr uint32_t ring = kGroups * kTileBytes;
  static constexpr uint32_t bars = ring + kStages * kTileBytes;
};

template <int KS>
struct alignas(8) Bars {
  uint64_t full[KS], empty[KS];      // ring of K and V tiles
  uint64_t clean[KS];                // padded rows of the V tile in a stage zeroed
  uint64_t q_full[kGroups];          // query rows staged (4 warps)
  uint64_t s_full[kGroups], p_half[kGroups], p_full[kGroups], o_done[kGroups];
  uint64_t s_free[kGroups];          // S is in registers (P in columns of its own)
  uint64_t drain;
  uint32_t tmem_base;
  int32_t abort;
};

struct Args {
  XaParams p;
  MapOrder ok, ov;
  int32_t n_rt;          // row tiles of an instance
  int32_t n_items;
  int32_t k_steps;       // 16-wide steps that cover head_dim
  bool wide;             // rows of out are 32-byte aligned
};

struct Item {
  int32_t inst, rt, split, key0, n_keys, n_tiles, length, active;
};

__device__ __forceinline__ Item decode_item(const Args& a, int32_t item) {
  const XaParams& p = a.p;
  Item it;
  const int32_t is = item / a.n_rt;
  it.rt = item - is * a.n_rt;
  it.inst = is / p.n_split;
  it.split = is - it.inst * p.n_split;
  it.length = xa_length(p, p.shared ? 0 : it.inst / p.groups);
  it.key0 = it.split * p.split_keys;
  const int32_t left = it.length - it.key0;
  it.n_keys = left < 0 ? 0 : (left < p.split_keys ? left : p.split_keys);
  it.n_tiles = (it.n_keys + BN - 1) / BN;
  it.active = p.rows - it.rt * kXaTileRows > BM ? 2 : 1;
  return it;
}

// Three-input maximum that keeps NaN (a NaN score makes its row NaN).
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float row_max(const uint32_t (&s)[BN]) {
  float m[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) m[i] = __uint_as_float(s[i]);
#pragma unroll
  for (int c = 8; c < BN; c += 16)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      m[i] = c + 8 + i < BN ? max3_nan(m[i], __uint_as_float(s[c + i]), __uint_as_float(s[c + 8 + i]))
                            : max3_nan(m[i], __uint_as_float(s[c + i]), __uint_as_float(s[c + i]));
  return max3_nan(max3_nan(m[0], m[1], m[2]), max3_nan(m[3], m[4], m[5]), max3_nan(m[6], m[7], m[7]));
}

template <int N>
__device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// Of each four key pairs, those whose exponentials run on the FMA pipe (the rest on the MUFU).
// One measured best: 239 us (none: 249, two: 242) at B4 H16 M2048 N4096 D128; the polynomial is
// within 7.5e-5, a fiftieth of a bf16 rounding and a sixth of an f16 one.  Head_dim 64 was not swept.
constexpr int kFmaPairs = 1;

template <int DP, bool BF16>
__global__ void __launch_bounds__(kThreads, 1)
xattn_tiles_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const Args a) {
  using L = Shape<DP>;
  constexpr int KS = L::kStages;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* ring_s = smem + L::ring;
  Bars<KS>* bars = reinterpret_cast<Bars<KS>*>(smem + L::bars);
  // read from lane 0: the compiler then knows the roles' values to be uniform
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const XaParams& p = a.p;
  volatile int32_t* abort_flag = &bars->abort;

  allow_next_kernel();
  if (threadIdx.x == 0) {
    for (int s = 0; s < KS; ++s) {
      mbar_init(&bars->full[s], 1);
      mbar_init(&bars->empty[s], 1);
      mbar_init(&bars->clean[s], 1);
    }
    for (int w = 0; w < kGroups; ++w) {
      mbar_init(&bars->q_full[w], 4);
      mbar_init(&bars->s_full[w], 1);
      mbar_init(&bars->p_half[w], 4);
      mbar_init(&bars->p_full[w], 4);
      mbar_init(&bars->s_free[w], 4);
      mbar_init(&bars->o_done[w], 1);
    }
    mbar_init(&bars->drain, 1);
    bars->abort = 0;
    mbar_fence_init();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(&bars->tmem_base, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, bars->tmem_base, 0);

  if (warp >= kGroups * 4) {
    regs_dec<kOtherRegs>();
    if (warp == kLoadWarp) {
      // -------------------------------------------------------------- producer
      uint32_t n_loaded = 0;
      bool ok = true;
      if (lane == 0) {
        tma_prefetch_desc(&tm_k);
        tma_prefetch_desc(&tm_v);
      }
      auto load = [&](const CUtensorMap* tm, const MapOrder& o, int32_t row, int32_t g, int32_t b) -> bool {
        const uint32_t s = n_loaded % KS, n = n_loaded / KS;
        if (n > 0 &&
            !warp_wait(&bars->empty[s], (n - 1) & 1, abort_flag, p.status, kDevTimeoutProducer, p.wait_ns))
          return false;
        if (lane == 0) {
          mbar_arrive_expect_tx(&bars->full[s], L::kTileBytes);
#pragma unroll
          for (int blk = 0; blk < L::kBlocks; ++blk)
            tma_load_4d(ring_s + s * L::kTileBytes + blk * kBlockBytes, tm, &bars->full[s], blk * 64,
                        map_coord(o, 1, row, g, b), map_coord(o, 2, row, g, b), map_coord(o, 3, row, g, b));
        }
        __syncwarp();
        ++n_loaded;
        return true;
      };
      for (int32_t item = blockIdx.x; item < a.n_items && ok; item += gridDim.x) {
        const Item it = decode_item(a, item);
        const int32_t b = p.shared ? 0 : it.inst / p.groups;
        const int32_t g = p.shared ? it.inst : it.inst - b * p.groups;
        for (int32_t j = 0; j < it.n_tiles && ok; ++j) {
          const int32_t row = it.key0 + j * BN;
          if (!load(&tm_k, a.ok, row, g, b) || !load(&tm_v, a.ov, row, g, b)) {
            ok = false;
            break;
          }
          const int32_t valid = it.key0 + it.n_keys - row;
          if (valid < BN && it.length < p.states) {
            // Padded states may hold anything (rows past the tensor's end arrive as zeros).
            const uint32_t s = (n_loaded - 1) % KS;
            if (!warp_wait(&bars->full[s], ((n_loaded - 1) / KS) & 1, abort_flag, p.status, kDevTimeoutProducer,
                           p.wait_ns)) {
              ok = false;
              break;
            }
            uint8_t* v_s = ring_s + s * L::kTileBytes;
            for (int i = valid * 8 + lane; i < BN * 8; i += 32)
#pragma unroll
              for (int blk = 0; blk < L::kBlocks; ++blk)
                reinterpret_cast<uint4*>(v_s + blk * kBlockBytes)[i] = make_uint4(0u, 0u, 0u, 0u);
            fence_proxy_async_shared();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars->clean[s]);
          }
        }
      }
      // No copy may be in flight into the shared memory of an exiting CTA.
      volatile int32_t no_abort = 0;
      for (uint32_t s = 0; s < KS; ++s) {
        const uint32_t cnt = n_loaded > s ? (n_loaded - s + KS - 1) / KS : 0;
        if (cnt > 0) mbar_wait(&bars->full[s], (cnt - 1) & 1, &no_abort, p.status, kDevTimeoutDrain);
      }
    } else if (warp == kMmaWarp) {
      // -------------------------------------------------------------- MMA issuer
      const uint32_t leader = elect_one();
      const uint32_t idesc_s = idesc_f16(BF16, false, BM, BN);
      const uint32_t idesc_o = idesc_f16(BF16, true, BM, a.k_steps * 16);
      const uint64_t q_desc = smem_desc_sw128(smem_u32(smem), 16, 1024);
      const uint64_t k_desc = smem_desc_sw128(smem_u32(ring_s), 16, 1024);
      const uint64_t v_desc = smem_desc_sw128(smem_u32(ring_s), kBlockBytes, 1024);
      uint32_t n_used = 0;                    // ring tiles consumed
      uint32_t clean_phase = 0;               // bit s: parity of stage s's next cleaned tile
      uint32_t gen[kGroups] = {0, 0};         // key tiles started per warpgroup
      uint32_t q_gen[kGroups] = {0, 0};
      bool ok = true, issued = false;
      auto wait = [&](uint64_t* bar, uint32_t phase) -> bool {
        return warp_wait(bar, phase & 1, abort_flag, p.status, kDevTimeoutMma, p.wait_ns);
      };
      // S_w = q_w k^T from ring stage s into the columns of the previous P_w.  The product that
      // reads that P was issued before by this warp, and products execute in issue order.
      auto issue_s = [&](int w, uint32_t s) {
        const uint64_t qd = q_desc + ((w * L::kTileBytes) >> 4), kd = k_desc + ((s * L::kTileBytes) >> 4);
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk) {
          const uint32_t off = ((kk >> 2) * kBlockBytes + (kk & 3) * 32) >> 4;
          if (kk < a.k_steps) mma_ss_warp(leader, tmem + w * BN, qd + off, kd + off, idesc_s, kk > 0 ? 1u : 0u);
        }
        mma_commit_warp(leader, &bars->s_full[w]);
        ++gen[w];
        issued = true;
      };
      for (int32_t item = blockIdx.x; item < a.n_items && ok; item += gridDim.x) {
        const Item it = decode_item(a, item);
        if (it.n_tiles == 0) continue;
        if (!wait(&bars->full[n_used % KS], n_used / KS)) break;
#pragma unroll
        for (int w = 0; w < kGroups; ++w) {
          if (w >= it.active || !ok) continue;
          ok = wait(&bars->q_full[w], q_gen[w]);
          ++q_gen[w];
          if (ok) issue_s(w, n_used % KS);
        }
        if (!ok) break;
        mma_commit_warp(leader, &bars->empty[n_used % KS]);
        for (int32_t j = 0; j < it.n_tiles && ok; ++j) {
          const uint32_t sv = (n_used + 1) % KS, sk = (n_used + 2) % KS;
          const bool more = j + 1 < it.n_tiles;
          const uint64_t vd = v_desc + ((sv * L::kTileBytes) >> 4);
          // S of the next tile for warpgroup w.
          auto next_s = [&](int w) {
            if (!more || w >= it.active || !ok) return;
            if (w == 0) ok = wait(&bars->full[sk], (n_used + 2) / KS);
            if (ok && L::kOwnP) ok = wait(&bars->s_free[w], gen[w] - 1);
            if (!ok) return;
            tc_fence_after();
            issue_s(w, sk);
            if (w == it.active - 1) mma_commit_warp(leader, &bars->empty[sk]);
          };
#pragma unroll
          for (int w = 0; w < kGroups; ++w) {
            if (w >= it.active || !ok) continue;
            if (L::kOwnP) next_s(w);
            if (w == 0 && ok) {
              ok = wait(&bars->full[sv], (n_used + 1) / KS);
              if (ok && it.n_keys - j * BN < BN && it.length < p.states) {
                ok = wait(&bars->clean[sv], clean_phase >> sv);
                clean_phase ^= 1u << sv;
              }
            }
            const uint32_t tile = gen[w] - (L::kOwnP && more ? 2 : 1);  // of this warpgroup, whose P comes next
            // Over S, P's first half is multiplied while the second half's exponentials are taken.
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              if (ok && (half == 0 || !L::kOwnP))
                ok = wait(half == 0 && !L::kOwnP ? &bars->p_half[w] : &bars->p_full[w], tile);
              if (!ok) continue;
              tc_fence_after();
#pragma unroll
              for (int kk = half * (BN / 32); kk < (half + 1) * (BN / 32); ++kk)
                mma_ts_warp(leader, tmem + L::kColO + w * DP, tmem + L::kColP + w * L::kStrideP + kk * 8,
                            vd + ((kk * 2048) >> 4), idesc_o, (j > 0 || kk > 0) ? 1u : 0u);
            }
            if (!ok) continue;
            mma_commit_warp(leader, &bars->o_done[w]);
            if (w == it.active - 1) mma_commit_warp(leader, &bars->empty[sv]);
            if (!L::kOwnP) next_s(w);
          }
          n_used += 2;
        }
      }
      if (issued) {
        mma_commit_warp(leader, &bars->drain);
        volatile int32_t no_abort = 0;
        mbar_wait(&bars->drain, 0, &no_abort, p.status, kDevTimeoutDrain);
      }
    }
  } else {
    // -------------------------------------------------------------- softmax warpgroups
    regs_inc<kSoftmaxRegs>();
    const int w = warp >> 2;
    const int row = threadIdx.x & 127;
    const uint32_t lane_base = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t s_addr = lane_base + w * BN, o_addr = lane_base + L::kColO + w * DP;
    const uint32_t p_addr = lane_base + L::kColP + w * L::kStrideP;
    const float scale_log2 = p.scale * kLog2e;  // > 0 (checked on the host)
    uint8_t* q_s = smem + w * L::kTileBytes;
    uint32_t gen = 0;
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t phase) -> bool {
      return warp_wait(bar, phase & 1, abort_flag, p.status, kDevTimeoutSoftmax, p.wait_ns);
    };
    // This thread's query row of an item into the swizzled tile; columns past head_dim are zero.
    auto stage_query = [&](const Item& it) {
      const int32_t r = it.rt * kXaTileRows + w * BM + row;
      const uint4* src = nullptr;
      if (r < p.rows) {
        const XaRow x = xa_row(p, it.inst, r);
        src = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.q) + x.b * p.qs[0] + x.h * p.qs[1] +
                                             x.m * p.qs[2]);
      }
#pragma unroll
      for (int c = 0; c < DP / 8; ++c) {
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (src != nullptr && c * 8 < p.head_dim) v = __ldg(src + c);
        reinterpret_cast<uint4*>(q_s + (c >> 3) * kBlockBytes + row * 128)[(c & 7) ^ (row & 7)] = v;
      }
      fence_proxy_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->q_full[w]);
    };
    // The next item with keys whose rows reach this warpgroup.
    auto next_item = [&](int32_t from) -> int32_t {
      for (int32_t i = from; i < a.n_items; i += gridDim.x) {
        const Item it = decode_item(a, i);
        if (it.n_tiles > 0 && it.active > w) return i;
      }
      return a.n_items;
    };
    const int32_t first = next_item(blockIdx.x);
    if (first < a.n_items) stage_query(decode_item(a, first));
    for (int32_t item = blockIdx.x; item < a.n_items && ok; item += gridDim.x) {
      const Item it = decode_item(a, item);
      if (it.active <= w) continue;
      float m = -INFINITY;                    // running maximum, log2 units
      float2 sum = make_float2(0.f, 0.f);
      for (int32_t j = 0; j < it.n_tiles; ++j) {
        if (!wait(&bars->s_full[w], gen)) {
          ok = false;
          break;
        }
        tc_fence_after();
        uint32_t s[BN];
#pragma unroll
        for (int c = 0; c < BN / 16; ++c) tmem_ld16(s_addr + c * 16, *reinterpret_cast<uint32_t(*)[16]>(s + 16 * c));
        tmem_wait_ld();
#pragma unroll
        for (int c = 0; c < BN / 16; ++c) reg_fence16(*reinterpret_cast<uint32_t(*)[16]>(s + 16 * c));
        if (L::kOwnP) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars->s_free[w]);
        }
        const int32_t valid = it.n_keys - j * BN;
        if (valid < BN) {
#pragma unroll
          for (int c = 0; c < BN; ++c)
            if (c >= valid) s[c] = 0xff800000u;  // -inf, whatever a padded state gave
        }
        const float mx = row_max(s) * scale_log2;
        // With P apart the last O += P v need not be done when S is: P's columns and O wait for it.
        if (L::kOwnP && j > 0) {
          if (!wait(&bars->o_done[w], gen - 1)) {
            ok = false;
            break;
          }
          tc_fence_after();
        }
        if (j == 0) {
          m = mx;
        } else {
          const bool need = !(mx <= m + kRescaleThreshold);
          if (__any_sync(0xffffffffu, need)) {
            // O is at rest: without columns for P, S of this tile was issued after the previous
            // O += P v and its barrier covers both.
            const float f = need ? fast_exp2(m - mx) : 1.f;
            for (int c = 0; c < a.k_steps; ++c) {
              uint32_t r[16];
              tmem_ld16(o_addr + c * 16, r);
              tmem_wait_ld();
              reg_fence16(r);
#pragma unroll
              for (int e = 0; e < 16; ++e) r[e] = __float_as_uint(__uint_as_float(r[e]) * f);
              tmem_st16(o_addr + c * 16, r);
            }
            sum = mul2(sum, make_float2(f, f));
            if (need) m = mx;
          }
        }
        // A row whose scores so far are all -inf keeps 0 as its reference (no inf - inf).
        const float ref = m == -INFINITY ? 0.f : m;
        const float2 c2 = make_float2(scale_log2, scale_log2), nm2 = make_float2(-ref, -ref);
#pragma unroll
        for (int c = 0; c < BN / 32; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float2 sv = make_float2(__uint_as_float(s[c * 32 + 2 * e]), __uint_as_float(s[c * 32 + 2 * e + 1]));
            const float2 x = fma2(sv, c2, nm2);
            const float2 e2 = (e & 3) < kFmaPairs ? exp2_fma(x) : make_float2(fast_exp2(x.x), fast_exp2(x.y));
            sum = add2(sum, e2);
            pk[e] = pack2<BF16>(e2.x, e2.y);
          }
          tmem_st16(p_addr + c * 16, pk);
          if (!L::kOwnP && c == BN / 64 - 1) {  // half of P: its product may start
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars->p_half[w]);
          }
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->p_full[w]);
        ++gen;
      }
      if (!ok) break;
      // The query tile is free (the item's last S is done): the next item's rows go in
      // while the last product runs.
      if (it.n_tiles > 0) {
        const int32_t next = next_item(item + gridDim.x);
        if (next < a.n_items) stage_query(decode_item(a, next));
        if (!wait(&bars->o_done[w], gen - 1)) {
          ok = false;
          break;
        }
        tc_fence_after();
      }
      const int32_t r = it.rt * kXaTileRows + w * BM + row;
      // A score of +inf makes its row NaN, as inf - inf does in a softmax.  The sum alone need not
      // say so: exp2_fma's clamp takes a NaN for the least exponent.
      const float l = m == INFINITY ? __int_as_float(0x7fffffff) : sum.x + sum.y;
      // No state, or every score -inf: zeros (exp2_fma leaves 2^-126 where a score is -inf).
      const bool none = m == -INFINITY;
      const float inv = none ? 0.f : 1.f / l;
      XaRow x = {0, 0, 0};
      int64_t lin = 0;
      if (r < p.rows) {
        x = xa_row(p, it.inst, r);
        lin = xa_linear(p, x);
      }
      const bool split = p.part_o != nullptr;
      const int64_t slot = static_cast<int64_t>(p.part_first + it.split) * p.rows_total + lin;
      for (int c = 0; c < a.k_steps; ++c) {
        uint32_t o[16];
        if (it.n_tiles > 0) {
          tmem_ld16(o_addr + c * 16, o);
          tmem_wait_ld();
          reg_fence16(o);
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) o[e] = 0u;
        }
        float v[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = none ? 0.f : __uint_as_float(o[e]) * inv;
        if (r < p.rows)  // a lane past the instance's rows only takes part in the TMEM loads
          store16<BF16>(v, static_cast<uint16_t*>(p.out) + x.b * p.os[0] + x.h * p.os[1] + x.m * p.os[2],
                        split ? p.part_o + slot * p.head_dim : nullptr, a.wide, c * 16, p.head_dim);
        __syncwarp();
      }
      tc_fence_before();
      if (r < p.rows) {
        const float lse2 = none ? -INFINITY : m + log2f(l);
        if (split)
          p.part_lse[slot] = lse2;
        else if (p.lse != nullptr)
          p.lse[lin] = lse2 * kLn2;
      }
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

template <int DP, bool BF16>
int32_t launch(const CUtensorMap& mk, const CUtensorMap& mv, const Args& a, int64_t grid, cudaStream_t stream,
               bool overlap) {
  auto kernel = xattn_tiles_kernel<DP, BF16>;
  constexpr int smem = Shape<DP>::bars + sizeof(Bars<Shape<DP>::kStages>) + 1024;
  static_assert(smem <= 227 * 1024, "shared memory of a CTA");
  static std::atomic<uint64_t> done{0};
  if (!allow_smem(kernel, smem, done)) return 6;
  return launch_kernel(kernel, dim3(static_cast<unsigned>(grid)), kThreads, smem, stream, overlap, mk, mv, a) ? 0 : 6;
}

}  // namespace

int32_t launch_xattn_tiles(const XaParams& p, cudaStream_t stream, int sm_count, bool overlap) {
  Args a;
  a.p = p;
  a.n_rt = (p.rows + kXaTileRows - 1) / kXaTileRows;
  const int64_t items = static_cast<int64_t>(a.n_rt) * p.instances * p.n_split;
  if (items > (1 << 30)) return 8;
  a.n_items = static_cast<int32_t>(items);
  a.k_steps = (p.head_dim + 15) / 16;
  a.wide = p.head_dim % 16 == 0 && reinterpret_cast<uintptr_t>(p.out) % 32 == 0 && p.os[0] % 16 == 0 &&
           p.os[1] % 16 == 0 && p.os[2] % 16 == 0;
  SlaParams t{};
  t.batch = p.shared ? 1 : p.batch;
  t.heads = p.groups;
  t.seq = p.states;
  t.head_dim = p.head_dim;
  t.dtype = p.dtype;
  const int64_t ks[4] = {p.ks[0], p.ks[1], p.ks[2], 1}, vs[4] = {p.vs[0], p.vs[1], p.vs[2], 1};
  CUtensorMap mk, mv;
  if (!make_map(&mk, &a.ok, p.k, ks, t, BN) || !make_map(&mv, &a.ov, p.v, vs, t, BN)) return 4;
  const int64_t grid = items < sm_count ? items : sm_count;
  if (p.head_dim <= 64)
    return p.dtype == 2 ? launch<64, true>(mk, mv, a, grid, stream, overlap)
                        : launch<64, false>(mk, mv, a, grid, stream, overlap);
  return p.dtype == 2 ? launch<128, true>(mk, mv, a, grid, stream, overlap)
                      : launch<128, false>(mk, mv, a, grid, stream, overlap);
}

}  // namespace intp
