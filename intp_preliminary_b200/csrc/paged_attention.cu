// paged_attention.cu - attention of few new tokens over a paged cache of 16-bit keys and values
// (sm_100a), the whole sequence or a sliding window with a few first states.
//
// Reading the states bounds this: the query heads of a key head (and a sequence's few new tokens)
// share each state, 16 rows at most to a pass, so a state of 4 D bytes carries at most 64 D
// multiply-adds.  What counts is bytes in flight on every SM and few instructions a byte.
// A warp streams slices of 16 keys through its own cp.async ring; every row of a slice is looked
// up in the page table by one lane, a step ahead of the copy, so pages may be of any size.  The
// products are 16 x 8 x 16 matrix instructions with the states as the 16-high operand,
//   S^T = k q^T (16 keys x 8 rows),   O^T += v^T P^T (16 columns x 8 rows),
// the probabilities two 16-bit numbers each, so that only the result's own rounding remains.
// The reference of the exponentials moves only when a score passes it by 2^8.
// The warps of a CTA join through shared memory, the CTAs of a cluster (each with its share of the
// sequence's actual length) through distributed shared memory, in a fixed order: results repeat.
//
// Row r of a sequence and key head is query head r % (H / G) of token r / (H / G), so that the rows
// of a tile stand at neighbouring positions.
#include <cooperative_groups.h>
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstring>
#include "../../include/intp_b200.h"
#include "row_mma.cuh"
#include "xattn_common.cuh"
#include "xattn_internal.h"

namespace intp {
namespace {

constexpr int kStep = 16;                  // keys of a slice
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRescale = 8.f;            // log2 units a score may pass its reference by

struct PagedParams {
  int32_t batch, heads, groups, queries, head_dim, per_group;
  int32_t pages, page_size;
  int32_t capacity;                        // states that a row of the page table has room for
  int32_t rows, n_rt;                      // rows of a sequence and key head, tiles of them
  int32_t window, sinks;                   // window 0: none
  float scale;
  const void* q; int64_t qs[3];            // sequence, head, token
  const void* k; int64_t ks[3];            // page, head, state
  const void* v; int64_t vs[3];
  void* out; int64_t os[3];
  const int32_t* table; int64_t table_stride;
  const int32_t* start; const int32_t* counts;
};

template <int DP>
struct Shape {
  static constexpr int kChunks = DP * 2 / 16;
  static constexpr int kSliceBytes = kStep * DP * 2;       // K or V of a slice
  static constexpr int kStages = DP == 128 ? 3 : 6;
  static constexpr int kWarpRing = kStages * 2 * kSliceBytes;
};

// What a tile of rows sees of its sequence.
struct View {
  int32_t first_pos, last_pos;             // of the tile's tokens that count
  int32_t end, low, sink_end;              // states [0, sink_end) and [low, end)
  int32_t sink_slices, low_slice, n_slices;
  __device__ __forceinline__ int32_t slice(int32_t i) const { return i < sink_slices ? i : i - sink_slices + low_slice; }
};

template <int kTile>
__device__ __forceinline__ View tile_view(const PagedParams& p, int32_t b, int32_t rt) {
  View x;
  const int32_t m0 = rt * kTile / p.per_group;
  int32_t m1 = (rt * kTile + kTile - 1) / p.per_group;
  int32_t count = p.queries;
  if (p.counts != nullptr) count = min(max(p.counts[b], 0), count);
  m1 = min(m1, count - 1);
  // Positions past 2^30 are behind every table, those below -2^30 before it for any row.
  const int32_t start = min(max(p.start[b], -(1 << 30)), 1 << 30);
  x.first_pos = min(start + m0, 1 << 30);
  x.last_pos = min(start + m1, 1 << 30);
  x.end = m1 < m0 ? 0 : min(max(x.last_pos, -1), p.capacity - 1) + 1;
  x.low = p.window > 0 ? max(x.first_pos - p.window + 1, 0) : 0;
  x.sink_end = p.window > 0 ? min(p.sinks, x.end) : 0;
  x.sink_slices = (x.sink_end + kStep - 1) / kStep;
  x.low_slice = max(x.low / kStep, x.sink_slices);
  x.n_slices = x.sink_slices + max((x.end + kStep - 1) / kStep - x.low_slice, 0);
  return x;
}

// NT: tiles of 8 query rows.  kWarps warps a CTA, a cluster of any size.
template <int DP, bool BF16, int NT, int kWarps>
__global__ void __launch_bounds__(kWarps * 32)
paged_attention_kernel(const PagedParams p) {
  namespace cg = cooperative_groups;
  using L = Shape<DP>;
  constexpr int CH = L::kChunks, NS = L::kStages;
  constexpr int kTile = 8 * NT;
  constexpr int kJoinStride = DP + 4;       // floats
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float m_s[kWarps][kTile], l_s[kWarps][kTile];
  __shared__ float top_s[kTile], total_s[kTile];
  __shared__ uint32_t seen_s[kWarps][NS];   // which keys of a ring's slice are read
  const cg::cluster_group cluster = cg::this_cluster();
  const int32_t n_ranks = static_cast<int32_t>(cluster.num_blocks()), rank = static_cast<int32_t>(cluster.block_rank());
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;    // fragment row and column pair

  const int32_t item = blockIdx.x / n_ranks;
  const int32_t bg = item / p.n_rt, rt = item - bg * p.n_rt;
  const int32_t b = bg / p.groups, grp = bg - b * p.groups;
  const int32_t D = p.head_dim;
  const View view = tile_view<kTile>(p, b, rt);
  // This CTA's share of the slices; warps take them in turn.
  const int32_t s0 = static_cast<int32_t>(static_cast<int64_t>(view.n_slices) * rank / n_ranks);
  const int32_t s1 = static_cast<int32_t>(static_cast<int64_t>(view.n_slices) * (rank + 1) / n_ranks);
  const int32_t mine = s1 - s0 > warp ? (s1 - s0 - warp + kWarps - 1) / kWarps : 0;
  const uint32_t ring = smem_u32(smem) + warp * NS * 2 * L::kSliceBytes;

  // Lanes 0-15 look up the slice's keys for K, 16-31 for V.
  const int32_t* table = p.table + b * p.table_stride;
  const bool for_v = lane >= 16;
  const uint8_t* base = static_cast<const uint8_t*>(for_v ? p.v : p.k) + grp * (for_v ? p.vs[1] : p.ks[1]) * 2;
  const int64_t page_bytes = (for_v ? p.vs[0] : p.ks[0]) * 2, row_bytes = (for_v ? p.vs[2] : p.ks[2]) * 2;
  int32_t looked = 0, next_page = -1, next_row = 0;
  auto look_up = [&]() {                    // the next slice's pages: used a step later
    next_page = -1;
    if (looked < mine) {
      const int32_t key = view.slice(s0 + looked * kWarps + warp) * kStep + (lane & 15);
      if (key < view.end && (key >= view.low || key < view.sink_end)) {
        const uint32_t index = static_cast<uint32_t>(key) / static_cast<uint32_t>(p.page_size);
        next_page = __ldg(table + index);
        next_row = key - static_cast<int32_t>(index) * p.page_size;
      }
    }
    ++looked;
  };
  const int cr = lane / CH, cc = lane % CH; // this lane copies chunk cc of rows cr, cr + 32 / CH, ...
  const bool chunk_read = cc * 8 < D;
  const bool chunk_used = cc * 8 < ((D + 15) & ~15);  // columns past D that the products read are zero
  int32_t issued = 0;
  auto issue = [&]() {
    if (issued < mine) {
      const bool there = next_page >= 0 && next_page < p.pages;
      const uint8_t* row = base + (there ? next_page * page_bytes + next_row * row_bytes : 0);
      const uint32_t seen = __ballot_sync(0xffffffffu, there) & 0xffffu;
      const int slot = issued % NS;
      if (lane == 0) seen_s[warp][slot] = seen;
      const uint32_t dst = ring + slot * 2 * L::kSliceBytes;
      const uint64_t bits = reinterpret_cast<uint64_t>(row);
      look_up();
#pragma unroll
      for (int u = 0; u < kStep * CH / 32; ++u) {
        const int r = cr + u * (32 / CH);
        const uint64_t ks = __shfl_sync(0xffffffffu, bits, r), vs = __shfl_sync(0xffffffffu, bits, 16 + r);
        const bool read = chunk_read && (seen >> r & 1u);
        const uint32_t to = dst + chunk_offset<CH>(r, cc);
        if (chunk_used) {
          cp_async16(to, read ? reinterpret_cast<const uint8_t*>(ks) + cc * 16 : static_cast<const uint8_t*>(p.q), read);
          cp_async16(to + L::kSliceBytes, read ? reinterpret_cast<const uint8_t*>(vs) + cc * 16 : static_cast<const uint8_t*>(p.q),
                     read);
        }
      }
    }
    ++issued;
    cp_async_commit();
  };
  look_up();
#pragma unroll
  for (int i = 0; i < NS - 1; ++i) issue();

  // Query fragments (rows 8 n + g as columns of q^T) and the positions of rows 8 n + 2 t, + 1.
  const int32_t row0 = rt * kTile;
  const int32_t n_rows = min(p.rows - row0, kTile);
  uint32_t qb[NT][DP / 16][2];
  int32_t pos[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int32_t r = row0 + 8 * n + g;
    const uint16_t* src = nullptr;
    if (r < p.rows) {
      const int32_t m = r / p.per_group, h = grp * p.per_group + (r - m * p.per_group);
      src = static_cast<const uint16_t*>(p.q) + b * p.qs[0] + h * p.qs[1] + m * p.qs[2];
    }
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) {
      const int d0 = kk * 16 + 2 * t, d1 = d0 + 8;
      qb[n][kk][0] = src != nullptr && d0 < D ? *reinterpret_cast<const uint32_t*>(src + d0) : 0u;
      qb[n][kk][1] = src != nullptr && d1 < D ? *reinterpret_cast<const uint32_t*>(src + d1) : 0u;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
      pos[n][h] = view.first_pos + (row0 + 8 * n + 2 * t + h) / p.per_group - row0 / p.per_group;
  }
  const float score_scale = p.scale * kLog2e;

  float o[NT][DP / 16][4];
  float m[NT][2], l[NT][2];                 // rows 8 n + 2 t + h: running reference, this lane's part of the sum
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int c = 0; c < DP / 16; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[n][c][e] = 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      m[n][h] = -INFINITY;
      l[n][h] = 0.f;
    }
  }
  const int mi = lane >> 3, mr = lane & 7;
  const bool one_token = view.first_pos == view.last_pos;

  for (int32_t i = 0; i < mine; ++i) {
    cp_async_wait<NS - 2>();
    __syncwarp();
    const uint32_t k_s = ring + (i % NS) * 2 * L::kSliceBytes, v_s = k_s + L::kSliceBytes;
    const uint32_t seen = seen_s[warp][i % NS];
    const int32_t k0 = view.slice(s0 + i * kWarps + warp) * kStep;
    float s[NT][4];                         // rows 2t, 2t+1 (e & 1), keys g, g + 8 (e >> 1)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) {
      if (kk * 16 >= D) break;
      uint32_t r[4];                        // keys 0-7 and 8-15 of chunk 2 kk, then of 2 kk + 1
      ldmatrix4(k_s + chunk_offset<CH>(mr + ((mi & 1) << 3), 2 * kk + (mi >> 1)), r);
#pragma unroll
      for (int n = 0; n < NT; ++n) mma16816<BF16>(s[n], r[0], r[1], r[2], r[3], qb[n][kk][0], qb[n][kk][1]);
    }
    // Whether rows of the tile differ in what they see of the slice.
    const bool mixed = !one_token && (k0 + kStep - 1 > view.first_pos ||
                                      (p.window > 0 && k0 <= view.last_pos - p.window && k0 + kStep > p.sinks));
    bool grow = false;
#pragma unroll
    for (int kh = 0; kh < 2; ++kh) {
      const int32_t key = k0 + kh * 8 + g;
      const bool there = seen >> (kh * 8 + g) & 1u;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float& x = s[n][2 * kh + h];
          x *= score_scale;
          bool hidden = !there;
          if (mixed)
            hidden = hidden || key > pos[n][h] || (p.window > 0 && key <= pos[n][h] - p.window && key >= p.sinks);
          if (hidden) x = -INFINITY;
          // a NaN score counts as growth: it has to reach the reference
          grow = grow || !(x <= m[n][h] + kRescale);
        }
    }
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float fo[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float top = keys_max(max_nan(m[n][h], max_nan(s[n][h], s[n][2 + h])));
          fo[h] = top == -INFINITY ? 1.f : fast_exp2(m[n][h] - top);
          l[n][h] *= fo[h];
          m[n][h] = top;
        }
#pragma unroll
        for (int c = 0; c < DP / 16; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[n][c][e] *= fo[e & 1];
      }
    }
    uint32_t pb[NT][2], pl[NT][2];          // P^T as the 8-wide operand: keys 2t, 2t+1 of each 8, row g; what 16 bits leave out
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      // A row without a score above -inf keeps 0 as its reference.
      const float ref[2] = {m[n][0] == -INFINITY ? 0.f : m[n][0], m[n][1] == -INFINITY ? 0.f : m[n][1]};
#pragma unroll
      for (int kh = 0; kh < 2; ++kh) {
        float pr[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          pr[h] = fast_exp2(s[n][2 * kh + h] - ref[h]);
          l[n][h] += pr[h];
        }
        const uint32_t high = pack2<BF16>(pr[0], pr[1]);
        pb[n][kh] = transpose8(high);
        const float2 f = unpack2<BF16>(high);
        pl[n][kh] = transpose8(pack2<BF16>(pr[0] - f.x, pr[1] - f.y));
      }
    }
    bool apart = false;
    if (mixed) {
      // A state that some rows do not see may hold infinities or NaN, which zero probabilities would
      // let through: such a slice goes token by token.
      bool odd = false;
#pragma unroll
      for (int c = 0; c < CH; c += 2) {
        if (c * 8 >= D) break;
        uint32_t r[4];
        ldmatrix4_trans(v_s + chunk_offset<CH>(mr + ((mi >> 1) << 3), c + (mi & 1)), r);
#pragma unroll
        for (int e = 0; e < 4; ++e) odd = odd || not_finite2<BF16>(r[e]);
      }
      apart = __any_sync(0xffffffffu, odd);
    }
    if (!apart) {
#pragma unroll
      for (int c = 0; c < CH; c += 2) {
        if (c * 8 >= D) break;
        uint32_t r[4];                      // chunk c and c + 1 of keys 0-7, then of 8-15
        ldmatrix4_trans(v_s + chunk_offset<CH>(mr + ((mi >> 1) << 3), c + (mi & 1)), r);
#pragma unroll
        for (int n = 0; n < NT; ++n) mma16816<BF16>(o[n][c / 2], r[0], r[1], r[2], r[3], pb[n][0], pb[n][1]);
        // the low parts may be zero or negative: against an infinite value they would turn the
        // high parts' infinity into NaN, so they meet finite values
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = finite2<BF16>(r[e]);
#pragma unroll
        for (int n = 0; n < NT; ++n) mma16816<BF16>(o[n][c / 2], r[0], r[1], r[2], r[3], pl[n][0], pl[n][1]);
      }
    } else {
#pragma unroll 1
      for (int32_t at = view.first_pos; at <= view.last_pos; ++at) {
        uint32_t keep[2];                   // keys 2t, 2t+1 of each 8 that position `at` sees
#pragma unroll
        for (int kh = 0; kh < 2; ++kh) {
          keep[kh] = 0u;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int32_t key = k0 + kh * 8 + 2 * t + e;
            const bool sees = key <= at && (p.window == 0 || key > at - p.window || key < p.sinks);
            if (sees) keep[kh] |= 0xffffu << (16 * e);
          }
        }
#pragma unroll
        for (int c = 0; c < CH; c += 2) {
          if (c * 8 >= D) break;
          uint32_t r[4];
          ldmatrix4_trans(v_s + chunk_offset<CH>(mr + ((mi >> 1) << 3), c + (mi & 1)), r);
#pragma unroll
          for (int e = 0; e < 4; ++e) r[e] &= keep[e >> 1];
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            float x[4] = {0.f, 0.f, 0.f, 0.f};
            mma16816<BF16>(x, r[0], r[1], r[2], r[3], pb[n][0], pb[n][1]);
            mma16816<BF16>(x, finite2<BF16>(r[0]), finite2<BF16>(r[1]), finite2<BF16>(r[2]), finite2<BF16>(r[3]), pl[n][0],
                           pl[n][1]);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (pos[n][e & 1] == at) o[n][c / 2][e] += x[e];
          }
        }
      }
    }
    __syncwarp();
    issue();
  }
  cp_async_wait<0>();
  __syncthreads();  // every ring is at rest: the space takes the warps' sums

  float* join = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = 8 * n + 2 * t + h;
      const float sum = keys_sum(l[n][h]);
      if (g == 0) {
        m_s[warp][r] = m[n][h];
        l_s[warp][r] = sum;
      }
      if (r < n_rows && mine > 0) {
        float* dst = join + (warp * kTile + r) * kJoinStride;
#pragma unroll
        for (int c = 0; c < DP / 16; ++c) {
          dst[c * 16 + g] = o[n][c][h];
          dst[c * 16 + 8 + g] = o[n][c][2 + h];
        }
      }
    }
  __syncthreads();
  const bool alone = n_ranks == 1;
  auto write = [&](int32_t r, float4 acc, float total) {
    const int32_t row = row0 + r, tok = row / p.per_group, h = grp * p.per_group + (row - tok * p.per_group);
    const bool counts = p.counts == nullptr || tok < p.counts[b];
    const float inv = counts && total != 0.f ? 1.f / total : 0.f;
    if (!counts) acc = make_float4(0.f, 0.f, 0.f, 0.f);
    if (lane * 4 < D)
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + b * p.os[0] + h * p.os[1] + tok * p.os[2] + lane * 4) =
          make_uint2(pack2<BF16>(acc.x * inv, acc.y * inv), pack2<BF16>(acc.z * inv, acc.w * inv));
  };
  auto add = [](float4& acc, const float4& v, float f) {
    acc.x = fmaf(v.x, f, acc.x);
    acc.y = fmaf(v.y, f, acc.y);
    acc.z = fmaf(v.z, f, acc.z);
    acc.w = fmaf(v.w, f, acc.w);
  };
  // The warps' parts of a row, relative to their largest reference.
  for (int r = warp; r < n_rows; r += kWarps) {
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = max_nan(top, m_s[w][r]);
    float total = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (m_s[w][r] == -INFINITY) continue;
      const float f = fast_exp2(m_s[w][r] - top);
      total = fmaf(l_s[w][r], f, total);
      if (lane * 4 < D) add(acc, *reinterpret_cast<const float4*>(join + (w * kTile + r) * kJoinStride + lane * 4), f);
    }
    if (alone) {
      write(r, acc, total);
    } else {
      __syncwarp();
      if (lane * 4 < D) *reinterpret_cast<float4*>(join + r * kJoinStride + lane * 4) = acc;  // this row's first part, read above
      if (lane == 0) {
        top_s[r] = top;
        total_s[r] = total;
      }
    }
  }
  if (alone) return;
  // The CTAs' parts: each CTA joins its share of the rows.
  cluster.sync();
  for (int r = rank * kWarps + warp; r < n_rows; r += n_ranks * kWarps) {
    float top = -INFINITY;
    for (int c = 0; c < n_ranks; ++c) top = max_nan(top, *cluster.map_shared_rank(&top_s[r], c));
    float total = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c = 0; c < n_ranks; ++c) {
      const float ref = *cluster.map_shared_rank(&top_s[r], c);
      if (ref == -INFINITY) continue;
      const float f = fast_exp2(ref - top);
      total = fmaf(*cluster.map_shared_rank(&total_s[r], c), f, total);
      if (lane * 4 < D)
        add(acc, *reinterpret_cast<const float4*>(cluster.map_shared_rank(join + r * kJoinStride + lane * 4, c)), f);
    }
    write(r, acc, total);
  }
  cluster.sync();  // nobody leaves while others read its sums
}

constexpr int64_t kPlanSms = 148;
constexpr int64_t kMaxSize = int64_t(1) << 30;

// Unit stride along D, 16-byte rows, positive strides that are multiples of 16 bytes below 2^40 bytes.
bool rows_ok(const void* x, const int64_t* stride, const int64_t* extent) {
  if (reinterpret_cast<uintptr_t>(x) % 16 || stride[3] != 1) return false;
  for (int d = 0; d < 3; ++d)
    if (extent[d] > 1 && (stride[d] <= 0 || stride[d] % 8 || stride[d] >= (int64_t(1) << 39))) return false;
  return true;
}
void take(int64_t* dst, const int64_t* src, const int64_t* extent) {
  for (int d = 0; d < 3; ++d) dst[d] = extent[d] > 1 ? src[d] : 0;
}

template <int DP, bool BF16, int NT, int W>
int32_t launch(PagedParams p, cudaStream_t stream) {
  using L = Shape<DP>;
  auto kernel = paged_attention_kernel<DP, BF16, NT, W>;
  constexpr int kRing = W * L::kWarpRing, kJoin = W * 8 * NT * (DP + 4) * 4;
  constexpr int kSmem = kRing > kJoin ? kRing : kJoin;
  static_assert(kSmem <= 224 * 1024, "shared memory of a CTA");
  static std::atomic<uint64_t> done{0};
  if (!allow_smem(kernel, kSmem, done)) return INTP_ERR_LAUNCH;
  p.n_rt = (p.rows + 8 * NT - 1) / (8 * NT);
  const int64_t items = static_cast<int64_t>(p.n_rt) * p.batch * p.groups;
  int ranks = 1;
  while (ranks < 8 && items * ranks * 2 <= 2 * kPlanSms) ranks *= 2;
  if (items * ranks > INT32_MAX) return INTP_ERR_SHAPE;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = static_cast<unsigned>(ranks);
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(items * ranks));
  cfg.blockDim = dim3(W * 32);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p) == cudaSuccess ? INTP_OK : INTP_ERR_LAUNCH;
}

template <int DP, bool BF16>
int32_t launch_rows(const PagedParams& p, cudaStream_t stream) {
  return p.rows <= 8 ? launch<DP, BF16, 1, 4>(p, stream) : launch<DP, BF16, 2, 4>(p, stream);
}

intp_status run(const paged_attention_args* a, cudaStream_t stream) {
  if (!a) return INTP_ERR_ARGUMENT;
  for (int64_t n : {a->batch, a->heads, a->groups, a->queries, a->pages, a->page_size, a->table_width})
    if (n < 0 || n > kMaxSize) return INTP_ERR_SHAPE;
  if (a->heads < 1 || a->groups < 1 || a->heads % a->groups) return INTP_ERR_SHAPE;
  if (a->head_dim < 8 || a->head_dim > 128 || a->head_dim % 8) return INTP_ERR_SHAPE;
  if (a->pages < 1 || a->page_size < 1 || a->table_width < 1) return INTP_ERR_SHAPE;
  if (a->table_width * a->page_size > kMaxSize) return INTP_ERR_SHAPE;
  if (a->window < 0 || a->window > kMaxSize || a->sinks < 0 || a->sinks > kMaxSize) return INTP_ERR_SHAPE;
  // Rows of a sequence and key head, and tiles of them, are 32-bit numbers.
  if (a->heads / a->groups * std::max<int64_t>(a->queries, 1) > kMaxSize || a->batch * a->groups > kMaxSize) return INTP_ERR_SHAPE;
  if (a->dtype != INTP_F16 && a->dtype != INTP_BF16) return INTP_ERR_DTYPE;
  if (!std::isfinite(a->scale) || !(a->scale > 0.f)) return INTP_ERR_ARGUMENT;
  if (a->batch == 0 || a->queries == 0) return INTP_OK;
  if (!a->q || !a->k || !a->v || !a->out || !a->page_table || !a->start) return INTP_ERR_ARGUMENT;
  const int64_t eq[3] = {a->batch, a->heads, a->queries}, ek[3] = {a->pages, a->groups, a->page_size};
  if (!rows_ok(a->q, a->q_stride, eq) || !rows_ok(a->out, a->out_stride, eq) || !rows_ok(a->k, a->k_stride, ek) ||
      !rows_ok(a->v, a->v_stride, ek))
    return INTP_ERR_LAYOUT;
  int sms = 0;
  const int32_t device = current_device_facts(&sms);
  if (device != INTP_OK) return device;
  PagedParams p;
  std::memset(&p, 0, sizeof(p));
  p.batch = static_cast<int32_t>(a->batch);
  p.heads = static_cast<int32_t>(a->heads);
  p.groups = static_cast<int32_t>(a->groups);
  p.queries = static_cast<int32_t>(a->queries);
  p.head_dim = static_cast<int32_t>(a->head_dim);
  p.per_group = static_cast<int32_t>(a->heads / a->groups);
  p.pages = static_cast<int32_t>(a->pages);
  p.page_size = static_cast<int32_t>(a->page_size);
  p.capacity = static_cast<int32_t>(a->table_width * a->page_size);
  p.rows = p.per_group * p.queries;
  p.window = static_cast<int32_t>(a->window);
  p.sinks = static_cast<int32_t>(a->sinks);
  p.scale = a->scale;
  p.q = a->q;
  take(p.qs, a->q_stride, eq);
  p.k = a->k;
  take(p.ks, a->k_stride, ek);
  p.v = a->v;
  take(p.vs, a->v_stride, ek);
  p.out = a->out;
  take(p.os, a->out_stride, eq);
  p.table = a->page_table;
  p.table_stride = a->table_stride;
  p.start = a->start;
  p.counts = a->counts;
  if (a->dtype == INTP_BF16) return p.head_dim <= 64 ? launch_rows<64, true>(p, stream) : launch_rows<128, true>(p, stream);
  return p.head_dim <= 64 ? launch_rows<64, false>(p, stream) : launch_rows<128, false>(p, stream);
}

}  // namespace
}  // namespace intp

extern "C" intp_status paged_attention(const paged_attention_args* a, void* stream) {
  return intp::run(a, static_cast<cudaStream_t>(stream));
}
