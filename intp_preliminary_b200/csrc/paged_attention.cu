// paged_attention.cu - attention of few new tokens over a paged cache of 16-bit keys and values
// (sm_100a), the whole sequence or a sliding window with a few first states.
//
// Reading the states bounds this: the query heads of a key head (and a sequence's few new tokens)
// share each state, 16 rows at most to a pass, so a state of 4 D bytes carries at most 64 D
// multiply-adds.  What counts is bytes in flight on every SM and few instructions a byte.
// A warp streams slices of 16 keys (32 of head_dim 64 or less) through its own cp.async ring; every
// row of a slice is looked up in the page table by one lane, a step ahead of the copy, so pages may be
// of any size.  The products are 16 x 8 x 16 matrix instructions with the states as the 16-high operand,
//   S^T = k q^T (16 keys x 8 rows),   O^T += v^T P^T (16 columns x 8 rows),
// the probabilities two 16-bit numbers each, so that only the result's own rounding remains (in f16 a probability
// below 2^-32 of its row's reference counts as zero, but for its infinite values).
// The reference of the exponentials moves only when a score passes it by 2^8.
//
// Row r of a sequence and key head is query head r % (H / G) of token r / (H / G), so that the rows
// of a tile stand at neighbouring positions.
//
// Two kernels share that loop.  paged_joined_kernel gives each sequence and key head one to eight CTAs:
// their warps join through shared memory, the CTAs of a cluster through distributed shared memory, in one
// launch.  paged_parts_kernel gives every warp of the GPU the same number of slices of the whole batch,
// and paged_combine_kernel joins the parts.  Both join in a fixed order: results repeat.
//
// Measured on one B200 (calls in a CUDA graph, us; floor at the measured copy rate): B64 G8 H32 D128 over
// 4096 to 8192 states 235 (237); one sequence of 131071 90 (82); a window of 1024 and 4 first states, B48 G4
// D64 10.5 (7.7); five tokens of B17 G4 H12 D80 over 2000 to 4001 states 22.5 (9.6); two sequences of 777 4.6
// (0.1: latency).  Steps: 327, 346, 24.6, -, 8 with one cluster kernel and 64-bit places handed round; 274, 111, 23 in
// parts; 238, 99, 14.6 with places in 16-byte units (718 -> 344 instructions a slice: issue, not memory, had bound
// it) and V not clamped; 11.5 with 32-key slices at D64; 240, 90, 11.1, 29 with the next slice asked for while the first
// products run; 233 with three CTAs an SM where parts are of many items; 10.5, 27 with values that are not finite
// left to a second pass over a warp's slices, and 22.5 with all of an SM's registers for a tile of 16 rows.
// Not kept: slices' rows an odd number of chunks apart instead of permuted (copies straddle lines: batch 276
// where this form took 255), 96-column slices (D96 in parts 114 us, in 128 columns 103), two slices a ring
// and three CTAs an SM for all parts (B1 G8 of 32000 states 26.4 instead of 23.9, 16 rows 40 instead of 27),
// packed fp32 pairs for the scores and P (a tenth fewer of those instructions, 0 to 2 % slower).
#include <cooperative_groups.h>
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstring>
#include <type_traits>
#include "../../include/intp_b200.h"
#include "row_mma.cuh"
#include "xattn_common.cuh"
#include "xattn_internal.h"

namespace intp {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRescale = 8.f;            // log2 units a score may pass its reference by

struct PagedParams {
  int32_t batch, heads, groups, queries, head_dim, per_group;
  int32_t pages, page_size;
  int32_t capacity;                        // states that a row of the page table has room for
  int32_t rows, n_rt;                      // rows of a sequence and key head, tiles of them
  int32_t depth;                           // slices that a warp's ring has room for, in one launch
  int32_t window, sinks;                   // window 0: none
  float scale;
  const void* q; int64_t qs[3];            // sequence, head, token
  const void* k; const void* v;            // of the same strides
  int64_t head_stride;
  uint32_t page_units, row_units;          // strides of a page and a state in 16-byte units
  uint32_t page_magic; int32_t page_shift; // p / page_size = umulhi(4 p, magic) >> shift for p < 2^30
  void* out; int64_t os[3];
  const int32_t* table; int64_t table_stride;
  const int32_t* start; const int32_t* counts;
};

// A call in parts: every warp of the GPU takes the same number of slices of the batch, laid end to
// end (sequence, key head, slice), whatever the sequences' lengths; a part is what one warp has of
// one item (sequence and key head), in slot warp + item, which no two parts share.
struct Parts {
  float* o;                                // [slot][tile row][D], not normalised
  float2* ml;                              // [slot][tile row]: reference (log2 units) and sum
  int32_t* plan;                           // [batch + 1] slices of one key head before each sequence; then slices a warp
  bool three;                              // CTAs an SM: three, or two
};
constexpr int kPartsWarps = 4;
constexpr int kPartsCtas = 296, kPartsAll = kPartsCtas * kPartsWarps;  // two CTAs an SM, rings of kStages slices
constexpr int kThreeCtas = 444, kThreeStages = 2;         // three, rings of two
constexpr int kPartsBatch = 1024;          // sequences whose prefix sums fit beside the rings

template <int DP>
struct Shape {
  static constexpr int kChunks = DP * 2 / 16;
  static constexpr int kStep = DP > 64 ? 16 : 32;          // keys of a slice
  static constexpr int kSliceBytes = kStep * DP * 2;       // K or V of a slice
  static constexpr int kStages = DP == 32 ? 6 : 3;         // 24 KB a warp
};

// The dynamic shared memory from its first 256-byte boundary on: slices' rows lie on their own length.
constexpr int kAlign = 256;
__device__ __forceinline__ uint8_t* aligned_smem() {
  extern __shared__ __align__(16) uint8_t raw_smem[];
  return raw_smem + (kAlign - smem_u32(raw_smem) % kAlign) % kAlign;
}

// Positions are held less 2^30: start goes up to 2^31 - 1 and a row's number to 2^30.  Positions below -2^30
// are before the sequence like -2^30.
constexpr int32_t kFar = 1 << 30;

// What a tile of rows sees of its sequence.
struct View {
  int32_t first_pos, last_pos;             // of the tile's tokens that count, less kFar
  int32_t end, low, sink_end;              // states [0, sink_end) and [low, end)
  int32_t sink_slices, low_slice, n_slices;
  __device__ __forceinline__ int32_t slice(int32_t i) const { return i < sink_slices ? i : i - sink_slices + low_slice; }
};

template <int kTile, int kStep>
__device__ __forceinline__ View tile_view(const PagedParams& p, int32_t b, int32_t rt) {
  View x;
  const int32_t m0 = rt * kTile / p.per_group;
  int32_t m1 = (rt * kTile + kTile - 1) / p.per_group;
  int32_t count = p.queries;
  if (p.counts != nullptr) count = min(max(p.counts[b], 0), count);
  m1 = min(m1, count - 1);
  const int32_t start = max(p.start[b], -kFar) - kFar;
  x.first_pos = start + m0;
  x.last_pos = start + m1;
  x.end = m1 < m0 ? 0 : min(max(x.last_pos, -1 - kFar), p.capacity - 1 - kFar) + kFar + 1;
  // from 2^31 - 1 on a row is past every window's reach
  x.low = p.window > 0 ? max(min(x.first_pos, kFar - 1) + (kFar + 1 - p.window), 0) : 0;
  x.sink_end = p.window > 0 ? min(p.sinks, x.end) : 0;
  x.sink_slices = (x.sink_end + kStep - 1) / kStep;
  x.low_slice = max(x.low / kStep, x.sink_slices);
  x.n_slices = x.sink_slices + max((x.end + kStep - 1) / kStep - x.low_slice, 0);
  return x;
}

// The slices of one warp, copied into its ring in turn.  A lane looks up the place of one key, in
// 16-byte units (32 bits reach 64 GB), and hands it to the lanes that copy the key's chunks.
template <int DP, bool FULL, int NS = Shape<DP>::kStages>
struct Feed {
  using L = Shape<DP>;
  static constexpr int CH = L::kChunks, kStep = L::kStep, kRowsAStep = 32 / CH;
  static constexpr uint32_t kAll = 0xffffffffu >> (32 - kStep);
  const PagedParams& p;
  uint32_t* seen_s;                         // [NS]: which keys of a ring's slice are read
  const int32_t* table;                     // of the item's sequence
  const uint8_t *k, *v;                     // of its key head, at this lane's chunk
  uint32_t to;                              // this lane's chunk of its first row, in the ring's first slice
  int lane, cr, cc;                         // this lane copies chunk cc of rows cr, cr + 32 / CH, ...
  bool chunk_read;
  int32_t issued, slot;

  __device__ __forceinline__ Feed(const PagedParams& params, uint32_t ring, int32_t depth, uint32_t* seen) : p(params), seen_s(seen) {
    lane = threadIdx.x & 31;
    cr = lane / CH;
    cc = lane % CH;
    chunk_read = FULL || cc * 8 < p.head_dim;
    to = ring;
    // The products read columns up to a multiple of 16; those past D are never copied and stay zero.
    if (!FULL && p.head_dim % 16 != 0)
      for (int i = lane; i < depth * 2 * kStep; i += 32)
        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(ring + (i / kStep) * L::kSliceBytes +
                                                                    chunk_offset<CH>(i % kStep, p.head_dim / 8)), "r"(0) : "memory");
    issued = slot = 0;
  }
  __device__ __forceinline__ void enter(int32_t b, int32_t grp) {
    table = p.table + b * p.table_stride;
    const int64_t at = grp * p.head_stride * 2 + cc * 16;
    k = static_cast<const uint8_t*>(p.k) + at;
    v = static_cast<const uint8_t*>(p.v) + at;
  }
  __device__ __forceinline__ void page_of(int32_t key, int32_t& page, uint32_t& row) const {
    const uint32_t index = __umulhi(static_cast<uint32_t>(key) << 2, p.page_magic) >> p.page_shift;
    page = __ldg(table + index);
    row = key - index * p.page_size;
  }
  // A slice's pages; what comes of the load is used a step later.
  __device__ __forceinline__ void look_up(const View& view, int32_t slice, int32_t& page, uint32_t& row) const {
    const int32_t key = view.slice(slice) * kStep + (lane & (kStep - 1));
    page = -1;
    if (key < view.end && (key >= view.low || key < view.sink_end)) page_of(key, page, row);
  }
  __device__ __forceinline__ void copy(int32_t page, uint32_t row, const uint8_t* k_at, const uint8_t* v_at) {
    const bool there = page >= 0 && page < p.pages;
    const uint32_t place = there ? page * p.page_units + row * p.row_units : 0u;
    const uint32_t seen = __ballot_sync(0xffffffffu, there) & kAll;
    if (lane == 0) seen_s[slot] = seen;
    const uint32_t dst = to + slot * 2 * L::kSliceBytes;
    if (seen == kAll) {
#pragma unroll
      for (int u = 0; u < kStep / kRowsAStep; ++u) {
        const int r = cr + u * kRowsAStep;
        const uint64_t at = static_cast<uint64_t>(__shfl_sync(0xffffffffu, place, r)) * 16;
        const uint32_t d = dst + chunk_offset<CH>(r, cc);
        if (chunk_read) {
          cp_async16(d, k_at + at);
          cp_async16(d + L::kSliceBytes, v_at + at);
        }
      }
    } else {                                // rows that are not there are zero
#pragma unroll
      for (int u = 0; u < kStep / kRowsAStep; ++u) {
        const int r = cr + u * kRowsAStep;
        const uint64_t at = static_cast<uint64_t>(__shfl_sync(0xffffffffu, place, r)) * 16;
        const bool read = seen >> r & 1u;
        const uint32_t d = dst + chunk_offset<CH>(r, cc);
        if (chunk_read) {
          const uint8_t* none = static_cast<const uint8_t*>(p.q);
          cp_async16(d, read ? k_at + at : none, read);
          cp_async16(d + L::kSliceBytes, read ? v_at + at : none, read);
        }
      }
    }
  }
  // From the first slice on once more, when every lane has read its last one.
  __device__ __forceinline__ void restart() {
    cp_async_wait<0>();
    issued = slot = 0;
  }
  __device__ __forceinline__ void commit() {
    ++issued;
    slot = slot + 1 == NS ? 0 : slot + 1;
    cp_async_commit();
  }
};

// What a warp holds of a tile of rows: the queries, and the sums over the slices so far.
template <int DP, bool FULL, bool BF16, int NT>
struct Rows {
  static constexpr int CH = Shape<DP>::kChunks;
  uint32_t qb[NT][DP / 16][2];              // rows 8 n + g as columns of q^T
  int32_t pos[NT][2];                       // positions of rows 8 n + 2 t, + 1
  float o[NT][DP / 16][4];
  // Rows 8 n + 2 t + h: running reference, what a score may reach before it moves, what is taken from a
  // score (0 for a row without one above -inf), this lane's part of the sum.
  float m[NT][2], limit[NT][2], ref[NT][2], l[NT][2];

  __device__ __forceinline__ void enter(const PagedParams& p, const View& view, int32_t b, int32_t grp, int32_t row0) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int32_t r = row0 + 8 * n + g;
      const uint16_t* src = nullptr;
      if (r < p.rows) {
        const int32_t tok = r / p.per_group, h = grp * p.per_group + (r - tok * p.per_group);
        src = static_cast<const uint16_t*>(p.q) + b * p.qs[0] + h * p.qs[1] + tok * p.qs[2];
      }
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk) {
        const int d0 = kk * 16 + 2 * t, d1 = d0 + 8;
        qb[n][kk][0] = src != nullptr && d0 < p.head_dim ? *reinterpret_cast<const uint32_t*>(src + d0) : 0u;
        qb[n][kk][1] = src != nullptr && d1 < p.head_dim ? *reinterpret_cast<const uint32_t*>(src + d1) : 0u;
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        pos[n][h] = view.first_pos + (row0 + 8 * n + 2 * t + h) / p.per_group - row0 / p.per_group;
        m[n][h] = -INFINITY;
        limit[n][h] = -INFINITY;
        ref[n][h] = BF16 ? 0.f : -7.f;
        l[n][h] = 0.f;
      }
#pragma unroll
      for (int c = 0; c < DP / 16; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][c][e] = 0.f;
    }
  }

  // Whether a sum of this lane, of a row that counts, is NaN.
  __device__ __forceinline__ bool any_nan(const View& view) const {
    bool nan = false;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float sum = 0.f;                    // of infinities of both signs: NaN too, which costs time alone
#pragma unroll
        for (int c = 0; c < DP / 16; ++c) sum += o[n][c][h] + o[n][c][2 + h];
        nan = nan || (sum != sum && pos[n][h] <= view.last_pos);
      }
    return nan;
  }

  // One slice, keys from k0 on, of which the bits of `seen` are there.
  // `meanwhile` runs while the first products are under way.
  // A zero times an infinity is NaN: where a state that holds infinities or NaN is not seen by every row of the
  // tile, or a part of its probability is zero, a column becomes NaN that may not be.  So whatever of a warp's
  // slices end in NaN is done again, with CAREFUL: slices are looked through for such values, and those that hold
  // any go token by token, infinities and NaN against 1 for a probability above zero.
  template <bool CAREFUL, class Meanwhile>
  __device__ __forceinline__ void step(const PagedParams& p, const View& view, uint32_t k_s, int32_t k0, uint32_t seen,
                                       Meanwhile&& meanwhile) {
    constexpr float kShift = BF16 ? 0.f : 7.f;
    constexpr int kStep = Shape<DP>::kStep, KB = kStep / 16, kBlock = 16 * CH * 16;  // blocks of 16 keys, bytes of one
    constexpr uint32_t kAll = 0xffffffffu >> (32 - kStep);
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, mi = lane >> 3, mr = lane & 7;
    const int D = p.head_dim;
    // Whether 16-column block c has columns below D, which is above DP / 2 (DP 32: at least 8).
    auto inside = [&](int c) { return FULL || c * 16 < DP / 2 || c * 16 < D; };
    // Matrix addresses of chunk 0 or 1; further chunks differ in the bits that the permutation leaves apart.
    const uint32_t k_at = k_s + chunk_offset<CH>(mr + ((mi & 1) << 3), mi >> 1);
    const uint32_t v_at = k_s + Shape<DP>::kSliceBytes + chunk_offset<CH>(mr + ((mi >> 1) << 3), mi & 1);
    // Two sums of products in turn where there is one block of keys and rows: a product waits for the one before it.
    constexpr int KS = KB * NT == 1 ? 2 : 1;
    float half[4] = {0.f, 0.f, 0.f, 0.f};
    float s[KB][NT][4];                     // rows 2t, 2t+1 (e & 1), keys g, g + 8 (e >> 1)
#pragma unroll
    for (int k = 0; k < KB; ++k)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[k][n][e] = 0.f;
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) {
      if (!inside(kk)) break;
#pragma unroll
      for (int k = 0; k < KB; ++k) {
        uint32_t r[4];                      // keys 0-7 and 8-15 of chunk 2 kk, then of 2 kk + 1
        ldmatrix4((k_at + k * kBlock) ^ (kk * 32), r);
#pragma unroll
        for (int n = 0; n < NT; ++n)
          mma16816<BF16>(KS == 2 && kk % 2 == 1 ? half : s[k][n], r[0], r[1], r[2], r[3], qb[n][kk][0], qb[n][kk][1]);
      }
    }
    meanwhile();
    // Whether rows of the tile differ in what they see of the slice.
    const int32_t from = k0 - kFar;         // held like the positions
    const bool mixed = view.first_pos != view.last_pos &&
                       (from + kStep - 1 > view.first_pos ||
                        (p.window > 0 && from + p.window <= view.last_pos && k0 + kStep > p.sinks));
    const float score_scale = p.scale * kLog2e;
#pragma unroll
    for (int k = 0; k < KB; ++k)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[k][n][e] = (KS == 2 ? s[k][n][e] + half[e] : s[k][n][e]) * score_scale;
    if (mixed || seen != kAll) {
#pragma unroll
      for (int kh = 0; kh < 2 * KB; ++kh) {
        const int32_t key = from + kh * 8 + g;
        const bool there = seen >> (kh * 8 + g) & 1u, sink = k0 + kh * 8 + g < p.sinks;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            if (!there || (mixed && (key > pos[n][h] || (p.window > 0 && key + p.window <= pos[n][h] && !sink))))
              s[kh / 2][n][2 * (kh & 1) + h] = -INFINITY;
      }
    }
    bool grow = false;                      // a NaN score counts as growth: it has to reach the reference
#pragma unroll
    for (int k = 0; k < KB; ++k)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) grow = grow || !(s[k][n][e] <= limit[n][e & 1]);
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float fo[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float top = m[n][h];
#pragma unroll
          for (int k = 0; k < KB; ++k) top = max_nan(top, max_nan(s[k][n][h], s[k][n][2 + h]));
          top = keys_max(top);
          fo[h] = top == -INFINITY ? 1.f : fast_exp2(m[n][h] - top);
          l[n][h] *= fo[h];
          m[n][h] = top;
          limit[n][h] = top + kRescale;
          ref[n][h] = (top == -INFINITY ? 0.f : top) - kShift;
        }
#pragma unroll
        for (int c = 0; c < DP / 16; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[n][c][e] *= fo[e & 1];
      }
    }
    // P^T as the 8-wide operand (keys 2t, 2t+1 of each 8, row g) in two 16-bit parts: cut off, and what that leaves
    // out, rounded.  In f16 P is 2^7 times itself: the parts are multiples of 2^-24, 2^-31 of P's unit.
    uint32_t pb[NT][2 * KB], pl[NT][2 * KB];
    uint32_t above = 0u;                    // CAREFUL: which of this lane's P's are not zero
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int kh = 0; kh < 2 * KB; ++kh) {
        float pr[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          pr[h] = fast_exp2(s[kh / 2][n][2 * (kh & 1) + h] - ref[n][h]);
          l[n][h] += pr[h];
          if (CAREFUL && pr[h] != 0.f) above |= 1u << ((n * 2 * KB + kh) * 2 + h);
        }
        const uint32_t high = pack2_down<BF16>(pr[0], pr[1]);
        const float2 f = unpack2<BF16>(high);
        pb[n][kh] = transpose8(high);
        pl[n][kh] = transpose8(pack2<BF16>(pr[0] - f.x, pr[1] - f.y));
      }
    bool apart = false;
    if (CAREFUL) {
      uint32_t odd = 0u;
#pragma unroll
      for (int c = 0; c < DP / 16; ++c) {
        if (!inside(c)) break;
#pragma unroll
        for (int k = 0; k < KB; ++k) {
          uint32_t r[4];
          ldmatrix4_trans((v_at + k * kBlock) ^ (c * 32), r);
#pragma unroll
          for (int e = 0; e < 4; ++e) odd |= not_finite2<BF16>(r[e]);
        }
      }
      apart = __any_sync(0xffffffffu, odd != 0u);
    }
    if (!apart) {
#pragma unroll
      for (int c = 0; c < DP / 16; ++c) {
        if (!inside(c)) break;
#pragma unroll
        for (int k = 0; k < KB; ++k) {
          uint32_t r[4];                    // chunk 2 c and 2 c + 1 of keys 0-7, then of 8-15
          ldmatrix4_trans((v_at + k * kBlock) ^ (c * 32), r);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma16816<BF16>(o[n][c], r[0], r[1], r[2], r[3], pb[n][2 * k], pb[n][2 * k + 1]);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma16816<BF16>(o[n][c], r[0], r[1], r[2], r[3], pl[n][2 * k], pl[n][2 * k + 1]);
        }
      }
      return;
    }
    uint32_t one[NT][2 * KB];               // 1 where P is not zero, as the operand
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int kh = 0; kh < 2 * KB; ++kh) {
        const uint32_t two = above >> ((n * 2 * KB + kh) * 2), kOne = BF16 ? 0x3f80u : 0x3c00u;
        one[n][kh] = transpose8((two & 1u ? kOne : 0u) | (two & 2u ? kOne << 16 : 0u));
      }
#pragma unroll 1
    for (int32_t at = view.first_pos; at <= view.last_pos; ++at) {
      uint32_t keep[2 * KB];                // keys 2t, 2t+1 of each 8 that position `at` sees
#pragma unroll
      for (int kh = 0; kh < 2 * KB; ++kh) {
        keep[kh] = 0u;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int32_t i = kh * 8 + 2 * t + e;
          const bool sees = from + i <= at && (p.window == 0 || from + i + p.window > at || k0 + i < p.sinks);
          if (sees) keep[kh] |= 0xffffu << (16 * e);
        }
      }
#pragma unroll
      for (int c = 0; c < DP / 16; ++c) {
        if (!inside(c)) break;
#pragma unroll
        for (int k = 0; k < KB; ++k) {
          uint32_t r[4];
          ldmatrix4_trans((v_at + k * kBlock) ^ (c * 32), r);
#pragma unroll
          for (int e = 0; e < 4; ++e) r[e] &= keep[2 * k + (e >> 1)];
          uint32_t odd[4];                  // what is not finite, taken out of r
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            odd[e] = r[e] & not_finite2<BF16>(r[e]);
            r[e] ^= odd[e];
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            float x[4] = {o[n][c][0], o[n][c][1], o[n][c][2], o[n][c][3]};  // the sums' order is the first pass's
            mma16816<BF16>(x, r[0], r[1], r[2], r[3], pb[n][2 * k], pb[n][2 * k + 1]);
            mma16816<BF16>(x, r[0], r[1], r[2], r[3], pl[n][2 * k], pl[n][2 * k + 1]);
            mma16816<BF16>(x, odd[0], odd[1], odd[2], odd[3], one[n][2 * k], one[n][2 * k + 1]);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (pos[n][e & 1] == at) o[n][c][e] = x[e];
          }
        }
      }
    }
  }
};

// Sums of a row that are held relative to references of their own (one a lane, -inf where there is
// none): the largest reference, and this lane's factor and part of the sum relative to it.
struct Joint {
  float top, total, factor;
};
__device__ __forceinline__ Joint join_references(float ref, float part) {
  Joint j;
  j.top = ref;
#pragma unroll
  for (int d = 4; d > 0; d >>= 1) j.top = max_nan(j.top, __shfl_xor_sync(0xffffffffu, j.top, d));
  j.top = __shfl_sync(0xffffffffu, j.top, 0);
  j.factor = ref == -INFINITY ? 0.f : fast_exp2(ref - j.top);
  j.total = ref == -INFINITY ? 0.f : part * j.factor;
#pragma unroll
  for (int d = 4; d > 0; d >>= 1) j.total += __shfl_xor_sync(0xffffffffu, j.total, d);
  j.total = __shfl_sync(0xffffffffu, j.total, 0);
  return j;
}
__device__ __forceinline__ void add_weighted(float4& acc, const float4& v, float f) {
  acc.x = fmaf(v.x, f, acc.x);
  acc.y = fmaf(v.y, f, acc.y);
  acc.z = fmaf(v.z, f, acc.z);
  acc.w = fmaf(v.w, f, acc.w);
}

constexpr int kMostWarps = 8, kMostRanks = 8;

// NT: tiles of 8 query rows.  Two CTAs an SM of 8 rows, which short sequences' rings leave room for; with 16 rows
// their registers would not do.  One to eight warps a CTA, one to eight CTAs an item: the item's warps take
// its slices in turn, so that the first look-up needs no length.
template <int DP, bool FULL, bool BF16, int NT>
__global__ void __launch_bounds__(kMostWarps * 32, NT == 1 ? 2 : 1)
paged_joined_kernel(const PagedParams p) {
  namespace cg = cooperative_groups;
  using L = Shape<DP>;
  constexpr int NS = L::kStages;
  constexpr int kTile = 8 * NT;
  constexpr int kJoinStride = DP + 4;       // floats
  uint8_t* smem = aligned_smem();
  __shared__ float m_s[kMostWarps][kTile], l_s[kMostWarps][kTile];
  __shared__ float top_s[kTile], total_s[kTile];
  __shared__ uint32_t seen_s[kMostWarps][NS];
  const cg::cluster_group cluster = cg::this_cluster();
  const int32_t n_ranks = static_cast<int32_t>(cluster.num_blocks()), rank = static_cast<int32_t>(cluster.block_rank());
  const int32_t n_warps = blockDim.x >> 5;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;    // fragment row and column pair

  const int32_t item = blockIdx.x / n_ranks;
  const int32_t bg = item / p.n_rt, rt = item - bg * p.n_rt;
  const int32_t b = bg / p.groups, grp = bg - b * p.groups;
  const int32_t D = p.head_dim;
  const int32_t first = rank * n_warps + warp, stride = n_ranks * n_warps;
  const uint32_t ring = smem_u32(smem) + warp * p.depth * 2 * L::kSliceBytes;
  Feed<DP, FULL> feed(p, ring, p.depth, seen_s[warp]);
  feed.enter(b, grp);
  // Without a window the first slice's pages are asked for together with the length.
  int32_t next_page = -1;
  uint32_t next_row = 0;
  const int32_t first_key = first * L::kStep + (lane & (L::kStep - 1));
  if (p.window == 0 && first_key < p.capacity) feed.page_of(first_key, next_page, next_row);
  const View view = tile_view<kTile, L::kStep>(p, b, rt);
  const int32_t mine = view.n_slices > first ? (view.n_slices - first + stride - 1) / stride : 0;
  if (p.window == 0) {
    if (first_key >= view.end) next_page = -1;
  } else if (mine > 0) {
    feed.look_up(view, first, next_page, next_row);
  }
  auto issue = [&]() {
    if (feed.issued < mine) {
      const int32_t page = next_page;
      const uint32_t row = next_row;
      if (feed.issued + 1 < mine) feed.look_up(view, first + (feed.issued + 1) * stride, next_page, next_row);
      feed.copy(page, row, feed.k, feed.v);
    }
    feed.commit();
  };
#pragma unroll
  for (int i = 0; i < NS - 1; ++i) issue();
  const int32_t row0 = rt * kTile;
  const int32_t n_rows = min(p.rows - row0, kTile);
  Rows<DP, FULL, BF16, NT> rows;
  auto slices = [&](auto careful) {
    rows.enter(p, view, b, grp, row0);
    for (int32_t i = 0, at = 0; i < mine; ++i, at = at + 1 == NS ? 0 : at + 1) {
      cp_async_wait<NS - 2>();
      __syncwarp();
      // the slice before this one has been read by every lane: its place is filled again
      rows.template step<careful>(p, view, ring + at * 2 * L::kSliceBytes, view.slice(first + i * stride) * L::kStep,
                                  seen_s[warp][at], issue);
    }
  };
  slices(std::false_type{});
  if (__any_sync(0xffffffffu, rows.any_nan(view))) {
    feed.restart();
    feed.look_up(view, first, next_page, next_row);
#pragma unroll
    for (int i = 0; i < NS - 1; ++i) issue();
    slices(std::true_type{});
  }
  cp_async_wait<0>();
  __syncthreads();  // every ring is at rest: the space takes the warps' sums

  float* join = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = 8 * n + 2 * t + h;
      const float sum = keys_sum(rows.l[n][h]);
      if (g == 0) {
        m_s[warp][r] = rows.m[n][h];
        l_s[warp][r] = sum;
      }
      if (r < n_rows && mine > 0) {
        float* dst = join + (warp * kTile + r) * kJoinStride;
#pragma unroll
        for (int c = 0; c < DP / 16; ++c) {
          dst[c * 16 + g] = rows.o[n][c][h];
          dst[c * 16 + 8 + g] = rows.o[n][c][2 + h];
        }
      }
    }
  __syncthreads();
  const bool alone = n_ranks == 1;
  const int d = lane * 4;
  auto write = [&](int32_t r, float4 acc, float total) {
    const int32_t row = row0 + r, tok = row / p.per_group, h = grp * p.per_group + (row - tok * p.per_group);
    const bool counts = p.counts == nullptr || tok < p.counts[b];
    const float inv = counts && total != 0.f ? 1.f / total : 0.f;
    if (!counts) acc = make_float4(0.f, 0.f, 0.f, 0.f);
    if (d < D)
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + b * p.os[0] + h * p.os[1] + tok * p.os[2] + d) =
          make_uint2(pack2<BF16>(acc.x * inv, acc.y * inv), pack2<BF16>(acc.z * inv, acc.w * inv));
  };
  // The warps' parts of a row.
  for (int r = warp; r < n_rows; r += n_warps) {
    const bool has = lane < n_warps;
    const Joint j = join_references(has ? m_s[lane & 7][r] : -INFINITY, has ? l_s[lane & 7][r] : 0.f);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kMostWarps; ++w) {
      const float f = __shfl_sync(0xffffffffu, j.factor, w);
      if (f != 0.f && d < D) add_weighted(acc, *reinterpret_cast<const float4*>(join + (w * kTile + r) * kJoinStride + d), f);
    }
    if (alone) {
      write(r, acc, j.total);
    } else {
      __syncwarp();
      if (d < D) *reinterpret_cast<float4*>(join + r * kJoinStride + d) = acc;  // this row's first part, read above
      if (lane == 0) {
        top_s[r] = j.top;
        total_s[r] = j.total;
      }
    }
  }
  if (alone) return;
  // The CTAs' parts: each CTA joins its share of the rows.
  cluster.sync();
  for (int r = first; r < n_rows; r += stride) {
    const bool has = lane < n_ranks;
    const Joint j = join_references(has ? *cluster.map_shared_rank(&top_s[r], lane) : -INFINITY,
                                    has ? *cluster.map_shared_rank(&total_s[r], lane) : 0.f);
    float4 v[kMostRanks];
#pragma unroll
    for (int c = 0; c < kMostRanks; ++c)
      if (c < n_ranks && d < D) v[c] = *reinterpret_cast<const float4*>(cluster.map_shared_rank(join + r * kJoinStride + d, c));
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int c = 0; c < kMostRanks; ++c) {
      const float f = __shfl_sync(0xffffffffu, j.factor, c);
      if (f != 0.f && d < D) add_weighted(acc, v[c], f);
    }
    write(r, acc, j.total);
  }
  cluster.sync();  // nobody leaves while others read its sums
}

// Every warp on its own, one wave of kCtas CTAs with rings of NS slices.
template <int DP, bool FULL, bool BF16, int NT, int kCtas, int NS>
__global__ void __launch_bounds__(kPartsWarps * 32, kCtas / 148)
paged_parts_kernel(const PagedParams p, const Parts parts) {
  using L = Shape<DP>;
  constexpr int kWarps = kPartsWarps, kTile = 8 * NT, kThreads = kWarps * 32, kAll = kCtas * kWarps;
  uint8_t* smem = aligned_smem();
  __shared__ uint32_t seen_s[kWarps][NS];
  __shared__ int32_t sum_s[kWarps];
  int32_t* before = reinterpret_cast<int32_t*>(smem + kWarps * NS * 2 * L::kSliceBytes);  // [batch + 1]
  allow_next_kernel();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // Prefix sums of the sequences' slices: a run of sequences a thread, the runs' sums across the CTA.
  const int32_t run = (p.batch + kThreads - 1) / kThreads, first = threadIdx.x * run;
  int32_t sum = 0;
  for (int32_t b = first; b < min(first + run, p.batch); ++b) {
    before[b] = sum;
    sum += tile_view<kTile, L::kStep>(p, b, 0).n_slices;
  }
  int32_t scan = sum;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int32_t x = __shfl_up_sync(0xffffffffu, scan, d);
    if (lane >= d) scan += x;
  }
  if (lane == 31) sum_s[warp] = scan;
  __syncthreads();
  int32_t base = scan - sum, all = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) base += sum_s[w];
    all += sum_s[w];
  }
  for (int32_t b = first; b < min(first + run, p.batch); ++b) before[b] += base;
  if (threadIdx.x == 0) before[p.batch] = all;
  __syncthreads();
  const int32_t total = all * p.groups;
  const int32_t per = max((total + kAll - 1) / kAll, 1);  // at least one slice; two: 6 items of 777 states 7.6 us instead of 6.6
  if (blockIdx.x == 0) {
    for (int32_t b = threadIdx.x; b <= p.batch; b += kThreads) parts.plan[b] = before[b];
    if (threadIdx.x == 0) parts.plan[p.batch + 1] = per;
  }
  // Consecutive warps' parts on different SMs, so that few parts find many.
  const int32_t me = warp * kCtas + blockIdx.x;
  if (static_cast<int64_t>(me) * per >= total) return;
  const int32_t f0 = me * per, mine = min(per, total - f0);
  int32_t lo = 0, hi = p.batch;             // the last sequence that starts at f0 or before
  while (hi - lo > 1) {
    const int32_t mid = (lo + hi) >> 1;
    if (before[mid] * p.groups <= f0) lo = mid; else hi = mid;
  }
  struct Cursor {
    int32_t b, grp, slice, n;
  };
  Cursor begin;
  begin.b = lo;
  begin.n = before[lo + 1] - before[lo];
  const int32_t rest = f0 - before[lo] * p.groups;
  begin.grp = rest / begin.n;
  begin.slice = rest - begin.grp * begin.n;
  // To the next slice; true where that is another item's.
  auto advance = [&](Cursor& c, View& v) {
    if (++c.slice < c.n) return false;
    c.slice = 0;
    if (++c.grp == p.groups) {
      c.grp = 0;
      do {
        ++c.b;
        c.n = before[c.b + 1] - before[c.b];
      } while (c.n == 0);
      v = tile_view<kTile, L::kStep>(p, c.b, 0);
    }
    return true;
  };
  const uint32_t ring = smem_u32(smem) + warp * NS * 2 * L::kSliceBytes;
  Feed<DP, FULL, NS> feed(p, ring, NS, seen_s[warp]);
  const int g = lane >> 2, t = lane & 3;
  auto slices = [&](auto careful) {         // true: there is NaN in a part
    Cursor out = begin, in = begin;
    View view = tile_view<kTile, L::kStep>(p, in.b, 0), view_in = view;
    feed.enter(in.b, in.grp);
    int32_t next_page = -1;
    uint32_t next_row = 0;
    auto issue = [&]() {
      if (feed.issued < mine) {
        const int32_t page = next_page;
        const uint32_t row = next_row;
        const uint8_t *k = feed.k, *v = feed.v;
        if (feed.issued + 1 < mine) {
          if (advance(in, view_in)) feed.enter(in.b, in.grp);
          feed.look_up(view_in, in.slice, next_page, next_row);
        }
        feed.copy(page, row, k, v);
      }
      feed.commit();
    };
    feed.look_up(view_in, in.slice, next_page, next_row);
#pragma unroll
    for (int i = 0; i < NS - 1; ++i) issue();
    Rows<DP, FULL, BF16, NT> rows;
    rows.enter(p, view, out.b, out.grp, 0);
    bool nan = false;
    for (int32_t i = 0, at = 0; i < mine; ++i, at = at + 1 == NS ? 0 : at + 1) {
      cp_async_wait<NS - 2>();
      __syncwarp();
      rows.template step<careful>(p, view, ring + at * 2 * L::kSliceBytes, view.slice(out.slice) * L::kStep, seen_s[warp][at],
                                  issue);
      if (i + 1 < mine && out.slice + 1 < out.n) {
        ++out.slice;
        continue;
      }
      nan = nan || rows.any_nan(view);
      const int64_t slot = static_cast<int64_t>(me) + out.b * p.groups + out.grp;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = 8 * n + 2 * t + h;
          const float part = keys_sum(rows.l[n][h]);
          if (r >= p.rows) continue;
          if (g == 0) parts.ml[slot * kTile + r] = make_float2(rows.m[n][h], part);
          float* dst = parts.o + (slot * kTile + r) * p.head_dim;
#pragma unroll
          for (int c = 0; c < DP / 16; ++c) {
            if (c * 16 + g < p.head_dim) dst[c * 16 + g] = rows.o[n][c][h];
            if (c * 16 + 8 + g < p.head_dim) dst[c * 16 + 8 + g] = rows.o[n][c][2 + h];
          }
        }
      if (i + 1 < mine) {
        advance(out, view);
        rows.enter(p, view, out.b, out.grp, 0);
      }
    }
    return __any_sync(0xffffffffu, nan);
  };
  if (slices(std::false_type{})) {          // all of the warp's parts once more
    feed.restart();
    slices(std::true_type{});
  }
  cp_async_wait<0>();
}

// Joins the parts of each row, WPR warps a row: warp i takes parts i, i + WPR, .. in order, the
// warps are joined in order.  Lane l holds the weight of its warp's l-th part, so that the parts'
// values are loaded without waiting for one another.
template <bool BF16, int WPR>
__global__ void __launch_bounds__(WPR > 4 ? WPR * 32 : 128)
paged_combine_kernel(const PagedParams p, const Parts parts, int32_t tile) {
  __shared__ float4 acc_s[WPR][32];
  __shared__ float total_s[WPR];
  wait_previous_kernel();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, mine = WPR > 1 ? warp : 0;
  const int64_t lin = WPR > 1 ? blockIdx.x : static_cast<int64_t>(blockIdx.x) * 4 + warp;  // (sequence, head, token)
  if (lin >= static_cast<int64_t>(p.batch) * p.heads * p.queries) return;
  const int32_t tok = static_cast<int32_t>(lin % p.queries), bh = static_cast<int32_t>(lin / p.queries);
  const int32_t b = bh / p.heads, h = bh - b * p.heads;
  const int32_t grp = h / p.per_group, item = b * p.groups + grp, row = tok * p.per_group + h - grp * p.per_group;
  const int32_t before = __ldcg(parts.plan + b), n = __ldcg(parts.plan + b + 1) - before, per = __ldcg(parts.plan + p.batch + 1);
  const bool counts = n > 0 && (p.counts == nullptr || tok < p.counts[b]);
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float total = 0.f;
  const int d = lane * 4;
  if (counts) {
    const int32_t f0 = before * p.groups + grp * n, w0 = f0 / per, n_parts = (f0 + n - 1) / per - w0 + 1;
    const int64_t first = (static_cast<int64_t>(w0) + item) * tile + row;
    float top = -INFINITY;
    for (int32_t s = lane; s < n_parts; s += 32) top = max_nan(top, __ldcg(&parts.ml[first + static_cast<int64_t>(s) * tile]).x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
    for (int32_t s0 = mine; s0 < n_parts; s0 += 32 * WPR) {
      float weight = 0.f, part = 0.f;
      if (s0 + lane * WPR < n_parts) {
        const float2 e = __ldcg(&parts.ml[first + static_cast<int64_t>(s0 + lane * WPR) * tile]);
        weight = e.x == -INFINITY ? 0.f : fast_exp2(e.x - top);
        part = e.x == -INFINITY ? 0.f : e.y * weight;
      }
      const int32_t left = (n_parts - s0 + WPR - 1) / WPR, m = left < 32 ? left : 32;
      const float* src = parts.o + (first + static_cast<int64_t>(s0) * tile) * p.head_dim + d;
#pragma unroll 8
      for (int s = 0; s < m; ++s) {
        const float w = __shfl_sync(0xffffffffu, weight, s);
        total += __shfl_sync(0xffffffffu, part, s);
        if (w != 0.f && d < p.head_dim) {
          const float4 v = __ldcg(reinterpret_cast<const float4*>(src + static_cast<int64_t>(s) * WPR * tile * p.head_dim));
          acc.x = fmaf(v.x, w, acc.x);
          acc.y = fmaf(v.y, w, acc.y);
          acc.z = fmaf(v.z, w, acc.z);
          acc.w = fmaf(v.w, w, acc.w);
        }
      }
    }
  }
  if (WPR > 1) {
    acc_s[mine][lane] = acc;
    if (lane == 0) total_s[mine] = total;
    __syncthreads();
    if (mine > 0) return;
#pragma unroll
    for (int i = 1; i < WPR; ++i) {
      const float4 v = acc_s[i][lane];
      acc = make_float4(acc.x + v.x, acc.y + v.y, acc.z + v.z, acc.w + v.w);
      total += total_s[i];
    }
  }
  const float inv = total != 0.f ? 1.f / total : 0.f;
  if (d < p.head_dim)
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + b * p.os[0] + h * p.os[1] + tok * p.os[2] + d) =
        make_uint2(pack2<BF16>(acc.x * inv, acc.y * inv), pack2<BF16>(acc.z * inv, acc.w * inv));
}

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

// Rows of a tile: 8 where they hold all.
int tile_rows(int64_t rows) { return rows <= 8 ? 8 : 16; }

struct Plan {
  bool parts, three;                       // three: CTAs an SM
  int64_t o_bytes, ml_bytes, bytes;        // of the workspace
};

int64_t align256(int64_t n) { return (n + 255) / 256 * 256; }

// Largest number of slices of a tile of `tokens` tokens, from what the host knows.
int64_t most_slices(const paged_attention_args* a, int64_t tokens) {
  const int64_t kStep = a->head_dim <= 64 ? Shape<64>::kStep : Shape<128>::kStep;
  const int64_t all = (a->table_width * a->page_size + kStep - 1) / kStep;
  // window + tokens - 1 states in a row touch less than two slices more than they fill
  return a->window > 0 ? std::min(all, (a->sinks + kStep - 1) / kStep + (a->window + tokens) / kStep + 2) : all;
}

// Warps and CTAs of an item in one launch.  Eight warps an SM hold the memory: an item gets the power of
// two of warps that leaves all of them at work, in CTAs of eight.  A cluster of eight (or four, two) CTAs
// that fill an SM each wants its SMs in one part of the GPU: 14, 32 and 72 of them find their place at
// once (B2 G8, 16 items: clusters of four 5.3 us, of eight 6.8).
// No more warps than slices: a sequence of up to 100 states 3.6 us instead of 4.8; two or more slices a warp
// before a cluster grows cost more than its join (500 states of D128, 3 items of 777 of D64: 5.1 -> 5.7, 4.8 -> 5.3).
struct Team {
  int warps, ranks;
};
Team team(int64_t items, int64_t slices) {
  Team t{1, 1};
  while (t.warps < kMostWarps && t.warps < slices && items * t.warps * 2 <= kPartsAll) t.warps *= 2;
  while (t.warps == kMostWarps && t.ranks < kMostRanks && t.warps * t.ranks < slices &&
         items * t.ranks * 2 <= (t.ranks == 1 ? 144 : t.ranks == 2 ? 128 : 112))
    t.ranks *= 2;
  return t;
}

Plan plan(const paged_attention_args* a) {
  Plan x{};
  const int64_t rows = a->heads / a->groups * a->queries, items = a->batch * a->groups;
  const int64_t slices = most_slices(a, a->queries);
  // A second launch costs 3 to 4 us; what it saves are warps that wait for others.  Equal parts are taken
  // where a warp would have more than 125 slices, or 24 while less than half of the warps are at work.
  // One launch / parts, us, G8, lengths from half of the given one up to it (all of it):
  //   D128 B32: 6000 states (94 slices a warp) 101 / 102 (115 / 124), 8000 (125) 126 / 126 (151 / 163), 8192 130 / 128,
  //   10000 (156) 162 / 159, 14000 (219) 220 / 210 (260 / 277); B64 of two warps an item: 4000 (125) 126 / 127, 5000 (156)
  //   157 / 159, 6000 (188) 193 / 185, 8192 (256) 250 / 239 (309 / 320).  D64 B64: 8000 (125) 124 / 127, 12000 (188) 192 / 188.
  //   D80 B64, where columns are checked: 3000 (94) 79 / 71 (88 / 89), 6000 (188) 153 / 124 (160 / 163).
  // Lengths that are equal would do better in one launch by 3 to 8 %, but the host does not know them.
  // One sequence, D128: 16000 (16, 512 warps) 15.6 / 17.1, 32000 (31) 24.7 / 24.0, 131071 109 / 90.
  const Team t = team(items, slices);
  const int64_t each = (slices + t.warps * t.ranks - 1) / (t.warps * t.ranks);
  const bool better = each > 125 || (each >= 24 && items * t.warps * t.ranks * 2 < kPartsAll);
  // One tile a key head, prefix sums that fit, 32-bit slice numbers.
  const bool able = rows <= 16 && a->batch <= kPartsBatch && items * slices <= INT32_MAX - 2 * kThreeCtas * kPartsWarps;
  x.parts = able && (a->kernel == PAGED_KERNEL_PARTS || (a->kernel == PAGED_KERNEL_AUTO && better));
  if (x.parts) {
    // Three CTAs an SM want a tile of 8 rows (16 do not fit their registers), and pay where the parts are long
    // and of many items.  Two / three, us, D128 and G8: 8 items of 32000 states 30.1 / 32.9, of 131071 89 / 93; 16 of 65000
    // 84.5 / 84.0; 32 of 32000 68.2 / 67.4; 64 of 32000 123 / 120; 128 of 16000 136 / 132; 512 of 8192 245 / 235.  D80, whose
    // columns are checked: 512 of 4096 89.2 / 90.6.
    x.three = rows <= 8 && a->head_dim == 128 && items >= 32;
    const int64_t slots = ((x.three ? kThreeCtas * kPartsWarps : kPartsAll) + items) * tile_rows(rows);
    x.o_bytes = align256(slots * a->head_dim * 4);
    x.ml_bytes = align256(slots * 8);
    x.bytes = x.o_bytes + x.ml_bytes + align256((a->batch + 2) * 4);
  }
  return x;
}

template <int DP, bool FULL, bool BF16, int NT>
int32_t launch_joined(PagedParams p, int64_t slices, cudaStream_t stream) {
  using L = Shape<DP>;
  auto kernel = paged_joined_kernel<DP, FULL, BF16, NT>;
  constexpr int kSlice = 2 * L::kSliceBytes, kJoin = 8 * NT * (DP + 4) * 4;  // of a warp
  constexpr int kMost = kMostWarps * std::max(L::kStages * kSlice, kJoin) + kAlign;
  static_assert(kMost <= 224 * 1024, "shared memory of a CTA");
  static std::atomic<uint64_t> done{0};
  if (!allow_smem(kernel, kMost, done)) return INTP_ERR_LAUNCH;
  p.n_rt = (p.rows + 8 * NT - 1) / (8 * NT);
  const int64_t items = static_cast<int64_t>(p.n_rt) * p.batch * p.groups;
  const Team t = team(items, slices);
  const int warps = t.warps, ranks = t.ranks;
  if (items * ranks > INT32_MAX) return INTP_ERR_SHAPE;
  p.depth = static_cast<int32_t>(std::min<int64_t>(L::kStages, (slices + warps * ranks - 1) / (warps * ranks)));
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = static_cast<unsigned>(ranks);
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(items * ranks));
  cfg.blockDim = dim3(static_cast<unsigned>(warps * 32));
  cfg.dynamicSmemBytes = static_cast<size_t>(warps * std::max(p.depth * kSlice, kJoin) + kAlign);
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p) == cudaSuccess ? INTP_OK : INTP_ERR_LAUNCH;
}

template <int DP, bool FULL, bool BF16, int NT, int kCtas, int NS>
int32_t launch_parts(PagedParams p, const Parts& parts, cudaStream_t stream) {
  using L = Shape<DP>;
  auto kernel = paged_parts_kernel<DP, FULL, BF16, NT, kCtas, NS>;
  constexpr int kRing = kPartsWarps * NS * 2 * L::kSliceBytes, kMost = kRing + kAlign + (kPartsBatch + 1) * 4;
  static_assert((kCtas / 148) * (kMost + 256 + 1024) <= 228 * 1024, "CTAs an SM, 1 KB of each the system's");
  static std::atomic<uint64_t> done{0};
  if (!allow_smem(kernel, kMost, done)) return INTP_ERR_LAUNCH;
  p.n_rt = 1;
  if (!launch_kernel(kernel, dim3(kCtas), kPartsWarps * 32, kRing + kAlign + (p.batch + 1) * 4, stream, false, p, parts))
    return INTP_ERR_LAUNCH;
  const int64_t rows = static_cast<int64_t>(p.batch) * p.heads * p.queries;
  // Few items have many parts each: a CTA per row, whose warps share them.  Sixteen warps / four: 37 parts
  // (B4 G8 of 32000 states) 69.5 / 71.4 us; sixteen / eight / thirty-two: 148 parts (B1 G8 of 131071) 90 / 94 / 94.
  const int64_t each = kPartsAll / (static_cast<int64_t>(p.batch) * p.groups);
  const int wide = each >= 24 ? 16 : each >= 16 ? 4 : 1;
  auto combine = wide == 16 ? paged_combine_kernel<BF16, 16> : wide == 4 ? paged_combine_kernel<BF16, 4> : paged_combine_kernel<BF16, 1>;
  const int64_t grid = wide > 1 ? rows : (rows + 3) / 4;
  return launch_kernel(combine, dim3(static_cast<unsigned>(grid)), wide == 16 ? 512 : 128, 0, stream, true, p, parts, 8 * NT)
             ? INTP_OK
             : INTP_ERR_LAUNCH;
}

template <int DP, bool FULL, bool BF16>
int32_t launch_rows(const PagedParams& p, const Parts* parts, int64_t slices, cudaStream_t stream) {
  constexpr int NS = Shape<DP>::kStages;
  if constexpr (FULL && DP == 128)
    if (parts != nullptr && parts->three) return launch_parts<DP, FULL, BF16, 1, kThreeCtas, kThreeStages>(p, *parts, stream);
  if (parts != nullptr)
    return p.rows <= 8 ? launch_parts<DP, FULL, BF16, 1, kPartsCtas, NS>(p, *parts, stream)
                       : launch_parts<DP, FULL, BF16, 2, kPartsCtas, NS>(p, *parts, stream);
  return p.rows <= 8 ? launch_joined<DP, FULL, BF16, 1>(p, slices, stream) : launch_joined<DP, FULL, BF16, 2>(p, slices, stream);
}

// Head dims that fill their slices' rows need no checks of columns.
template <bool BF16>
int32_t launch_dim(const PagedParams& p, const Parts* parts, int64_t slices, cudaStream_t stream) {
  const int32_t d = p.head_dim;
  if (d == 32) return launch_rows<32, true, BF16>(p, parts, slices, stream);
  if (d == 64) return launch_rows<64, true, BF16>(p, parts, slices, stream);
  if (d == 128) return launch_rows<128, true, BF16>(p, parts, slices, stream);
  if (d < 32) return launch_rows<32, false, BF16>(p, parts, slices, stream);
  if (d < 64) return launch_rows<64, false, BF16>(p, parts, slices, stream);
  return launch_rows<128, false, BF16>(p, parts, slices, stream);
}

intp_status check_shape(const paged_attention_args* a) {
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
  if (a->kernel < PAGED_KERNEL_AUTO || a->kernel > PAGED_KERNEL_PARTS) return INTP_ERR_ARGUMENT;
  if (a->kernel == PAGED_KERNEL_PARTS && a->batch > 0 && a->queries > 0 && !plan(a).parts) return INTP_ERR_UNSUPPORTED;
  return INTP_OK;
}

intp_status run(const paged_attention_args* a, cudaStream_t stream) {
  if (!a) return INTP_ERR_ARGUMENT;
  const intp_status st = check_shape(a);
  if (st != INTP_OK) return st;
  if (a->batch == 0 || a->queries == 0) return INTP_OK;
  if (!a->q || !a->k || !a->v || !a->out || !a->page_table || !a->start) return INTP_ERR_ARGUMENT;
  const int64_t eq[3] = {a->batch, a->heads, a->queries}, ek[3] = {a->pages, a->groups, a->page_size};
  if (!rows_ok(a->q, a->q_stride, eq) || !rows_ok(a->out, a->out_stride, eq) || !rows_ok(a->k, a->cache_stride, ek) ||
      !rows_ok(a->v, a->cache_stride, ek))
    return INTP_ERR_LAYOUT;
  int64_t cache[3];
  take(cache, a->cache_stride, ek);
  // Places are 32-bit numbers of 16-byte units.
  if (cache[0] / 8 > UINT32_MAX || cache[2] / 8 > UINT32_MAX ||
      (a->pages - 1) * (cache[0] / 8) + (a->page_size - 1) * (cache[2] / 8) > UINT32_MAX) return INTP_ERR_LAYOUT;
  const Plan how = plan(a);
  if (how.bytes > 0 &&
      (!a->workspace || reinterpret_cast<uintptr_t>(a->workspace) % 256 || a->workspace_bytes < how.bytes))
    return INTP_ERR_ARGUMENT;
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
  p.v = a->v;
  p.head_stride = cache[1];
  p.page_units = static_cast<uint32_t>(cache[0] / 8);
  p.row_units = static_cast<uint32_t>(cache[2] / 8);
  // With 2^shift >= page_size, magic = ceil(2^(30 + shift) / page_size) is off by less than
  // 2^shift / page_size of 2^30: the quotient is exact for every p < 2^30.
  while ((int64_t(1) << p.page_shift) < a->page_size) ++p.page_shift;
  p.page_magic = static_cast<uint32_t>(((uint64_t(1) << (30 + p.page_shift)) + a->page_size - 1) / a->page_size);
  p.out = a->out;
  take(p.os, a->out_stride, eq);
  p.table = a->page_table;
  p.table_stride = a->table_stride;
  p.start = a->start;
  p.counts = a->counts;
  Parts parts{};
  if (how.parts) {
    uint8_t* ws = static_cast<uint8_t*>(a->workspace);
    parts.o = reinterpret_cast<float*>(ws);
    parts.ml = reinterpret_cast<float2*>(ws + how.o_bytes);
    parts.plan = reinterpret_cast<int32_t*>(ws + how.o_bytes + how.ml_bytes);
    parts.three = how.three;
  }
  const Parts* x = how.parts ? &parts : nullptr;
  const int64_t tokens = std::min<int64_t>(a->queries, 16), slices = most_slices(a, tokens);  // a tile has 16 rows at most
  return a->dtype == INTP_BF16 ? launch_dim<true>(p, x, slices, stream) : launch_dim<false>(p, x, slices, stream);
}

}  // namespace
}  // namespace intp

extern "C" {

intp_status paged_attention_workspace(const paged_attention_args* a, int64_t* bytes) {
  if (!a || !bytes) return INTP_ERR_ARGUMENT;
  const intp_status st = intp::check_shape(a);
  if (st != INTP_OK) return st;
  *bytes = a->batch == 0 || a->queries == 0 ? 0 : intp::plan(a).bytes;
  return INTP_OK;
}

intp_status paged_attention(const paged_attention_args* a, void* stream) {
  return intp::run(a, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
