// cross_attention_rows.cu - cross attention of few query rows over many states
// (sm_100a): single tokens and small batches of them, over 16-bit or 8-bit
// (e4m3 with a power of two per state) keys and values, and the kernel that
// joins the parts of a split pass.
//
// Reading the states bounds this: 16 rows or fewer share each key, so a 16-bit
// state of 4 D bytes carries at most 64 D multiply-adds, far below the tensor
// cores' ratio.  What counts is bytes in flight and few instructions per byte.
// A CTA of 4 (or 8) warps takes 8 or 16 rows and a range of keys; each warp streams its
// own slices of keys through a private cp.async ring (no CTA barrier in the
// loop) and keeps its own running maximum and sum.  The products are 16 x 8 x 16
// matrix instructions with the states as the 16-high operand,
//   S^T = k q^T (16 keys x 8 rows),   O^T += v^T P^T (16 columns x 8 rows),
// so 8 rows fill them (a 128-row tcgen05 tile would idle on 112 rows or more).
// P^T goes from the first product's layout to the second's by an 8 x 8 transpose
// in registers.  The reference of the exponentials moves only when a score
// passes it by 2^8, so a step needs one vote and no shuffles.  Over 16-bit states the
// probabilities go in as two 16-bit numbers each, the value and what it leaves out: the
// second product is hidden under the reads, and only the result's own rounding remains
// (one number each: 1.4 times the error of a 32-bit computation rounded once).
// The warps join through shared memory at the end; ranges of keys join through a
// workspace (combine kernel) in a fixed order, so results repeat.
//
// 8-bit states are widened to f16 (exact) as they leave shared memory.  The
// key's power of two multiplies the score; the value's joins the exponent of the
// probability, whose own reference (score + value exponent) keeps the f16
// product operand below 2^8 whatever the exponents are.  It goes in as one f16 number: its 2^-11
// is a hundredth of the codes' own 2^-4, and issue slots, not only memory, bound this form.  A bf16 query row is
// first scaled by a power of two into the f16 range.
#include <cstdint>
#include "xattn_common.cuh"
#include "xattn_internal.h"

namespace intp {
namespace {

constexpr int kStep = 16;                  // keys of a warp's slice
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kRescale = 8.f;            // log2 units a score may pass its reference by

template <int DP, bool FP8>
struct RowsShape {
  static constexpr int kElem = FP8 ? 1 : 2;                // bytes of a state's value
  static constexpr int kChunks = DP * kElem / 16;          // 16-byte chunks of a state
  static constexpr int kPerChunk = 16 / kElem;             // values of a chunk
  static constexpr int kSliceBytes = kStep * DP * kElem;   // K or V of a slice
  // 8-bit states cost more instructions a byte: less shared memory a CTA and twice the warps an
  // SM (16-key slices, 48 KB: 142 us at B64 G8 H32 N8192 D128; 32-key slices, 96 KB: 178 us).
  static constexpr int kStages = DP == 128 ? 3 : 6;
  static constexpr int kWarpRing = kStages * 2 * kSliceBytes;
};

template <int CH>
__device__ __forceinline__ uint32_t chunk_offset(int row, int c) {
  const int sw = CH == 4 ? (row >> 1) & 3 : row & 7;
  return static_cast<uint32_t>(row * CH + (c ^ sw)) * 16;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool read) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(read ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// Transpose of the 8 x 8 16-bit matrix whose row g this lane quad holds.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
  return d;
}
// C += A B for 16 rows, 8 columns and a depth of 16.
template <bool BF16>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  if (BF16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Four e4m3 codes (low byte first) to two pairs of f16 values, exact.
__device__ __forceinline__ void widen4(uint32_t codes, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(codes));
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
// Over the eight lanes that hold a query row's keys.
__device__ __forceinline__ float keys_max(float v) {
#pragma unroll
  for (int s = 4; s < 32; s <<= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, s));
  return v;
}
__device__ __forceinline__ float keys_sum(float v) {
#pragma unroll
  for (int s = 4; s < 32; s <<= 1) v += __shfl_xor_sync(0xffffffffu, v, s);
  return v;
}

struct RowsArgs {
  XaParams p;
  int32_t n_rt;
  int32_t smem_scales;   // bytes from the dynamic shared memory's start to the exponents' values
};

// NT: tiles of 8 query rows.  kWarps: 4, or 8 where a grid of one part leaves SMs empty.
template <int DP, bool BF16, bool FP8, int NT, int kWarps>
__global__ void __launch_bounds__(kWarps * 32)
xattn_rows_kernel(const RowsArgs a) {
  using L = RowsShape<DP, FP8>;
  constexpr int CH = L::kChunks, NS = L::kStages;
  constexpr bool MMA_BF16 = BF16 && !FP8;   // element type of the products
  constexpr int kTile = 8 * NT;             // rows of a CTA
  constexpr int kJoinStride = DP + 4;       // floats
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float m_s[kWarps][kTile], l_s[kWarps][kTile], w_s[kWarps][kTile];
  allow_next_kernel();
  const XaParams& p = a.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;    // fragment row and column pair

  const int32_t is = blockIdx.x / a.n_rt, rt = blockIdx.x - is * a.n_rt;
  const int32_t inst = is / p.n_split, split = is - inst * p.n_split;
  const int32_t b = p.shared ? 0 : inst / p.groups, grp = p.shared ? inst : inst - b * p.groups;
  const int32_t length = xa_length(p, b);
  const int32_t key0 = split * p.split_keys;
  const int32_t left = length - key0;
  const int32_t n_keys = left < 0 ? 0 : (left < p.split_keys ? left : p.split_keys);
  const int32_t row0 = rt * kTile;
  const int32_t n_rows = p.rows - row0 < kTile ? p.rows - row0 : kTile;
  const int32_t D = p.head_dim;

  const uint32_t ring = smem_u32(smem) + warp * NS * 2 * L::kSliceBytes;
  // Slices: those of a prefix that is read in the same pass (16-bit states), then the range's own.
  const int32_t n_prefix = FP8 ? 0 : p.prefix;
  const int32_t pre_slices = (n_prefix + kStep - 1) / kStep;
  const int32_t n_slices = pre_slices + (n_keys + kStep - 1) / kStep;
  const int32_t mine = n_slices > warp ? (n_slices - warp + kWarps - 1) / kWarps : 0;

  // This lane copies chunk `cc` of states `cr`, cr + 32 / CH, ... of each slice.
  const int cr = lane / CH, cc = lane % CH;
  const bool chunk_read = cc * L::kPerChunk < D;
  const bool chunk_used = cc * L::kPerChunk < ((D + 15) & ~15);  // columns past D that the products read are zero
  const int32_t lane_byte = chunk_read ? cc * 16 : 0;
  int64_t k_row = 0, v_row = 0;
  const uint8_t *k_src = nullptr, *v_src = nullptr;
  // Points this lane at its first state of slice `first` of a segment's states.
  auto enter = [&](const void* k, const void* v, int64_t k_base, int64_t v_base, int64_t k_stride, int64_t v_stride,
                   int32_t first) {
    k_row = k_stride * L::kElem;
    v_row = v_stride * L::kElem;
    const int64_t state = static_cast<int64_t>(first) * kStep + cr;
    k_src = static_cast<const uint8_t*>(k) + k_base * L::kElem + state * k_row + lane_byte;
    v_src = static_cast<const uint8_t*>(v) + v_base * L::kElem + state * v_row + lane_byte;
  };
  auto enter_own = [&](int32_t first) {
    enter(p.k, p.v, b * p.ks[0] + grp * p.ks[1] + key0 * p.ks[2], b * p.vs[0] + grp * p.vs[1] + key0 * p.vs[2], p.ks[2],
          p.vs[2], first);
  };
  if (!FP8 && warp < pre_slices)
    enter(p.pre_k, p.pre_v, grp * p.pre_ks[0], grp * p.pre_vs[0], p.pre_ks[1], p.pre_vs[1], warp);
  else
    enter_own(warp - pre_slices);
  int32_t issued = 0;
  // The next slice of this warp (warp, warp + 4, ...) into its ring; keys past the end are zero.
  auto issue = [&]() {
    if (issued < mine) {
      const int32_t slice = issued * kWarps + warp;
      const bool pre = !FP8 && slice < pre_slices;
      const int32_t left = pre ? n_prefix - slice * kStep : n_keys - (slice - pre_slices) * kStep;
      const uint32_t dst = ring + (issued % NS) * 2 * L::kSliceBytes;
      const int64_t k_next = (32 / CH) * k_row, v_next = (32 / CH) * v_row;
      const uint8_t *ks = k_src, *vs = v_src;
      if (left >= kStep && chunk_read) {
#pragma unroll
        for (int u = 0; u < kStep * CH / 32; ++u, ks += k_next, vs += v_next) {
          const uint32_t to = dst + chunk_offset<CH>(cr + u * (32 / CH), cc);
          cp_async16(to, ks);
          cp_async16(to + L::kSliceBytes, vs);
        }
      } else if (chunk_used) {
#pragma unroll
        for (int u = 0; u < kStep * CH / 32; ++u, ks += k_next, vs += v_next) {
          const int row = cr + u * (32 / CH);
          const bool read = row < left && chunk_read;
          const uint32_t to = dst + chunk_offset<CH>(row, cc);
          cp_async16(to, read ? ks : static_cast<const uint8_t*>(p.q), read);
          cp_async16(to + L::kSliceBytes, read ? vs : static_cast<const uint8_t*>(p.q), read);
        }
      }
      if (pre && slice + kWarps >= pre_slices) {
        enter_own(slice + kWarps - pre_slices);
      } else {
        k_src += kWarps * kStep * k_row;
        v_src += kWarps * kStep * v_row;
      }
    }
    ++issued;
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < NS - 1; ++i) issue();

  // 8-bit states: each state's exponent bytes, the key's low and the value's high.
  uint16_t* exp_s = reinterpret_cast<uint16_t*>(smem + a.smem_scales);
  if (FP8) {
    const int64_t base = b * p.es[0] + grp * p.es[1] + key0;
    for (int i = threadIdx.x; i < n_keys; i += kWarps * 32)
      exp_s[i] = static_cast<uint16_t>(p.k_exp[base + i] | (p.v_exp[base + i] << 8));
  }

  // Query fragments (rows 8 n + g as columns of q^T); the depth order follows the K fragments
  // (16-bit: columns 2t, 2t+1 and 2t+8, 2t+9 of each 16; 8-bit: 4t .. 4t+3).
  uint32_t qb[NT][DP / 16][2];
  float row_scale[NT][2];                   // of rows 8 n + 2 t, + 1 (the score fragment's columns)
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int32_t r = row0 + 8 * n + g;
    const uint16_t* src = nullptr;
    if (r < p.rows) {
      const XaRow x = xa_row(p, inst, r);
      src = static_cast<const uint16_t*>(p.q) + x.b * p.qs[0] + x.h * p.qs[1] + x.m * p.qs[2];
    }
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) {
      const int d0 = kk * 16 + (FP8 ? 4 * t : 2 * t), d1 = d0 + (FP8 ? 2 : 8);
      qb[n][kk][0] = src != nullptr && d0 < D ? *reinterpret_cast<const uint32_t*>(src + d0) : 0u;
      qb[n][kk][1] = src != nullptr && d1 < D ? *reinterpret_cast<const uint32_t*>(src + d1) : 0u;
    }
    float up = p.scale * kLog2e;
    if (FP8 && BF16) {
      // Largest magnitude to [2^14, 2^15): every value within 2^-28 of it is exact in f16.
      float top = 0.f;
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float2 f = unpack2<true>(qb[n][kk][e]);
          top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
        }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      int e = top >= 1.17549435e-38f ? static_cast<int>(__float_as_uint(top) >> 23) - 127 - 14 : 0;
      e = e < -126 ? -126 : e;
      const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
      up *= __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float2 f = unpack2<true>(qb[n][kk][i]);
          qb[n][kk][i] = pack_f16x2(f.x * down, f.y * down);
        }
    }
    row_scale[n][0] = __shfl_sync(0xffffffffu, up, 8 * t);       // the lanes of g = 2 t
    row_scale[n][1] = __shfl_sync(0xffffffffu, up, 8 * t + 4);
  }
  if (FP8) __syncthreads();  // the exponents are in

  float o[NT][DP / 16][4];
  // Per row (8 n + 2 t + h): running reference, that of score + value exponent, this lane's part of the sum.
  float m[NT][2], mw[NT][2], l[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int c = 0; c < DP / 16; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[n][c][e] = 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      m[n][h] = mw[n][h] = -INFINITY;
      l[n][h] = 0.f;
    }
  }
  const int mi = lane >> 3, mr = lane & 7;

  for (int32_t i = 0; i < mine; ++i) {
    cp_async_wait<NS - 2>();
    __syncwarp();
    const uint32_t k_s = ring + (i % NS) * 2 * L::kSliceBytes, v_s = k_s + L::kSliceBytes;
    // First key of the slice, and the segment's end, in the segment's own count.
    const int32_t slice = i * kWarps + warp;
    const bool pre = !FP8 && slice < pre_slices;
    const int32_t k0 = (pre ? slice : slice - pre_slices) * kStep, end = pre ? n_prefix : n_keys;
    float s[NT][4];                         // rows 2t, 2t+1 (e & 1), keys g, g + 8 (e >> 1)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
    if (FP8) {
#pragma unroll
      for (int c = 0; c < CH; c += 2) {
        if (c * 16 >= D) break;
        uint32_t r[4];                    // keys 0-7 and 8-15 of chunk c, then of c + 1
        ldmatrix4(k_s + chunk_offset<CH>(mr + ((mi & 1) << 3), c + (mi >> 1)), r);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          if ((c + u) * 16 >= D) break;
          uint32_t a0, a1, a2, a3;
          widen4(r[2 * u], a0, a2);
          widen4(r[2 * u + 1], a1, a3);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma16816<false>(s[n], a0, a1, a2, a3, qb[n][c + u][0], qb[n][c + u][1]);
        }
      }
    } else {
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk) {
        if (kk * 16 >= D) break;
        uint32_t r[4];                    // keys 0-7 and 8-15 of chunk 2 kk, then of 2 kk + 1
        ldmatrix4(k_s + chunk_offset<CH>(mr + ((mi & 1) << 3), 2 * kk + (mi >> 1)), r);
#pragma unroll
        for (int n = 0; n < NT; ++n) mma16816<MMA_BF16>(s[n], r[0], r[1], r[2], r[3], qb[n][kk][0], qb[n][kk][1]);
      }
    }
    // Scores in log2 units; padded keys -inf.
    float w[2];                             // value exponents
    bool grow = false;
    const bool padded = k0 + kStep > end;
#pragma unroll
    for (int kh = 0; kh < 2; ++kh) {
      const int32_t key = k0 + kh * 8 + g;
      float2 f = make_float2(1.f, 0.f);   // the key's power of two, the value's exponent
      if (FP8) {
        const uint32_t e = exp_s[!padded || key < end ? key : 0];
        // a byte below 2^23's mantissa is that number above it
        f = make_float2(__uint_as_float((e & 0xffu) << 23), __uint_as_float(0x4b000000u | (e >> 8)) - 8388735.f);
      }
      w[kh] = f.y;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float& v = s[n][2 * kh + h];
          v *= row_scale[n][h];
          if (FP8) v *= f.x;
          if (padded && key >= end) v = -INFINITY;
          // a NaN score counts as growth: it has to reach the reference
          grow = grow || !(v <= m[n][h] + kRescale) || (FP8 && !(v + f.y <= mw[n][h] + kRescale));
        }
    }
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float fo[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float top = m[n][h], topw = mw[n][h];
#pragma unroll
          for (int kh = 0; kh < 2; ++kh) {
            top = max_nan(top, s[n][2 * kh + h]);
            if (FP8) topw = max_nan(topw, s[n][2 * kh + h] + w[kh]);
          }
          top = keys_max(top);
          topw = FP8 ? keys_max(topw) : top;
          l[n][h] *= top == -INFINITY ? 1.f : fast_exp2(m[n][h] - top);
          fo[h] = topw == -INFINITY ? 1.f : fast_exp2((FP8 ? mw[n][h] : m[n][h]) - topw);
          m[n][h] = top;
          mw[n][h] = topw;
        }
#pragma unroll
        for (int c = 0; c < DP / 16; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[n][c][e] *= fo[e & 1];
      }
    }
    uint32_t pb[NT][2];                     // P^T as the 8-wide operand: keys 2t, 2t+1 of each 8, row g
    uint32_t pl[NT][2];                     // what its 16 bits leave out (16-bit states)
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      // A row without a score above -inf keeps 0 as its reference.
      const float ref[2] = {m[n][0] == -INFINITY ? 0.f : m[n][0], m[n][1] == -INFINITY ? 0.f : m[n][1]};
      const float refw[2] = {mw[n][0] == -INFINITY ? 0.f : mw[n][0], mw[n][1] == -INFINITY ? 0.f : mw[n][1]};
#pragma unroll
      for (int kh = 0; kh < 2; ++kh) {
        float pr[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float v = s[n][2 * kh + h];
          pr[h] = fast_exp2(v - ref[h]);
          l[n][h] += pr[h];
          if (FP8) pr[h] = fast_exp2(v + w[kh] - refw[h]);
        }
        const uint32_t high = pack2<MMA_BF16>(pr[0], pr[1]);
        pb[n][kh] = transpose8(high);
        if (!FP8) {
          const float2 h = unpack2<MMA_BF16>(high);
          pl[n][kh] = transpose8(pack2<MMA_BF16>(pr[0] - h.x, pr[1] - h.y));
        }
      }
    }
#pragma unroll
    for (int c = 0; c < CH; c += 2) {
      if (c * L::kPerChunk >= D) break;
      uint32_t r[4];
      if (FP8) {
        // keys 0-7 and 8-15 of chunk c, then of c + 1: two columns of two keys each
        ldmatrix4_trans(v_s + chunk_offset<CH>(mr + ((mi & 1) << 3), c + (mi >> 1)), r);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          if ((c + u) * 16 >= D) break;
          // -> key pairs of the even, then of the odd column
          uint32_t a0, a1, a2, a3;
          widen4(__byte_perm(r[2 * u], 0u, 0x3120), a0, a1);
          widen4(__byte_perm(r[2 * u + 1], 0u, 0x3120), a2, a3);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma16816<false>(o[n][c + u], a0, a1, a2, a3, pb[n][0], pb[n][1]);
        }
      } else {
        // chunk c and c + 1 of keys 0-7, then of 8-15
        ldmatrix4_trans(v_s + chunk_offset<CH>(mr + ((mi >> 1) << 3), c + (mi & 1)), r);
#pragma unroll
        for (int n = 0; n < NT; ++n) mma16816<MMA_BF16>(o[n][c / 2], r[0], r[1], r[2], r[3], pb[n][0], pb[n][1]);
        // the low parts may be zero or negative: against an infinite value they would turn the
        // high parts' infinity into NaN, so they meet finite values
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = finite2<MMA_BF16>(r[e]);
#pragma unroll
        for (int n = 0; n < NT; ++n) mma16816<MMA_BF16>(o[n][c / 2], r[0], r[1], r[2], r[3], pl[n][0], pl[n][1]);
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
        w_s[warp][r] = FP8 ? mw[n][h] : m[n][h];
      }
      if (r < n_rows && mine > 0) {
        float* dst = join + (warp * kTile + r) * kJoinStride;
#pragma unroll
        for (int c = 0; c < DP / 16; ++c) {
          // fragment rows g, g + 8: columns 2 g, 2 g + 1 (8-bit) or g, g + 8 of each 16
          if (FP8) {
            *reinterpret_cast<float2*>(dst + c * 16 + 2 * g) = make_float2(o[n][c][h], o[n][c][2 + h]);
          } else {
            dst[c * 16 + g] = o[n][c][h];
            dst[c * 16 + 8 + g] = o[n][c][2 + h];
          }
        }
      }
    }
  __syncthreads();
  const bool part = p.part_o != nullptr;
  for (int r = warp; r < n_rows; r += kWarps) {
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = max_nan(top, m_s[w][r]);
    const bool none = top == -INFINITY;
    float total = 0.f, f[kWarps];
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const bool has = m_s[w][r] != -INFINITY;
      total += has ? l_s[w][r] * fast_exp2(m_s[w][r] - top) : 0.f;
      f[w] = has ? fast_exp2(w_s[w][r] - top) : 0.f;
    }
    const float inv = none ? 0.f : 1.f / total;
    const XaRow x = xa_row(p, inst, row0 + r);
    const int64_t lin = xa_linear(p, x);
    const int64_t slot = static_cast<int64_t>(p.part_first + split) * p.rows_total + lin;
    const int d = lane * 4;
    if (d < D) {
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w)
        if (f[w] != 0.f) {
          const float4 v = *reinterpret_cast<const float4*>(join + (w * kTile + r) * kJoinStride + d);
          acc.x = fmaf(v.x, f[w], acc.x);
          acc.y = fmaf(v.y, f[w], acc.y);
          acc.z = fmaf(v.z, f[w], acc.z);
          acc.w = fmaf(v.w, f[w], acc.w);
        }
      acc = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
      if (part)
        *reinterpret_cast<float4*>(p.part_o + slot * D + d) = acc;
      else
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + x.b * p.os[0] + x.h * p.os[1] + x.m * p.os[2] + d) =
            make_uint2(pack2<BF16>(acc.x, acc.y), pack2<BF16>(acc.z, acc.w));
    }
    if (lane == 0) {
      const float lse2 = none ? -INFINITY : top + log2f(total);
      if (part)
        p.part_lse[slot] = lse2;
      else if (p.lse != nullptr)
        p.lse[lin] = lse2 * kLn2;
    }
  }
  wait_previous_kernel();
}

// out = sum_s 2^(lse_s - max) part_s / sum_s 2^(lse_s - max), WPR warps per row (warp i takes parts
// i, i + WPR, .. in order, warps are joined in order).  Lane l holds the weight of its warp's l-th
// part, so the parts' values are loaded without waiting for one another.
template <bool BF16, int WPR>
__global__ void __launch_bounds__(128)
xattn_combine_kernel(const XaParams p, int32_t n_slots) {
  __shared__ float4 acc_s[WPR > 1 ? WPR : 1][32];
  __shared__ float total_s[WPR > 1 ? WPR : 1];
  wait_previous_kernel();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = WPR > 1 ? warp : 0;
  const int64_t lin = WPR > 1 ? blockIdx.x : static_cast<int64_t>(blockIdx.x) * 4 + warp;
  if (lin >= p.rows_total) return;
  float top = -INFINITY;
  for (int s = lane; s < n_slots; s += 32) top = max_nan(top, p.part_lse[s * p.rows_total + lin]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
  const bool none = top == -INFINITY;
  const int d = lane * 4;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float total = 0.f;
  for (int s0 = part; s0 < n_slots; s0 += 32 * WPR) {
    float mine = 0.f;
    if (s0 + lane * WPR < n_slots) {
      const float e = p.part_lse[(s0 + lane * WPR) * p.rows_total + lin];
      mine = e == -INFINITY ? 0.f : fast_exp2(e - top);
    }
    const int left = (n_slots - s0 + WPR - 1) / WPR, n = left < 32 ? left : 32;
    const float* src = p.part_o + (s0 * p.rows_total + lin) * p.head_dim + d;
#pragma unroll 8
    for (int s = 0; s < n; ++s) {
      const float w = __shfl_sync(0xffffffffu, mine, s);
      total += w;
      if (w != 0.f && d < p.head_dim) {  // an empty part's values were never written
        const float4 v = __ldcs(reinterpret_cast<const float4*>(src + s * WPR * p.rows_total * p.head_dim));
        acc.x = fmaf(v.x, w, acc.x);
        acc.y = fmaf(v.y, w, acc.y);
        acc.z = fmaf(v.z, w, acc.z);
        acc.w = fmaf(v.w, w, acc.w);
      }
    }
  }
  if (WPR > 1) {
    acc_s[part][lane] = acc;
    if (lane == 0) total_s[part] = total;
    __syncthreads();
    if (part > 0) return;
#pragma unroll
    for (int i = 1; i < WPR; ++i) {
      const float4 v = acc_s[i][lane];
      acc = make_float4(acc.x + v.x, acc.y + v.y, acc.z + v.z, acc.w + v.w);
      total += total_s[i];
    }
  }
  const float inv = none ? 0.f : 1.f / total;
  const int64_t bh = lin / p.queries;
  const int32_t m = static_cast<int32_t>(lin - bh * p.queries);
  const int32_t b = static_cast<int32_t>(bh / p.heads), h = static_cast<int32_t>(bh - static_cast<int64_t>(b) * p.heads);
  if (d < p.head_dim)
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + b * p.os[0] + h * p.os[1] + m * p.os[2] + d) =
        make_uint2(pack2<BF16>(acc.x * inv, acc.y * inv), pack2<BF16>(acc.z * inv, acc.w * inv));
  if (lane == 0 && p.lse != nullptr) p.lse[lin] = none ? -INFINITY : (top + log2f(total)) * kLn2;
}

template <int DP, bool BF16, bool FP8, int NT, int W>
int32_t launch(RowsArgs a, cudaStream_t stream, bool overlap) {
  using L = RowsShape<DP, FP8>;
  auto kernel = xattn_rows_kernel<DP, BF16, FP8, NT, W>;
  constexpr int kRing = W * L::kWarpRing;
  constexpr int kJoin = W * 8 * NT * (DP + 4) * 4;   // the warps' sums, in the rings' place
  constexpr int kData = kRing > kJoin ? kRing : kJoin;
  constexpr int kMost = kData + (FP8 ? 2 * kXaRowsKeys8 : 0);
  static_assert(kMost <= 224 * 1024, "shared memory of a CTA");
  a.smem_scales = kData;
  const int smem = kData + (FP8 ? 2 * a.p.split_keys : 0);
  static std::atomic<uint64_t> done{0};
  if (smem > kMost) return 8;
  if (!allow_smem(kernel, kMost, done)) return 6;
  a.n_rt = (a.p.rows + 8 * NT - 1) / (8 * NT);
  const int64_t grid = static_cast<int64_t>(a.n_rt) * a.p.instances * a.p.n_split;
  if (grid > INT32_MAX) return 8;
  return launch_kernel(kernel, dim3(static_cast<unsigned>(grid)), W * 32, smem, stream, overlap, a) ? 0 : 6;
}

template <int DP, bool BF16, bool FP8>
int32_t launch_rows(const RowsArgs& a, cudaStream_t stream, bool overlap) {
  const bool narrow = a.p.rows <= 8;
  if (a.p.warps == 8)
    return narrow ? launch<DP, BF16, FP8, 1, 8>(a, stream, overlap) : launch<DP, BF16, FP8, 2, 8>(a, stream, overlap);
  return narrow ? launch<DP, BF16, FP8, 1, 4>(a, stream, overlap) : launch<DP, BF16, FP8, 2, 4>(a, stream, overlap);
}

template <bool BF16, bool FP8>
int32_t launch_dim(const RowsArgs& a, cudaStream_t stream, bool overlap) {
  return a.p.head_dim <= 64 ? launch_rows<64, BF16, FP8>(a, stream, overlap)
                            : launch_rows<128, BF16, FP8>(a, stream, overlap);
}

}  // namespace

int32_t launch_xattn_rows(const XaParams& p, cudaStream_t stream, bool overlap) {
  RowsArgs a;
  a.p = p;
  const bool fp8 = p.k_exp != nullptr, bf16 = p.dtype == 2;
  if (fp8) return bf16 ? launch_dim<true, true>(a, stream, overlap) : launch_dim<false, true>(a, stream, overlap);
  return bf16 ? launch_dim<true, false>(a, stream, overlap) : launch_dim<false, false>(a, stream, overlap);
}

int32_t launch_xattn_combine(const XaParams& p, int32_t n_slots, cudaStream_t stream) {
  // Many parts: a CTA per row, whose four warps share them.
  const bool many = n_slots >= 8;
  const int64_t grid = many ? p.rows_total : (p.rows_total + 3) / 4;
  if (grid > INT32_MAX) return 8;
  auto kernel = p.dtype == 2 ? (many ? xattn_combine_kernel<true, 4> : xattn_combine_kernel<true, 1>)
                             : (many ? xattn_combine_kernel<false, 4> : xattn_combine_kernel<false, 1>);
  return launch_kernel(kernel, dim3(static_cast<unsigned>(grid)), 128, 0, stream, true, p, n_slots) ? 0 : 6;
}

}  // namespace intp
