// cross_attention_rows.cu - cross attention of few query rows over many states
// (sm_100a): single tokens and small batches of them, over 16-bit or 8-bit
// (e4m3 with a power of two per state) keys and values, and the kernel that
// joins the parts of a split pass.
//
// Reading the states bounds this: 16 rows or fewer share each key, so a 16-bit
// state of 4 D bytes carries at most 64 D multiply-adds, far below the tensor
// cores' ratio.  What counts is bytes in flight.  A CTA of 4 warps takes 16 rows
// and a range of keys; each warp streams its own 16-key slices through a private
// cp.async ring (no CTA barrier in the loop), forms S = q k^T and O += P v with
// 16 x 8 x 16 matrix instructions (16 rows is their natural height; a 128-row
// tcgen05 tile would idle on 112 of them), and keeps its own running maximum and
// sum.  The warps join through shared memory at the end; ranges of keys join
// through a workspace (combine kernel) in a fixed order, so results repeat.
//
// 8-bit states are widened to f16 (exact) as they leave shared memory.  The
// key's power of two multiplies the score; the value's joins the exponent of the
// probability, whose own running maximum (of score + value exponent) keeps the
// f16 product operand in (0, 1] whatever the exponents are.  A bf16 query row is
// first scaled by a power of two into the f16 range.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>
#include "sm100_ptx.cuh"
#include "xattn_internal.h"

namespace intp {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kStep = 16;                  // keys of a warp's slice
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

template <int DP, bool FP8>
struct RowsShape {
  static constexpr int kElem = FP8 ? 1 : 2;                // bytes of a state's value
  static constexpr int kChunks = DP * kElem / 16;          // 16-byte chunks of a state
  static constexpr int kPerChunk = 16 / kElem;             // values of a chunk
  static constexpr int kSliceBytes = kStep * DP * kElem;   // K or V of a slice
  static constexpr int kStages = DP * kElem == 256 ? 3 : (DP * kElem == 128 ? 6 : 8);
  static constexpr int kRing = kWarps * kStages * 2 * kSliceBytes;
  static constexpr int kJoinStride = DP + 8;               // floats; rows land on different banks
  static constexpr int kJoin = kWarps * kXaRowsTile * kJoinStride * 4;
  static constexpr int kData = kRing > kJoin ? kRing : kJoin;
};

template <int CH>
__device__ __forceinline__ uint32_t chunk_offset(int row, int c) {
  const int sw = CH == 4 ? (row >> 1) & 3 : row & 7;
  return static_cast<uint32_t>(row * CH + (c ^ sw)) * 16;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool read) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(read ? 16 : 0) : "memory");
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
// C += A B for 16 rows, 8 columns and a depth of 16.
template <bool BF16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (BF16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Two e4m3 codes (low byte first) to two f16 values, exact.
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t codes) {
  uint32_t d;
  asm("{\n\t.reg .b16 h;\n\tcvt.u16.u32 h, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}" : "=r"(d) : "r"(codes & 0xffffu));
  return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
// Over the four lanes that hold a row's columns.
__device__ __forceinline__ float quad_max(float v) {
  v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return max_nan(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  return BF16 ? pack_bf16x2(lo, hi) : pack_f16x2(lo, hi);
}
__device__ __forceinline__ float2 bf16x2_to_float2(uint32_t v) {
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}

struct RowsArgs {
  XaParams p;
  int32_t n_rt;
};

template <int DP, bool BF16, bool FP8>
__global__ void __launch_bounds__(kThreads)
xattn_rows_kernel(const RowsArgs a) {
  using L = RowsShape<DP, FP8>;
  constexpr int CH = L::kChunks, NS = L::kStages;
  constexpr bool MMA_BF16 = BF16 && !FP8;   // element type of the products
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float m_s[kWarps][kXaRowsTile], l_s[kWarps][kXaRowsTile], w_s[kWarps][kXaRowsTile];
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
  const int32_t row0 = rt * kXaRowsTile;
  const int32_t n_rows = p.rows - row0 < kXaRowsTile ? p.rows - row0 : kXaRowsTile;
  const int32_t D = p.head_dim;

  const uint8_t* k_src = static_cast<const uint8_t*>(p.k) +
                         (b * p.ks[0] + grp * p.ks[1] + static_cast<int64_t>(key0) * p.ks[2]) * L::kElem;
  const uint8_t* v_src = static_cast<const uint8_t*>(p.v) +
                         (b * p.vs[0] + grp * p.vs[1] + static_cast<int64_t>(key0) * p.vs[2]) * L::kElem;
  const int64_t k_row = p.ks[2] * L::kElem, v_row = p.vs[2] * L::kElem;
  const uint32_t ring = smem_u32(smem) + warp * NS * 2 * L::kSliceBytes;
  const int32_t n_slices = (n_keys + kStep - 1) / kStep;
  const int32_t mine = n_slices > warp ? (n_slices - warp + kWarps - 1) / kWarps : 0;
  const int32_t d_read = (D + 15) & ~15;    // columns the products read

  // Slice i of this warp (keys 16 (warp + 4 i) ..) into its ring; keys past the end and columns past D are zero.
  auto issue = [&](int32_t i) {
    if (i < mine) {
      const int32_t k0 = (i * kWarps + warp) * kStep;
      const uint32_t dst = ring + (i % NS) * 2 * L::kSliceBytes;
#pragma unroll
      for (int u = 0; u < kStep * CH / 32; ++u) {
        const int idx = lane + 32 * u, row = idx / CH, c = idx % CH;
        if (c * L::kPerChunk < d_read) {
          const bool read = k0 + row < n_keys && c * L::kPerChunk < D;
          const int64_t at = read ? k0 + row : 0;
          const int col = read ? c * 16 : 0;
          cp_async16(dst + chunk_offset<CH>(row, c), k_src + at * k_row + col, read);
          cp_async16(dst + L::kSliceBytes + chunk_offset<CH>(row, c), v_src + at * v_row + col, read);
        }
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < NS - 1; ++i) issue(i);

  // Exponent bytes of the range (8-bit states), keys' then values'.
  uint8_t* exp_s = smem + L::kData;
  if (FP8) {
    const int64_t base = b * p.es[0] + grp * p.es[1] + key0;
    for (int i = threadIdx.x; i < n_keys; i += kThreads) {
      exp_s[i] = p.k_exp[base + i];
      exp_s[p.split_keys + i] = p.v_exp[base + i];
    }
  }

  // Query fragments: rows g and g + 8; the depth order follows the K fragments
  // (16-bit: columns 2t, 2t+1 and 2t+8, 2t+9 of each 16; 8-bit: 4t .. 4t+3).
  uint32_t qa[DP / 16][4];
  float row_scale[2] = {p.scale * kLog2e, p.scale * kLog2e};
#pragma unroll
  for (int hf = 0; hf < 2; ++hf) {
    const int32_t r = row0 + g + 8 * hf;
    const uint16_t* src = nullptr;
    if (r < p.rows) {
      const XaRow x = xa_row(p, inst, r);
      src = static_cast<const uint16_t*>(p.q) + x.b * p.qs[0] + x.h * p.qs[1] + x.m * p.qs[2];
    }
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) {
      const int d0 = kk * 16 + (FP8 ? 4 * t : 2 * t), d1 = d0 + (FP8 ? 2 : 8);
      qa[kk][hf] = src != nullptr && d0 < D ? *reinterpret_cast<const uint32_t*>(src + d0) : 0u;
      qa[kk][2 + hf] = src != nullptr && d1 < D ? *reinterpret_cast<const uint32_t*>(src + d1) : 0u;
    }
    if (FP8 && BF16) {
      // Largest magnitude to [2^14, 2^15): every value within 2^-28 of it is exact in f16.
      float top = 0.f;
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float2 f = bf16x2_to_float2(qa[kk][2 * e + hf]);
          top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
        }
      top = quad_max(top);
      const int e = top >= 1.17549435e-38f ? static_cast<int>(__float_as_uint(top) >> 23) - 127 - 14 : 0;
      const float down = __uint_as_float(static_cast<uint32_t>(127 - (e < -126 ? -126 : e)) << 23);
      row_scale[hf] *= __uint_as_float(static_cast<uint32_t>(127 + (e < -126 ? -126 : e)) << 23);
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float2 f = bf16x2_to_float2(qa[kk][2 * i + hf]);
          qa[kk][2 * i + hf] = pack_f16x2(f.x * down, f.y * down);
        }
    }
  }
  if (FP8) __syncthreads();  // exponents are in

  float o[DP / 8][4];
#pragma unroll
  for (int n = 0; n < DP / 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[n][e] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, mw[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  const int mi = lane >> 3, mr = lane & 7;

  for (int32_t i = 0; i < mine; ++i) {
    cp_async_wait<NS - 2>();
    __syncwarp();
    const uint32_t k_s = ring + (i % NS) * 2 * L::kSliceBytes, v_s = k_s + L::kSliceBytes;
    const int32_t k0 = (i * kWarps + warp) * kStep;
    float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
    if (FP8) {
#pragma unroll
      for (int c = 0; c < CH; c += 2) {
        if (c * 16 >= D) break;
        uint32_t r[4];
        ldmatrix4(k_s + chunk_offset<CH>(mr + ((mi & 1) << 3), c + (mi >> 1)), r);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          if ((c + u) * 16 >= D) break;
#pragma unroll
          for (int n = 0; n < 2; ++n)
            mma16816<false>(s[n], qa[c + u], e4m3x2_to_f16x2(r[2 * u + n]), e4m3x2_to_f16x2(r[2 * u + n] >> 16));
        }
      }
    } else {
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk) {
        if (kk * 16 >= D) break;
        uint32_t r[4];
        ldmatrix4(k_s + chunk_offset<CH>(mr + ((mi >> 1) << 3), 2 * kk + (mi & 1)), r);
        mma16816<MMA_BF16>(s[0], qa[kk], r[0], r[1]);
        mma16816<MMA_BF16>(s[1], qa[kk], r[2], r[3]);
      }
    }
    // Scores of rows g, g + 8 and keys 8 n + 2 t, + 1 in log2 units; padded keys -inf.
    float tv[2][4];                         // with the value's exponent (8-bit states)
    float mx[2] = {-INFINITY, -INFINITY}, mxw[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int32_t key = k0 + 8 * n + 2 * t + (e & 1);
        const int hf = e >> 1;
        float v = s[n][e] * row_scale[hf], w = 0.f;
        if (FP8 && key < n_keys) {
          v *= __uint_as_float(static_cast<uint32_t>(exp_s[key]) << 23);
          w = static_cast<float>(exp_s[p.split_keys + key]) - 127.f;
        }
        v = key < n_keys ? v : -INFINITY;
        s[n][e] = v;
        mx[hf] = max_nan(mx[hf], v);
        if (FP8) {
          tv[n][e] = v + w;
          mxw[hf] = max_nan(mxw[hf], tv[n][e]);
        }
      }
    float ref[2], refw[2], fo[2];
    bool grow = false;
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const float top = max_nan(m[hf], quad_max(mx[hf]));
      const float topw = FP8 ? max_nan(mw[hf], quad_max(mxw[hf])) : top;
      grow = grow || !(top <= m[hf]) || (FP8 && !(topw <= mw[hf]));
      // A row without a score above -inf keeps 0 as its reference.
      ref[hf] = top == -INFINITY ? 0.f : top;
      refw[hf] = topw == -INFINITY ? 0.f : topw;
      l[hf] *= fast_exp2(m[hf] - ref[hf]);
      fo[hf] = FP8 ? fast_exp2(mw[hf] - refw[hf]) : fast_exp2(m[hf] - ref[hf]);
      m[hf] = top;
      mw[hf] = topw;
    }
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int n = 0; n < DP / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][e] *= fo[e >> 1];
    }
    uint32_t pa[4];                         // P as the A operand: keys 2t, 2t+1 | 2t+8, 2t+9
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      float pr[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        pr[e] = fast_exp2(s[n][e] - ref[e >> 1]);
        l[e >> 1] += pr[e];
        if (FP8) pr[e] = fast_exp2(tv[n][e] - refw[e >> 1]);
      }
      pa[2 * n] = pack2<MMA_BF16>(pr[0], pr[1]);
      pa[2 * n + 1] = pack2<MMA_BF16>(pr[2], pr[3]);
    }
#pragma unroll
    for (int c = 0; c < CH; c += 2) {
      if (c * L::kPerChunk >= D) break;
      uint32_t r[4];
      ldmatrix4_trans(v_s + chunk_offset<CH>(mr + ((mi & 1) << 3), c + (mi >> 1)), r);
      if (FP8) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          if ((c + u) * 16 >= D) break;
          // r: keys 2t, 2t+1 of two columns each -> key pairs of the even, then of the odd column
          const uint32_t lo = __byte_perm(r[2 * u], 0u, 0x3120), hi = __byte_perm(r[2 * u + 1], 0u, 0x3120);
          mma16816<false>(o[2 * (c + u)], pa, e4m3x2_to_f16x2(lo), e4m3x2_to_f16x2(hi));
          mma16816<false>(o[2 * (c + u) + 1], pa, e4m3x2_to_f16x2(lo >> 16), e4m3x2_to_f16x2(hi >> 16));
        }
      } else {
        mma16816<MMA_BF16>(o[c], pa, r[0], r[1]);
        mma16816<MMA_BF16>(o[c + 1], pa, r[2], r[3]);
      }
    }
    __syncwarp();
    issue(i + NS - 1);
  }
  cp_async_wait<0>();
  __syncthreads();  // every ring is at rest: the space takes the warps' sums

  float* join = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int hf = 0; hf < 2; ++hf) {
    const int r = g + 8 * hf;
    const float sum = quad_sum(l[hf]);
    if (t == 0) {
      m_s[warp][r] = m[hf];
      l_s[warp][r] = sum;
      w_s[warp][r] = FP8 ? mw[hf] : m[hf];
    }
    if (r < n_rows && mine > 0) {
      float* dst = join + (warp * kXaRowsTile + r) * L::kJoinStride;
      if (FP8) {
#pragma unroll
        for (int c = 0; c < DP / 16; ++c)
          *reinterpret_cast<float4*>(dst + c * 16 + 4 * t) =
              make_float4(o[2 * c][2 * hf], o[2 * c + 1][2 * hf], o[2 * c][2 * hf + 1], o[2 * c + 1][2 * hf + 1]);
      } else {
#pragma unroll
        for (int n = 0; n < DP / 8; ++n)
          *reinterpret_cast<float2*>(dst + n * 8 + 2 * t) = make_float2(o[n][2 * hf], o[n][2 * hf + 1]);
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
          const float4 v = *reinterpret_cast<const float4*>(join + (w * kXaRowsTile + r) * L::kJoinStride + d);
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
}

// out = sum_s 2^(lse_s - max) part_s / sum_s 2^(lse_s - max), one warp per row, parts in order.
template <bool BF16>
__global__ void __launch_bounds__(128)
xattn_combine_kernel(const XaParams p, int32_t n_slots) {
  const int lane = threadIdx.x & 31;
  const int64_t lin = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (lin >= p.rows_total) return;
  float top = -INFINITY;
  for (int s = lane; s < n_slots; s += 32) top = max_nan(top, p.part_lse[s * p.rows_total + lin]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
  const bool none = top == -INFINITY;
  const int d = lane * 4;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float total = 0.f;
#pragma unroll 4
  for (int s = 0; s < n_slots; ++s) {
    const float e = p.part_lse[s * p.rows_total + lin];
    const float w = e == -INFINITY ? 0.f : fast_exp2(e - top);
    total += w;
    if (w != 0.f && d < p.head_dim) {  // an empty part's values were never written
      const float4 v = *reinterpret_cast<const float4*>(p.part_o + (s * p.rows_total + lin) * p.head_dim + d);
      acc.x = fmaf(v.x, w, acc.x);
      acc.y = fmaf(v.y, w, acc.y);
      acc.z = fmaf(v.z, w, acc.z);
      acc.w = fmaf(v.w, w, acc.w);
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

template <int DP, bool BF16, bool FP8>
int32_t launch(const RowsArgs& a, int64_t grid, cudaStream_t stream) {
  using L = RowsShape<DP, FP8>;
  auto kernel = xattn_rows_kernel<DP, BF16, FP8>;
  const int smem = L::kData + (FP8 ? 2 * a.p.split_keys : 0);
  constexpr int most = L::kData + (FP8 ? 2 * kXaRowsKeys8 : 0);
  static std::atomic<uint64_t> done{0};
  if (smem > most) return 8;
  if (!allow_smem(kernel, most, done)) return 6;
  kernel<<<static_cast<unsigned>(grid), kThreads, smem, stream>>>(a);
  return cudaGetLastError() == cudaSuccess ? 0 : 6;
}

template <bool BF16, bool FP8>
int32_t launch_dim(const RowsArgs& a, int64_t grid, cudaStream_t stream) {
  return a.p.head_dim <= 64 ? launch<64, BF16, FP8>(a, grid, stream) : launch<128, BF16, FP8>(a, grid, stream);
}

}  // namespace

int32_t launch_xattn_rows(const XaParams& p, cudaStream_t stream) {
  RowsArgs a;
  a.p = p;
  a.n_rt = (p.rows + kXaRowsTile - 1) / kXaRowsTile;
  const int64_t grid = static_cast<int64_t>(a.n_rt) * p.instances * p.n_split;
  if (grid > INT32_MAX) return 8;
  const bool fp8 = p.k_exp != nullptr, bf16 = p.dtype == 2;
  if (fp8) return bf16 ? launch_dim<true, true>(a, grid, stream) : launch_dim<false, true>(a, grid, stream);
  return bf16 ? launch_dim<true, false>(a, grid, stream) : launch_dim<false, false>(a, grid, stream);
}

int32_t launch_xattn_combine(const XaParams& p, int32_t n_slots, cudaStream_t stream) {
  const int64_t grid = (p.rows_total + 3) / 4;
  if (grid > INT32_MAX) return 8;
  if (p.dtype == 2)
    xattn_combine_kernel<true><<<static_cast<unsigned>(grid), 128, 0, stream>>>(p, n_slots);
  else
    xattn_combine_kernel<false><<<static_cast<unsigned>(grid), 128, 0, stream>>>(p, n_slots);
  return cudaGetLastError() == cudaSuccess ? 0 : 6;
}

}  // namespace intp
