// xattn_common.cuh - device pieces that the tensor-core cross-attention kernels share.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "sm100_ptx.cuh"

namespace intp {

// mbar_wait of a whole warp in step: every lane gets the same answer, so the warp stays
// converged around the .aligned instructions that follow.  A budget below the hardware's
// suspend quantum is spun out, so that it is kept to the letter.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t phase, volatile int32_t* abort, int32_t* status,
                                          int32_t code, uint64_t budget_ns) {
  const uint32_t parity = phase & 1;
  if (__all_sync(0xffffffffu, mbar_test_wait(bar, parity))) return true;
  const uint64_t start = global_ns();
  const bool spin = budget_ns < 2000ull;
  while (true) {
    const bool done = spin ? mbar_test_wait(bar, parity) : mbar_try_wait(bar, parity);
    if (__all_sync(0xffffffffu, done)) return true;
    if (__any_sync(0xffffffffu, *abort != 0)) return false;
    if (__any_sync(0xffffffffu, global_ns() - start > budget_ns)) {
      *abort = 1;
      if (status) atomicCAS(status, 0, code);
      return false;
    }
  }
}

// Programmatic dependent launch within one call: the next kernel may start once every CTA of
// this one has said so (or left); it waits where it needs this one's results, and at the latest
// before its own end, so that a kernel's end always means its predecessors' too.  Both are
// no-ops in a kernel that was launched plainly.
__device__ __forceinline__ void allow_next_kernel() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_previous_kernel() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  return BF16 ? pack_bf16x2(lo, hi) : pack_f16x2(lo, hi);
}
// Cut off instead of rounded.
template <bool BF16>
__device__ __forceinline__ uint32_t pack2_down(float lo, float hi) {
  uint32_t d;
  if (BF16)
    asm("cvt.rz.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  else
    asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
  if (BF16) return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}

// Both values with infinities (and NaN) at the type's largest finite value.
template <bool BF16>
__device__ __forceinline__ uint32_t finite2(uint32_t v) {
  if (BF16) {
    const uint32_t top = 0x7f7f7f7fu, bottom = 0xff7fff7fu;
    __nv_bfloat162 r = *reinterpret_cast<const __nv_bfloat162*>(&v);
    r = __hmax2(__hmin2(r, *reinterpret_cast<const __nv_bfloat162*>(&top)), *reinterpret_cast<const __nv_bfloat162*>(&bottom));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  const uint32_t top = 0x7bff7bffu, bottom = 0xfbfffbffu;
  __half2 r = *reinterpret_cast<const __half2*>(&v);
  r = __hmax2(__hmin2(r, *reinterpret_cast<const __half2*>(&top)), *reinterpret_cast<const __half2*>(&bottom));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// All bits of those of the two values that are infinities or NaN.
template <bool BF16>
__device__ __forceinline__ uint32_t not_finite2(uint32_t v) {
  constexpr uint32_t kExp = BF16 ? 0x7f80u : 0x7c00u;
  return ((v & kExp) == kExp ? 0xffffu : 0u) | ((v >> 16 & kExp) == kExp ? 0xffff0000u : 0u);
}

// 32 bytes of one thread, a whole memory sector (dst 32-byte aligned).
__device__ __forceinline__ void store32(void* dst, uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t e, uint32_t f,
                                        uint32_t g, uint32_t h) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(a), "r"(b), "r"(c), "r"(d),
               "r"(e), "r"(f), "r"(g), "r"(h)
               : "memory");
}
// 16 columns [c0, c0 + 16) of a row-per-thread result: fp32 to `part` if it is not null, else
// rounded to 16 bits to `dst`; `wide` says that 16-bit rows are 32-byte aligned.  Rows differ
// by thread, so a store is worth a sector each or it is worth less.
template <bool BF16>
__device__ __forceinline__ void store16(const float (&v)[16], uint16_t* dst, float* part, bool wide, int32_t c0,
                                        int32_t head_dim) {
  if (part != nullptr) {
#pragma unroll
    for (int e = 0; e < 16; e += 8)
      if (c0 + e < head_dim)
        store32(part + c0 + e, __float_as_uint(v[e]), __float_as_uint(v[e + 1]), __float_as_uint(v[e + 2]),
                __float_as_uint(v[e + 3]), __float_as_uint(v[e + 4]), __float_as_uint(v[e + 5]), __float_as_uint(v[e + 6]),
                __float_as_uint(v[e + 7]));
    return;
  }
  uint32_t w[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) w[e] = pack2<BF16>(v[2 * e], v[2 * e + 1]);
  if (wide) {
    if (c0 < head_dim) store32(dst + c0, w[0], w[1], w[2], w[3], w[4], w[5], w[6], w[7]);
    return;
  }
  if (c0 < head_dim) *reinterpret_cast<uint4*>(dst + c0) = make_uint4(w[0], w[1], w[2], w[3]);
  if (c0 + 8 < head_dim) *reinterpret_cast<uint4*>(dst + c0 + 8) = make_uint4(w[4], w[5], w[6], w[7]);
}

}  // namespace intp
