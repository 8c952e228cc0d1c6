// xattn_common.cuh - device pieces that the tensor-core cross-attention kernels share.
#pragma once
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

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  return BF16 ? pack_bf16x2(lo, hi) : pack_f16x2(lo, hi);
}
template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
  if (BF16) return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}

}  // namespace intp
