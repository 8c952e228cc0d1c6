// xattn_internal.h - kernel-side parameters shared by the cross-attention
// kernels and their C-ABI dispatcher (cross_attention_capi.cu).
#pragma once
#include <atomic>
#include <cstdint>
#include <cuda_runtime.h>
#include "sla_internal.h"

namespace intp {

// One pass of query rows over key / value states.  An "instance" is a set of
// rows that read the same states: the rows of one sequence and key head
// (r = g * queries + m over the key head's query heads g), or, for a shared
// prefix, the rows of every sequence for one key head
// (r = (b * heads/groups + g) * queries + m).
struct XaParams {
  int32_t batch, heads, groups, queries, states, head_dim;
  int32_t per_group;           // heads / groups
  int32_t shared;              // 1: the states belong to every sequence (no batch dimension)
  int32_t rows;                // rows of an instance
  int32_t instances;
  float scale;
  int32_t dtype;               // 1 f16, 2 bf16
  const void* q; int64_t qs[3];
  const void* k; int64_t ks[3];  // batch, group, state
  const void* v; int64_t vs[3];
  const uint8_t* k_exp; const uint8_t* v_exp; int64_t es[2];
  // Few-rows kernel only: states that every sequence reads before its own (group and state
  // strides as in ks, vs), in one unsplit pass.
  const void* pre_k; const void* pre_v; int64_t pre_ks[2], pre_vs[2];
  int32_t prefix;
  const int32_t* lengths;
  void* out; int64_t os[3];
  float* lse;
  // Split passes: slot part_first + s of part_o [slot][rows_total][head_dim]
  // (normalised, fp32) and part_lse [slot][rows_total] (log2 units), row =
  // (b * heads + h) * queries + m.  part_o null: the pass writes out / lse itself.
  float* part_o; float* part_lse;
  int64_t rows_total;
  int32_t n_split, split_keys, part_first;
  int32_t warps;               // few-rows kernel: warps of a CTA (4 or 8)
  int32_t* status;
  uint64_t wait_ns;
};

struct XaBwdParams {
  XaParams f;
  const void* dout; int64_t ds[3];
  void* dq; void* dk; void* dv;      // 16-bit, contiguous; null when not wanted
  float* delta;                      // row statistics: [B * H][ceil(M / 64)][-lse 64 | -delta 64]
  // f16 only, what bounds dS: the length |dO| of a query row, [B * H][ceil(M / 64)][64]; the largest of
  // that and of |delta| in 64 rows, two numbers each; the length |v| of a state, [B * G][N], and the
  // largest of 64 states, [B * G][ceil(N / 64)].
  float* row_norm; float* tile_max; float* v_norm; float* v_max;
  // Splits of the streamed axis: fp32 partial sums [split][elements], null when 1.
  float* dq_part; int32_t dq_split, dq_split_tiles;
  float* dk_part; float* dv_part; int32_t kv_split, kv_split_tiles;
};

// SMs of the current device, asked for once; an error status where it is not sm_100.
int32_t current_device_facts(int* sms);

// Raises a kernel's dynamic shared memory limit, once per device (`done` is the kernel's own).
template <class K>
inline bool allow_smem(K kernel, int bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
  if (done.load(std::memory_order_relaxed) & bit) return true;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
  done.fetch_or(bit, std::memory_order_relaxed);
  return true;
}

// Launches a kernel that may overlap the end of the one before it on the stream (`overlap`), or plainly.
template <class... P, class... A>
inline bool launch_kernel(void (*kernel)(P...), dim3 grid, int threads, int smem, cudaStream_t stream, bool overlap,
                          A&&... args) {
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = overlap ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...) == cudaSuccess;
}

constexpr int kXaTileRows = 256;   // rows of a tcgen05 work item (two warpgroups of 128)
constexpr int kXaTileKeys = 128;
constexpr int kXaRowsTile = 16;    // rows of a few-rows work item
constexpr int kXaRowsKeys8 = 2048; // keys of an 8-bit part at most: their exponents sit in shared memory

// `overlap`: the call's second pass; it does not read what the first one writes.
int32_t launch_xattn_tiles(const XaParams& p, cudaStream_t stream, int sm_count, bool overlap);
int32_t launch_xattn_rows(const XaParams& p, cudaStream_t stream, bool overlap);
// Joins n slots of part_o / part_lse into out / lse.
int32_t launch_xattn_combine(const XaParams& p, int32_t n_slots, cudaStream_t stream);
int32_t launch_xattn_backward(const XaBwdParams& p, cudaStream_t stream, int sm_count);

// Row r of instance `inst`: sequence, head and query.
struct XaRow {
  int32_t b, h, m;
};
__device__ __forceinline__ XaRow xa_row(const XaParams& p, int32_t inst, int32_t r) {
  XaRow x;
  if (p.shared) {
    const int32_t bg = r / p.queries;
    x.m = r - bg * p.queries;
    x.b = bg / p.per_group;
    x.h = inst * p.per_group + (bg - x.b * p.per_group);
  } else {
    const int32_t g = r / p.queries;
    x.m = r - g * p.queries;
    x.b = inst / p.groups;
    x.h = (inst - x.b * p.groups) * p.per_group + g;
  }
  return x;
}
__device__ __forceinline__ int64_t xa_linear(const XaParams& p, const XaRow& x) {
  return (static_cast<int64_t>(x.b) * p.heads + x.h) * p.queries + x.m;
}
// States of an instance's sequence, clamped to what is there.
__device__ __forceinline__ int32_t xa_length(const XaParams& p, int32_t b) {
  if (p.shared || p.lengths == nullptr) return p.states;
  const int32_t l = p.lengths[b];
  return l < 0 ? 0 : (l > p.states ? p.states : l);
}

}  // namespace intp
