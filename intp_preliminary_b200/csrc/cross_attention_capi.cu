// cross_attention_capi.cu - extern "C" boundary of the cross-attention operators
// (include/intp_b200.h): checks, the choice of kernel and of splits,
// workspace layout, launches.  No exception crosses it and nothing allocates
// device memory.
#include <cuda_runtime.h>
#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>
#include <cstring>
#include "../../include/intp_b200.h"
#include "sla_tc_common.cuh"
#include "xattn_internal.h"

namespace {

using intp::XaBwdParams;
using intp::XaParams;

constexpr int64_t kPlanSms = 148;            // SMs of a B200: the splits' target
constexpr int64_t kMaxInt = (int64_t(1) << 31) - 1;

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t align256(int64_t n) { return (n + 255) / 256 * 256; }

// Unit stride along D, 16-byte rows, positive 16-byte-multiple strides below 2^40 bytes where there is more than one element.
bool layout_ok(const void* p, const int64_t* stride, const int64_t* extent, int dims, int64_t elem) {
  if (reinterpret_cast<uintptr_t>(p) % 16 || stride[dims] != 1) return false;
  for (int d = 0; d < dims; ++d)
    if (extent[d] > 1 && (stride[d] <= 0 || stride[d] * elem % 16 || stride[d] * elem >= (int64_t(1) << 40)))
      return false;
  return true;
}

// Strides of one-element dimensions are never used; a tensor map still wants them valid.
void take_strides(int64_t* dst, const int64_t* src, const int64_t* extent, int dims, int64_t head_dim) {
  for (int d = 0; d < dims; ++d) dst[d] = extent[d] > 1 ? src[d] : (head_dim + 15) / 16 * 16;
}

intp_status check_shape(const xattn_args* a) {
  for (int64_t n : {a->batch, a->heads, a->groups, a->queries, a->states, a->prefix})
    if (n < 0 || n > (int64_t(1) << 30)) return INTP_ERR_SHAPE;
  if (a->heads < 1 || a->groups < 1 || a->heads % a->groups) return INTP_ERR_SHAPE;
  const int64_t unit = a->eight_bit ? 16 : 8;
  if (a->head_dim < unit || a->head_dim > 128 || a->head_dim % unit) return INTP_ERR_SHAPE;
  if (a->dtype != INTP_F16 && a->dtype != INTP_BF16) return INTP_ERR_DTYPE;
  if (!std::isfinite(a->scale) || !(a->scale > 0.f)) return INTP_ERR_ARGUMENT;
  if (a->kernel < XATTN_KERNEL_AUTO || a->kernel > XATTN_KERNEL_TILES) return INTP_ERR_ARGUMENT;
  if (a->eight_bit != 0 && a->eight_bit != 1) return INTP_ERR_ARGUMENT;
  if (a->eight_bit && a->kernel == XATTN_KERNEL_TILES) return INTP_ERR_UNSUPPORTED;
  // Rows of an instance, instances and their tiles are 32-bit numbers in the kernels, the end of
  // the last row tile among them.
  if (a->batch * a->heads > (kMaxInt - intp::kXaTileRows) / std::max<int64_t>(a->queries, 1)) return INTP_ERR_SHAPE;
  return INTP_OK;
}

struct Pass {
  bool tiles;            // tcgen05 kernel, else the few-rows kernel
  int64_t n_split, split_keys;
  int32_t warps;         // of a few-rows CTA
};

// Rows of an instance up to which the few-rows kernel is taken.  It reads the states once for each
// 16 rows, a 128-row tcgen05 tile costs the same for 1 row as for 128: at B64 G8 N2000 D128 16 rows
// take 91.6 us (tiles 104.4), 24 rows 159.3 (105.0).
constexpr int64_t kRowsMax = 16;
// While a few states and CTAs fill no more than the SMs, more rows cost it nothing: 64 rows at
// B8 G4 N300 D64 7.2 us (tiles 9.0), at B1 G3 N196 6.5 (7.7).
constexpr int64_t kRowsMaxSmall = 64, kSmallStates = 512;

bool few_rows(int64_t rows, int64_t instances, int64_t states) {
  return rows <= kRowsMax || (rows <= kRowsMaxSmall && states <= kSmallStates &&
                              instances * ceil_div(rows, intp::kXaRowsTile) <= kPlanSms);
}

// Few states and no more CTAs than SMs: one part, read by 8 warps, and no second launch that
// joins parts.  Measured, one part against several (a pass among others, and on the GPU alone):
// 600 states of D128 10.7 / 14.6 us (8.4 / 8.0), 1000 of D64 10.5 / 13.7 (9.0 / 6.9), 1000 of D128
// 12.4 / 14.6 (11.0 / 7.5), 1500 of D128 16.5 / 14.7 (14.4 / 7.7).
bool one_part(int64_t items, int64_t states) { return items <= kPlanSms && states <= 1024; }

Pass plan_pass(const xattn_args* a, int64_t rows, int64_t instances, int64_t states) {
  Pass s;
  s.tiles = a->kernel == XATTN_KERNEL_TILES ||
            (a->kernel == XATTN_KERNEL_AUTO && !a->eight_bit && !few_rows(rows, instances, states));
  if (s.tiles) {
    // One CTA per SM: the key axis is split until every SM has work, two tiles a part at least.
    const int64_t items = instances * ceil_div(rows, intp::kXaTileRows), tiles = ceil_div(states, intp::kXaTileKeys);
    int64_t split = items >= kPlanSms ? 1 : std::min(kPlanSms / items, std::max<int64_t>(tiles / 2, 1));
    s.split_keys = ceil_div(tiles, split) * intp::kXaTileKeys;
  } else {
    const int64_t items = instances * ceil_div(rows, intp::kXaRowsTile);
    int64_t split = 1;
    if (one_part(items, states)) {
      s.warps = 8;
    } else {
      // As many CTAs as the GPU holds at once: two an SM, four of 8-bit states.  At B32 G8 N1000
      // D128 that is one part, 24.9 us (two: 30.4, five: 34.7); at B8 G8 N4000 of 8 bits nine
      // parts, 17.7 us (four: 21.3).  Parts of 128 keys at least (B2 G2 N1000: 7.7 us, of 256
      // 9.2), of 256 where there would be more than 16 (N16000: 18.5 us, of 128 29.1).
      s.warps = 4;
      const int64_t held = kPlanSms * (a->eight_bit ? 4 : 2);
      split = std::min({std::max<int64_t>(held / items, 1), ceil_div(states, 128),
                        std::max<int64_t>(ceil_div(states, 256), 16)});
      if (a->eight_bit) split = std::max(split, ceil_div(states, intp::kXaRowsKeys8));
    }
    s.split_keys = ceil_div(ceil_div(states, split), 128) * 128;
  }
  s.n_split = ceil_div(states, s.split_keys);
  return s;
}

// Whether a shared prefix is better read by each sequence before its own states, in one pass and
// one launch, than once for all rows with its part joined by a third kernel: few rows and few
// states.  Measured, one pass against three (prefix + own states, re-read bytes): 196 + 33
// 4.9 / 10.0 us (B4 G3 D64, 0.6 MB) and 13.6 / 24.4 us (B64 G8 D128, 51 MB), 512 + 256 13.1 / 17.9
// us (8 MB), 512 + 64 22.3 / 24.6 us (134 MB), 1024 + 256 19.3 / 18.9 us (17 MB), 1024 + 64
// 36.4 / 25.6 us (268 MB), 2048 + 256 31.8 / 19.0 us (34 MB).
constexpr int64_t kJoinedStates = 1024, kJoinedBytes = 128 << 20;

bool joined_prefix(const xattn_args* a) {
  const int64_t per_group = a->heads / a->groups;
  return a->prefix > 0 && a->kernel != XATTN_KERNEL_TILES && !a->eight_bit && per_group * a->queries <= kRowsMax &&
         a->prefix + a->states <= kJoinedStates && a->batch * a->groups * a->prefix * a->head_dim * 4 <= kJoinedBytes;
}

struct Plan {
  bool joined;
  Pass own, pre;
  int64_t own_slots, pre_slots;      // parts written to the workspace
  int64_t rows_total, o_bytes, bytes;
  bool parts;
};

Plan plan_forward(const xattn_args* a) {
  Plan p{};
  const int64_t per_group = a->heads / a->groups;
  p.rows_total = a->batch * a->heads * a->queries;
  p.joined = joined_prefix(a);
  if (p.joined) {
    p.own.n_split = 1;
    p.own.split_keys = std::max<int64_t>(a->states, 1);
    p.own.warps = a->batch * a->groups * ceil_div(per_group * a->queries, intp::kXaRowsTile) <= kPlanSms ? 8 : 4;
    p.own_slots = 1;
    return p;
  }
  if (a->states > 0) {
    p.own = plan_pass(a, per_group * a->queries, a->batch * a->groups, a->states);
    p.own_slots = p.own.n_split;
  }
  if (a->prefix > 0) {
    p.pre = plan_pass(a, a->batch * per_group * a->queries, a->groups, a->prefix);
    p.pre_slots = p.pre.n_split;
  }
  p.parts = p.own_slots + p.pre_slots > 1;
  if (p.parts) {
    const int64_t slots = p.own_slots + p.pre_slots;
    p.o_bytes = align256(slots * p.rows_total * a->head_dim * 4);
    p.bytes = p.o_bytes + align256(slots * p.rows_total * 4);
  }
  return p;
}

// Checks pointers and layouts and fills the parameters that every pass shares.
intp_status to_params(const xattn_args* a, XaParams* p) {
  const int64_t elem = a->eight_bit ? 1 : 2;
  const int64_t eq[3] = {a->batch, a->heads, a->queries}, ek[3] = {a->batch, a->groups, a->states};
  const int64_t ep[2] = {a->groups, a->prefix};
  if (!a->q || !a->out || !a->status) return INTP_ERR_ARGUMENT;
  if ((a->k_exponents != nullptr) != (a->eight_bit == 1 && a->states > 0) ||
      (a->v_exponents != nullptr) != (a->eight_bit == 1 && a->states > 0))
    return INTP_ERR_ARGUMENT;
  if (!layout_ok(a->q, a->q_stride, eq, 3, 2) || !layout_ok(a->out, a->out_stride, eq, 3, 2)) return INTP_ERR_LAYOUT;
  if (a->states > 0) {
    if (!a->k || !a->v) return INTP_ERR_ARGUMENT;
    if (!layout_ok(a->k, a->k_stride, ek, 3, elem) || !layout_ok(a->v, a->v_stride, ek, 3, elem))
      return INTP_ERR_LAYOUT;
  }
  if (a->prefix > 0) {
    if (!a->prefix_k || !a->prefix_v) return INTP_ERR_ARGUMENT;
    if (!layout_ok(a->prefix_k, a->prefix_k_stride, ep, 2, 2) || !layout_ok(a->prefix_v, a->prefix_v_stride, ep, 2, 2))
      return INTP_ERR_LAYOUT;
  }
  std::memset(p, 0, sizeof(*p));
  p->batch = static_cast<int32_t>(a->batch);
  p->heads = static_cast<int32_t>(a->heads);
  p->groups = static_cast<int32_t>(a->groups);
  p->queries = static_cast<int32_t>(a->queries);
  p->states = static_cast<int32_t>(a->states);
  p->head_dim = static_cast<int32_t>(a->head_dim);
  p->per_group = static_cast<int32_t>(a->heads / a->groups);
  p->rows = static_cast<int32_t>(p->per_group * a->queries);
  p->instances = static_cast<int32_t>(a->batch * a->groups);
  p->scale = a->scale;
  p->dtype = a->dtype;
  p->q = a->q;
  take_strides(p->qs, a->q_stride, eq, 3, a->head_dim);
  p->k = a->k;
  take_strides(p->ks, a->k_stride, ek, 3, a->head_dim);
  p->v = a->v;
  take_strides(p->vs, a->v_stride, ek, 3, a->head_dim);
  p->k_exp = a->k_exponents;
  p->v_exp = a->v_exponents;
  p->es[0] = a->exponent_stride[0];
  p->es[1] = a->exponent_stride[1];
  p->lengths = a->lengths;
  p->out = a->out;
  take_strides(p->os, a->out_stride, eq, 3, a->head_dim);
  p->lse = a->lse;
  p->rows_total = a->batch * a->heads * a->queries;
  p->n_split = 1;
  p->split_keys = p->states;
  p->status = a->status;
  p->wait_ns = intp::tc_wait_budget_ns();
  return INTP_OK;
}

int32_t launch_pass(XaParams p, const Pass& s, int64_t first, cudaStream_t stream, int sms, bool overlap) {
  p.n_split = static_cast<int32_t>(s.n_split);
  p.split_keys = static_cast<int32_t>(s.split_keys);
  p.part_first = static_cast<int32_t>(first);
  p.warps = s.warps;
  return s.tiles ? intp::launch_xattn_tiles(p, stream, sms, overlap) : intp::launch_xattn_rows(p, stream, overlap);
}

struct BackwardPlan {
  int64_t row_norm, tile_max, v_norm, v_max;         // byte offsets (f16); the statistics come first
  int64_t dq_part, dk_part, dv_part, bytes;          // byte offsets; 0 = no part buffer
  int32_t dq_split, dq_tiles, kv_split, kv_tiles;
};

// The streamed axis is split until every SM has an item, four 64-wide tiles a part at least.
void plan_split(int64_t items, int64_t tiles, int32_t* split, int32_t* split_tiles) {
  const int64_t want =
      items >= kPlanSms ? 1 : std::min(kPlanSms / std::max<int64_t>(items, 1), std::max<int64_t>(tiles / 4, 1));
  *split_tiles = static_cast<int32_t>(std::max<int64_t>(ceil_div(tiles, want), 1));
  *split = static_cast<int32_t>(std::max<int64_t>(ceil_div(tiles, *split_tiles), 1));
}

BackwardPlan plan_backward(const xattn_backward_args* b) {
  const xattn_args* a = &b->fwd;
  BackwardPlan p{};
  const int64_t m64 = ceil_div(a->queries, 64), n64 = ceil_div(a->states, 64);
  plan_split(a->batch * a->heads * ceil_div(a->queries, 128), n64, &p.dq_split, &p.dq_tiles);
  plan_split(a->batch * a->groups * ceil_div(a->states, 128), m64 * (a->heads / a->groups), &p.kv_split, &p.kv_tiles);
  const int64_t row_tiles = a->batch * a->heads * m64;
  int64_t at = align256(row_tiles * 128 * 4);
  if (a->dtype == INTP_F16) {
    p.row_norm = at;
    at += align256(row_tiles * 64 * 4);
    p.tile_max = at;
    at += align256(row_tiles * 2 * 4);
    p.v_norm = at;
    at += align256(a->batch * a->groups * a->states * 4);
    p.v_max = at;
    at += align256(a->batch * a->groups * n64 * 4);
  }
  const int64_t nq = a->batch * a->heads * a->queries * a->head_dim * 4;
  const int64_t nk = a->batch * a->groups * a->states * a->head_dim * 4;
  if (p.dq_split > 1) {
    p.dq_part = at;
    at += align256(p.dq_split * nq);
  }
  if (p.kv_split > 1) {
    p.dk_part = at;
    at += align256(p.kv_split * nk);
    p.dv_part = at;
    at += align256(p.kv_split * nk);
  }
  p.bytes = at;
  return p;
}

bool workspace_ok(const xattn_args* a, int64_t bytes) {
  return bytes == 0 ||
         (a->workspace && reinterpret_cast<uintptr_t>(a->workspace) % 256 == 0 && a->workspace_bytes >= bytes);
}

}  // namespace

namespace intp {
int32_t current_device_facts(int* sms) {
  static std::atomic<int> known[64];   // 0: not asked; else SMs + 1, negative if not sm_100
  int dev = 0, major = 0, count = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return INTP_ERR_LAUNCH;
  int v = dev < 64 ? known[dev].load(std::memory_order_relaxed) : 0;
  if (v == 0) {
    if (cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&count, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
      return INTP_ERR_LAUNCH;
    v = major == 10 ? count + 1 : -1;
    if (dev < 64) known[dev].store(v, std::memory_order_relaxed);
  }
  *sms = v - 1;
  return v > 0 ? INTP_OK : INTP_ERR_ARCH;
}
}  // namespace intp

extern "C" {

intp_status xattn_forward_workspace(const xattn_args* a, int64_t* bytes) {
  if (!a || !bytes) return INTP_ERR_ARGUMENT;
  const intp_status st = check_shape(a);
  if (st != INTP_OK) return st;
  *bytes = a->batch == 0 || a->queries == 0 ? 0 : plan_forward(a).bytes;
  return INTP_OK;
}

intp_status xattn_backward_workspace(const xattn_backward_args* b, int64_t* bytes) {
  if (!b || !bytes) return INTP_ERR_ARGUMENT;
  const intp_status st = check_shape(&b->fwd);
  if (st != INTP_OK) return st;
  *bytes = b->fwd.batch == 0 || b->fwd.queries == 0 || b->fwd.states == 0 ? 0 : plan_backward(b).bytes;
  return INTP_OK;
}

intp_status xattn_forward(const xattn_args* a, void* stream) {
  if (!a) return INTP_ERR_ARGUMENT;
  intp_status st = check_shape(a);
  if (st != INTP_OK) return st;
  if (a->batch == 0 || a->queries == 0) return INTP_OK;
  if (a->states == 0 && a->prefix == 0) return INTP_ERR_SHAPE;
  if (a->prefix > 0 && a->prefix_k == nullptr) return INTP_ERR_ARGUMENT;
  XaParams p;
  st = to_params(a, &p);
  if (st != INTP_OK) return st;
  const Plan plan = plan_forward(a);
  if (!workspace_ok(a, plan.bytes)) return INTP_ERR_ARGUMENT;
  int sms = 0;
  st = intp::current_device_facts(&sms);
  if (st != INTP_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (plan.parts) {
    p.part_o = static_cast<float*>(a->workspace);
    p.part_lse = reinterpret_cast<float*>(static_cast<uint8_t*>(a->workspace) + plan.o_bytes);
  }
  const int64_t ep[2] = {a->groups, a->prefix};
  if (plan.joined) {
    p.pre_k = a->prefix_k;
    p.pre_v = a->prefix_v;
    take_strides(p.pre_ks, a->prefix_k_stride, ep, 2, a->head_dim);
    take_strides(p.pre_vs, a->prefix_v_stride, ep, 2, a->head_dim);
    p.prefix = static_cast<int32_t>(a->prefix);
    return launch_pass(p, plan.own, 0, s, sms, false);
  }
  if (a->states > 0) {
    st = launch_pass(p, plan.own, 0, s, sms, false);
    if (st != INTP_OK) return st;
  }
  if (a->prefix > 0) {
    // After the own states' pass, which ends in a partly filled GPU: this one moves in.
    XaParams x = p;
    x.shared = 1;
    x.states = static_cast<int32_t>(a->prefix);
    x.rows = static_cast<int32_t>(a->batch * x.per_group * a->queries);
    x.instances = x.groups;
    x.k = a->prefix_k;
    x.v = a->prefix_v;
    x.k_exp = x.v_exp = nullptr;
    x.ks[0] = x.vs[0] = 0;
    take_strides(x.ks + 1, a->prefix_k_stride, ep, 2, a->head_dim);
    take_strides(x.vs + 1, a->prefix_v_stride, ep, 2, a->head_dim);
    st = launch_pass(x, plan.pre, plan.own_slots, s, sms, a->states > 0);
    if (st != INTP_OK) return st;
  }
  if (!plan.parts) return INTP_OK;
  return intp::launch_xattn_combine(p, static_cast<int32_t>(plan.own_slots + plan.pre_slots), s);
}

intp_status xattn_backward(const xattn_backward_args* b, void* stream) {
  if (!b) return INTP_ERR_ARGUMENT;
  const xattn_args* a = &b->fwd;
  intp_status st = check_shape(a);
  if (st != INTP_OK) return st;
  if (a->eight_bit || a->prefix > 0) return INTP_ERR_UNSUPPORTED;
  if (a->batch == 0) return INTP_OK;
  if (a->queries == 0) {
    // No row reads the states: their gradients are there, and zero.
    const size_t bytes = static_cast<size_t>(a->batch) * a->groups * a->states * a->head_dim * 2;
    for (void* g : {b->grad_k, b->grad_v})
      if (g != nullptr && bytes > 0 && cudaMemsetAsync(g, 0, bytes, static_cast<cudaStream_t>(stream)) != cudaSuccess)
        return INTP_ERR_LAUNCH;
    return INTP_OK;
  }
  if (a->states == 0) return INTP_ERR_SHAPE;
  if (!b->grad_q && !b->grad_k && !b->grad_v) return INTP_OK;
  if (!a->lse || !b->grad_out) return INTP_ERR_ARGUMENT;
  XaBwdParams p;
  std::memset(&p, 0, sizeof(p));
  st = to_params(a, &p.f);
  if (st != INTP_OK) return st;
  const int64_t eq[3] = {a->batch, a->heads, a->queries};
  if (!layout_ok(b->grad_out, b->grad_out_stride, eq, 3, 2)) return INTP_ERR_LAYOUT;
  for (const void* g : {b->grad_q, b->grad_k, b->grad_v})
    if (reinterpret_cast<uintptr_t>(g) % 16) return INTP_ERR_LAYOUT;
  const BackwardPlan plan = plan_backward(b);
  if (!workspace_ok(a, plan.bytes)) return INTP_ERR_ARGUMENT;
  int sms = 0;
  st = intp::current_device_facts(&sms);
  if (st != INTP_OK) return st;
  uint8_t* ws = static_cast<uint8_t*>(a->workspace);
  p.dout = b->grad_out;
  take_strides(p.ds, b->grad_out_stride, eq, 3, a->head_dim);
  p.dq = b->grad_q;
  p.dk = b->grad_k;
  p.dv = b->grad_v;
  p.delta = reinterpret_cast<float*>(ws);
  if (a->dtype == INTP_F16) {
    p.row_norm = reinterpret_cast<float*>(ws + plan.row_norm);
    p.tile_max = reinterpret_cast<float*>(ws + plan.tile_max);
    p.v_norm = reinterpret_cast<float*>(ws + plan.v_norm);
    p.v_max = reinterpret_cast<float*>(ws + plan.v_max);
  }
  p.dq_part = plan.dq_part ? reinterpret_cast<float*>(ws + plan.dq_part) : nullptr;
  p.dk_part = plan.dk_part ? reinterpret_cast<float*>(ws + plan.dk_part) : nullptr;
  p.dv_part = plan.dv_part ? reinterpret_cast<float*>(ws + plan.dv_part) : nullptr;
  p.dq_split = plan.dq_split;
  p.dq_split_tiles = plan.dq_tiles;
  p.kv_split = plan.kv_split;
  p.kv_split_tiles = plan.kv_tiles;
  return intp::launch_xattn_backward(p, static_cast<cudaStream_t>(stream), sms);
}

}  // extern "C"
