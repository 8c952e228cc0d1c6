// state_cache.cu - the 8-bit cache of key / value states: quantised as written, read back.
//
// A state's row x (D values of one head) is held as e4m3 codes c and one exponent byte
// e + 127 with x ~ c 2^e, e the smallest integer with max|x| <= 448 2^e (448 is e4m3's
// largest value).  A power of two loses nothing that e4m3 keeps: the codes' own three
// mantissa bits bound the error (2^-4 relative for normal codes), and code * 2^e is exact
// in bf16 and fp32.
// Bound by memory: one pass, 32-byte loads and 16-byte code stores a lane.  A lane holds 16
// values, LPR lanes (D / 16, rounded to a power of two) a row, so its maximum is a few shuffles
// of 16-bit integers (magnitudes order like their bits); each lane group takes kUnroll rows at
// once to keep loads in flight.
#include <cstdint>
#include <cstring>
#include "../../include/intp_b200.h"
#include "xattn_common.cuh"
#include "xattn_internal.h"

namespace intp {
namespace {

constexpr int kThreads = 128;
constexpr int kUnroll = 4;

struct CacheArgs {
  int32_t batch, groups, capacity, count, head_dim;
  int32_t blocks;                        // of one sequence and key head
  void* x[2]; int64_t xs[2][3];          // k, v: batch, group, state strides
  uint8_t* codes[2];
  uint8_t* exps[2];
  const int32_t* start; const int32_t* counts;
};

// The rows of one block: consecutive states of one sequence and key head, of k or of v, so what
// a row's place takes of arithmetic is a block's.
struct Rows {
  uint16_t* x; int64_t stride;           // the 16-bit rows
  uint8_t* codes; uint8_t* exps;         // the cache's, of the sequence and head
  int64_t start;                         // cache row of state 0
  int32_t first, counted;                // this thread's first state; states that are copied
};

template <int LPR>
__device__ __forceinline__ Rows block_rows(const CacheArgs& a) {
  const int32_t outer = blockIdx.x / a.blocks, bg = outer >> 1, which = outer & 1;
  const int32_t b = bg / a.groups, g = bg - b * a.groups;
  const int64_t* s = a.xs[which];
  Rows r;
  r.x = static_cast<uint16_t*>(a.x[which]) + b * s[0] + g * s[1];
  r.stride = s[2];
  r.codes = a.codes[which] + static_cast<int64_t>(bg) * a.capacity * a.head_dim;
  r.exps = a.exps[which] + static_cast<int64_t>(bg) * a.capacity;
  r.start = a.start == nullptr ? 0 : a.start[b];
  r.counted = a.counts == nullptr || a.counts[b] > a.count ? a.count : a.counts[b];
  r.first = (blockIdx.x - outer * a.blocks) * (kThreads / LPR * kUnroll) + threadIdx.x / LPR;
  return r;
}
// Cache row of state i, or -1 outside the cache or past the sequence's count.
__device__ __forceinline__ int64_t cache_row(const CacheArgs& a, const Rows& r, int32_t i) {
  const int64_t at = r.start + i;
  return i < r.counted && at >= 0 && at < a.capacity ? at : -1;
}

// The smallest e >= -126 with amax <= 448 * 2^e (448 = 1.75 * 2^8), 0 for amax = 0.
__device__ __forceinline__ int32_t row_exponent(float amax) {
  if (amax == 0.f) return 0;
  const uint32_t bits = __float_as_uint(amax);
  const int32_t e = static_cast<int32_t>(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return e < -126 ? -126 : e;
}
__device__ __forceinline__ float power_of_two(int32_t e) {  // e in [-126, 127]
  return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}

template <int LPR, bool BF16>
__global__ void __launch_bounds__(kThreads)
cache_write_kernel(const CacheArgs a) {
  constexpr int kRowsPer = kThreads / LPR;
  constexpr uint32_t kInf = BF16 ? 0x7f80u : 0x7c00u;     // bits of infinity: magnitudes at or above are not finite
  const int sub = threadIdx.x % LPR;
  const Rows rows = block_rows<LPR>(a);
  const bool col = sub * 16 < a.head_dim;
  int64_t at[kUnroll];
  uint4 v[kUnroll][2];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int32_t i = rows.first + u * kRowsPer;
    at[u] = cache_row(a, rows, i);
    v[u][0] = v[u][1] = make_uint4(0u, 0u, 0u, 0u);
    if (col && at[u] >= 0) {
      const uint4* src = reinterpret_cast<const uint4*>(rows.x + i * rows.stride + sub * 16);
      v[u][0] = __ldcs(src);
      v[u][1] = __ldcs(src + 1);
    }
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    uint32_t w[8] = {v[u][0].x, v[u][0].y, v[u][0].z, v[u][0].w, v[u][1].x, v[u][1].y, v[u][1].z, v[u][1].w};
    uint32_t top = 0u;                   // two running maxima of magnitude bits
#pragma unroll
    for (int e = 0; e < 8; ++e) top = __vmaxu2(top, w[e] & 0x7fff7fffu);
    if ((top & 0xffffu) >= kInf || (top >> 16) >= kInf) {
      // Not finite: such values do not count and become NaN (e4m3 has no infinity).
      top = 0u;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if ((w[e] & 0x7fffu) >= kInf) w[e] |= 0x7fffu;
        else top = __vmaxu2(top, w[e] & 0x7fffu);
        if (((w[e] >> 16) & 0x7fffu) >= kInf) w[e] |= 0x7fff0000u;
        else top = __vmaxu2(top, w[e] & 0x7fff0000u);
      }
    }
#pragma unroll
    for (int s = LPR / 2; s > 0; s >>= 1) top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, s));
    const float2 pair = unpack2<BF16>(top);
    const int32_t e = row_exponent(fmaxf(pair.x, pair.y));
    const float down = power_of_two(-e);
    uint32_t codes[4];
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      uint32_t c[2];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const float2 f = mul2(unpack2<BF16>(w[2 * h + q]), make_float2(down, down));
        asm("{\n\t.reg .b16 h;\n\tcvt.rn.satfinite.e4m3x2.f32 h, %1, %2;\n\tcvt.u32.u16 %0, h;\n\t}"
            : "=r"(c[q])
            : "f"(f.y), "f"(f.x));
      }
      codes[h] = __byte_perm(c[0], c[1], 0x5410);
    }
    if (at[u] >= 0 && col) {
      __stcs(reinterpret_cast<uint4*>(rows.codes + at[u] * a.head_dim + sub * 16),
             make_uint4(codes[0], codes[1], codes[2], codes[3]));
      if (sub == 0) rows.exps[at[u]] = static_cast<uint8_t>(e + 127);
    }
  }
}

// Four codes times 2^e, rounded to the output type.  With `clamp`, values past its range (a
// row's largest may have been rounded up) become its largest finite value.
template <bool BF16>
__device__ __forceinline__ uint2 decode4(uint32_t codes, float up, bool clamp) {
  uint32_t h[2], r[2];
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
      : "=r"(h[0]), "=r"(h[1])
      : "r"(codes));
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float2 f = mul2(unpack2<false>(h[i]), make_float2(up, up));
    if (clamp) {
      const float top = BF16 ? __uint_as_float(0x7f7f0000u) : 65504.f;
      if (f.x == f.x) f.x = fminf(fmaxf(f.x, -top), top);
      if (f.y == f.y) f.y = fminf(fmaxf(f.y, -top), top);
    }
    r[i] = pack2<BF16>(f.x, f.y);
  }
  return make_uint2(r[0], r[1]);
}

template <int LPR, bool BF16>
__global__ void __launch_bounds__(kThreads)
cache_read_kernel(const CacheArgs a) {
  constexpr int kRowsPer = kThreads / LPR;
  constexpr int32_t kSafe = BF16 ? 119 : 7;   // 448 * 2^e is within the type
  const int sub = threadIdx.x % LPR;
  if (sub * 16 >= a.head_dim) return;
  const Rows rows = block_rows<LPR>(a);
  uint4 c[kUnroll];
  int32_t e[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int64_t at = cache_row(a, rows, rows.first + u * kRowsPer);
    c[u] = make_uint4(0u, 0u, 0u, 0u);
    e[u] = 0;
    if (at >= 0) {
      c[u] = __ldcs(reinterpret_cast<const uint4*>(rows.codes + at * a.head_dim + sub * 16));
      e[u] = static_cast<int32_t>(__ldg(rows.exps + at)) - 127;
    }
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int32_t i = rows.first + u * kRowsPer;
    if (i >= a.count) continue;
    const float up = power_of_two(e[u]);
    const bool clamp = e[u] > kSafe;
    const uint2 r0 = decode4<BF16>(c[u].x, up, clamp), r1 = decode4<BF16>(c[u].y, up, clamp);
    const uint2 r2 = decode4<BF16>(c[u].z, up, clamp), r3 = decode4<BF16>(c[u].w, up, clamp);
    uint4* dst = reinterpret_cast<uint4*>(rows.x + i * rows.stride + sub * 16);
    __stcs(dst, make_uint4(r0.x, r0.y, r1.x, r1.y));
    __stcs(dst + 1, make_uint4(r2.x, r2.y, r3.x, r3.y));
  }
}

template <int LPR, bool BF16>
int32_t launch(CacheArgs a, bool write, cudaStream_t stream) {
  constexpr int32_t per = kThreads / LPR * kUnroll;
  a.blocks = static_cast<int32_t>((static_cast<int64_t>(a.count) + per - 1) / per);
  const int64_t grid = 2 * static_cast<int64_t>(a.batch) * a.groups * a.blocks;
  if (grid > INT32_MAX) return INTP_ERR_SHAPE;
  if (write)
    cache_write_kernel<LPR, BF16><<<static_cast<unsigned>(grid), kThreads, 0, stream>>>(a);
  else
    cache_read_kernel<LPR, BF16><<<static_cast<unsigned>(grid), kThreads, 0, stream>>>(a);
  return cudaGetLastError() == cudaSuccess ? INTP_OK : INTP_ERR_LAUNCH;
}

bool row_layout_ok(const void* p, const int64_t* stride, const int64_t* extent) {
  if (reinterpret_cast<uintptr_t>(p) % 16 || stride[3] != 1) return false;
  for (int d = 0; d < 3; ++d)
    if (extent[d] > 1 && (stride[d] <= 0 || stride[d] % 8)) return false;
  return true;
}

int32_t run(const state_cache_args* c, bool write, cudaStream_t stream) {
  if (!c) return INTP_ERR_ARGUMENT;
  if (c->batch < 0 || c->groups < 0 || c->capacity < 0 || c->count < 0) return INTP_ERR_SHAPE;
  if (c->head_dim < 16 || c->head_dim > 128 || c->head_dim % 16) return INTP_ERR_SHAPE;
  if (c->dtype != INTP_F16 && c->dtype != INTP_BF16) return INTP_ERR_DTYPE;
  if (c->batch == 0 || c->groups == 0 || c->count == 0) return INTP_OK;
  for (int64_t n : {c->batch, c->groups, c->capacity, c->count})
    if (n > (int64_t(1) << 30)) return INTP_ERR_SHAPE;
  if (c->batch * c->groups > INT32_MAX / 2) return INTP_ERR_SHAPE;
  if (!c->k || !c->v) return INTP_ERR_ARGUMENT;
  if (c->capacity > 0 && (!c->k_codes || !c->v_codes || !c->k_exponents || !c->v_exponents)) return INTP_ERR_ARGUMENT;
  const int64_t extent[3] = {c->batch, c->groups, c->count};
  if (!row_layout_ok(c->k, c->k_stride, extent) || !row_layout_ok(c->v, c->v_stride, extent)) return INTP_ERR_LAYOUT;
  if (reinterpret_cast<uintptr_t>(c->k_codes) % 16 || reinterpret_cast<uintptr_t>(c->v_codes) % 16)
    return INTP_ERR_LAYOUT;
  if (write && c->capacity == 0) return INTP_OK;  // every row falls outside; a read has zeros to write
  int sms = 0;
  const int32_t device = current_device_facts(&sms);
  if (device != INTP_OK) return device;
  CacheArgs a;
  a.batch = static_cast<int32_t>(c->batch);
  a.groups = static_cast<int32_t>(c->groups);
  a.capacity = static_cast<int32_t>(c->capacity);
  a.count = static_cast<int32_t>(c->count);
  a.head_dim = static_cast<int32_t>(c->head_dim);
  a.x[0] = c->k;
  a.x[1] = c->v;
  std::memcpy(a.xs[0], c->k_stride, sizeof(a.xs[0]));
  std::memcpy(a.xs[1], c->v_stride, sizeof(a.xs[1]));
  a.codes[0] = c->k_codes;
  a.codes[1] = c->v_codes;
  a.exps[0] = c->k_exponents;
  a.exps[1] = c->v_exponents;
  a.start = c->start;
  a.counts = c->counts;
  const bool bf16 = c->dtype == INTP_BF16;
  if (a.head_dim <= 32) return bf16 ? launch<2, true>(a, write, stream) : launch<2, false>(a, write, stream);
  if (a.head_dim <= 64) return bf16 ? launch<4, true>(a, write, stream) : launch<4, false>(a, write, stream);
  return bf16 ? launch<8, true>(a, write, stream) : launch<8, false>(a, write, stream);
}

}  // namespace
}  // namespace intp

extern "C" {

intp_status state_cache_write(const state_cache_args* a, void* stream) {
  return intp::run(a, true, static_cast<cudaStream_t>(stream));
}

intp_status state_cache_read(const state_cache_args* a, void* stream) {
  return intp::run(a, false, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
