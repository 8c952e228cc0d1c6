// state_cache.cu - the 8-bit cache of key / value states: quantised as written, read back.
//
// A state's row x (D values of one head) is held as e4m3 codes c and one exponent byte
// e + 127 with x ~ c 2^e, e the smallest integer with max|x| <= 448 2^e (448 is e4m3's
// largest value).  A power of two loses nothing that e4m3 keeps: the codes' own three
// mantissa bits bound the error (2^-4 relative for normal codes), and code * 2^e is exact
// in bf16 and fp32.
// Bound by memory: one pass, 16-byte loads, 8-byte code stores.  LPR = D / 8 lanes (rounded
// to a power of two) hold a row, so its maximum is a few shuffles; each lane group takes
// kUnroll rows at once to keep loads in flight.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>
#include <cstring>
#include "../../include/intp_b200.h"
#include "sm100_ptx.cuh"

namespace intp {
namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 4;

struct CacheArgs {
  int32_t batch, groups, capacity, count, head_dim;
  int64_t n_rows;                        // of k (as many again of v)
  void* x[2]; int64_t xs[2][3];          // k, v: batch, group, state strides
  uint8_t* codes[2];
  uint8_t* exps[2];
  const int32_t* start; const int32_t* counts;
};

struct RowAt {
  int32_t which, b, g, i;
  int64_t cache;                         // cache row, or -1 outside it / past the sequence's count
};

__device__ __forceinline__ RowAt row_at(const CacheArgs& a, int64_t row) {
  RowAt r;
  r.which = row >= a.n_rows ? 1 : 0;
  uint32_t x = static_cast<uint32_t>(row - (r.which ? a.n_rows : 0));  // n_rows < 2^31 (checked on the host)
  const uint32_t bg = x / static_cast<uint32_t>(a.count);
  r.i = static_cast<int32_t>(x - bg * a.count);
  r.b = static_cast<int32_t>(bg / a.groups);
  r.g = static_cast<int32_t>(bg - r.b * a.groups);
  const int64_t at = (a.start == nullptr ? 0 : static_cast<int64_t>(a.start[r.b])) + r.i;
  const bool in = at >= 0 && at < a.capacity && (a.counts == nullptr || r.i < a.counts[r.b]);
  r.cache = in ? (static_cast<int64_t>(r.b) * a.groups + r.g) * a.capacity + at : -1;
  return r;
}

template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
  if (BF16) return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
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
  const int sub = threadIdx.x % LPR;
  const int64_t first = (static_cast<int64_t>(blockIdx.x) * kUnroll) * kRowsPer + threadIdx.x / LPR;
  const bool col = sub * 8 < a.head_dim;
  RowAt at[kUnroll];
  uint4 v[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int64_t row = first + u * kRowsPer;
    at[u].cache = -1;
    v[u] = make_uint4(0u, 0u, 0u, 0u);
    if (row < 2 * a.n_rows) {
      at[u] = row_at(a, row);
      if (col && at[u].cache >= 0) {
        const int64_t* s = a.xs[at[u].which];
        v[u] = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.x[at[u].which]) + at[u].b * s[0] +
                                                    at[u].g * s[1] + at[u].i * s[2] + sub * 8));
      }
    }
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const uint32_t w[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
    float f[8];
    float amax = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 p = unpack2<BF16>(w[e]);
      f[2 * e] = p.x;
      f[2 * e + 1] = p.y;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float m = fabsf(f[e]);
      if (m < INFINITY)
        amax = fmaxf(amax, m);
      else
        f[e] = __uint_as_float(0x7fffffffu);  // e4m3 has no infinity: infinities and NaN are its NaN
    }
#pragma unroll
    for (int s = LPR / 2; s > 0; s >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, s));
    const int32_t e = row_exponent(amax);
    const float down = power_of_two(-e);
    uint32_t codes[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t c[2];
#pragma unroll
      for (int q = 0; q < 2; ++q)
        asm("{\n\t.reg .b16 h;\n\tcvt.rn.satfinite.e4m3x2.f32 h, %1, %2;\n\tcvt.u32.u16 %0, h;\n\t}"
            : "=r"(c[q])
            : "f"(f[4 * h + 2 * q + 1] * down), "f"(f[4 * h + 2 * q] * down));
      codes[h] = c[0] | (c[1] << 16);
    }
    if (at[u].cache >= 0 && col) {
      *reinterpret_cast<uint2*>(a.codes[at[u].which] + at[u].cache * a.head_dim + sub * 8) =
          make_uint2(codes[0], codes[1]);
      if (sub == 0) a.exps[at[u].which][at[u].cache] = static_cast<uint8_t>(e + 127);
    }
  }
}

// Two codes times 2^e, rounded to the output type; values past its range (a row's largest
// may have been rounded up) become its largest finite value.
template <bool BF16>
__device__ __forceinline__ uint32_t decode2(uint32_t codes, float up) {
  uint32_t h;
  asm("{\n\t.reg .b16 c;\n\tcvt.u16.u32 c, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, c;\n\t}" : "=r"(h) : "r"(codes & 0xffffu));
  float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
  f.x *= up;
  f.y *= up;
  const float top = BF16 ? __uint_as_float(0x7f7f0000u) : 65504.f;
  if (f.x == f.x) f.x = fminf(fmaxf(f.x, -top), top);
  if (f.y == f.y) f.y = fminf(fmaxf(f.y, -top), top);
  return BF16 ? pack_bf16x2(f.x, f.y) : pack_f16x2(f.x, f.y);
}

template <int LPR, bool BF16>
__global__ void __launch_bounds__(kThreads)
cache_read_kernel(const CacheArgs a) {
  constexpr int kRowsPer = kThreads / LPR;
  const int sub = threadIdx.x % LPR;
  if (sub * 8 >= a.head_dim) return;
  const int64_t first = (static_cast<int64_t>(blockIdx.x) * kUnroll) * kRowsPer + threadIdx.x / LPR;
  RowAt at[kUnroll];
  uint2 c[kUnroll];
  uint32_t e[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int64_t row = first + u * kRowsPer;
    at[u].cache = -1;
    c[u] = make_uint2(0u, 0u);
    e[u] = 127u;
    if (row < 2 * a.n_rows) {
      at[u] = row_at(a, row);
      if (at[u].cache >= 0) {
        c[u] = __ldg(reinterpret_cast<const uint2*>(a.codes[at[u].which] + at[u].cache * a.head_dim + sub * 8));
        e[u] = __ldg(a.exps[at[u].which] + at[u].cache);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    if (first + u * kRowsPer >= 2 * a.n_rows) continue;
    const float up = power_of_two(static_cast<int32_t>(e[u]) - 127);
    const int64_t* s = a.xs[at[u].which];
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.x[at[u].which]) + at[u].b * s[0] + at[u].g * s[1] +
                              at[u].i * s[2] + sub * 8) =
        make_uint4(decode2<BF16>(c[u].x, up), decode2<BF16>(c[u].x >> 16, up), decode2<BF16>(c[u].y, up),
                   decode2<BF16>(c[u].y >> 16, up));
  }
}

template <int LPR, bool BF16>
int32_t launch(const CacheArgs& a, bool write, cudaStream_t stream) {
  const int64_t per = static_cast<int64_t>(kThreads / LPR) * kUnroll;
  const int64_t grid = (2 * a.n_rows + per - 1) / per;
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
    if (n > INT32_MAX) return INTP_ERR_SHAPE;
  if (c->batch * c->groups > INT32_MAX / c->count) return INTP_ERR_SHAPE;
  if (!c->k || !c->v || !c->k_codes || !c->v_codes || !c->k_exponents || !c->v_exponents) return INTP_ERR_ARGUMENT;
  const int64_t extent[3] = {c->batch, c->groups, c->count};
  if (!row_layout_ok(c->k, c->k_stride, extent) || !row_layout_ok(c->v, c->v_stride, extent)) return INTP_ERR_LAYOUT;
  if (reinterpret_cast<uintptr_t>(c->k_codes) % 16 || reinterpret_cast<uintptr_t>(c->v_codes) % 16)
    return INTP_ERR_LAYOUT;
  int dev = 0, major = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess)
    return INTP_ERR_LAUNCH;
  if (major != 10) return INTP_ERR_ARCH;
  CacheArgs a;
  a.batch = static_cast<int32_t>(c->batch);
  a.groups = static_cast<int32_t>(c->groups);
  a.capacity = static_cast<int32_t>(c->capacity);
  a.count = static_cast<int32_t>(c->count);
  a.head_dim = static_cast<int32_t>(c->head_dim);
  a.n_rows = c->batch * c->groups * c->count;
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
  if (a.head_dim <= 32) return bf16 ? launch<4, true>(a, write, stream) : launch<4, false>(a, write, stream);
  if (a.head_dim <= 64) return bf16 ? launch<8, true>(a, write, stream) : launch<8, false>(a, write, stream);
  return bf16 ? launch<16, true>(a, write, stream) : launch<16, false>(a, write, stream);
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
