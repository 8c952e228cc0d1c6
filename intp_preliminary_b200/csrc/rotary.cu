// rotary.cu - queries and keys turned by their positions, and a step's keys and values appended
// to a paged cache with that rotation on the way (sm_100a).
//
// Pair i of a head's first R columns turns by t = position[axis(i)] * frequency(i):
//   y1 = x1 cos t - x2 sin t,  y2 = x2 cos t + x1 sin t.
// Bound by memory: every value is read once and written once.  A thread owns one "unit" of a
// token's row, two 16-byte chunks that hold whole pairs (columns i and R / 2 + i, or neighbours),
// takes its angles once and applies them to several heads, so that the angles' cost is shared and
// many loads are in flight.  Columns past R and rows of v are units that are copied.
//
// Angles: the frequencies come in turns (radians / 2 pi) as 64-bit numbers and the product with the
// position is reduced to an eighth of a turn in 64 bits, so that far positions keep their angle:
// what is left is rounded once to 32 bits and goes through the power series of sin and cos.
//
// Measured on one B200 (us a launch in a CUDA graph; floor at the measured copy rate): q and k of two
// sequences of 16384 tokens, 40 heads of 128, both ways 216 for two launches (205); a prompt of 16 x 4096
// tokens into pages 232 (225); 256 images of 196 tokens, 6 heads of 64, both ways 33 (24), where a thread's
// eight angles cost as much as its six heads; one token of 32 sequences 3.1.  Steps: 64 -> 39 for the
// images with the angles shared over q's and k's heads, 33 with the power series and packed pairs.
#include <cstdint>
#include <cstring>
#include <algorithm>
#include "../../include/intp_b200.h"
#include "xattn_common.cuh"
#include "xattn_internal.h"

namespace intp {
namespace {

constexpr int kThreads = 128;
constexpr int kUnroll = 4;               // heads whose loads are in flight together

enum PositionType : int32_t { kRow = 0, kInt32 = 1, kInt64 = 2, kFloat32 = 3 };

// q, k or v: (sequence, head, row) strides in elements.
struct Stream {
  const void* x; int64_t xs[3];
  void* out; int64_t os[3];              // a cache's: page, head, row
  int32_t heads;
};

struct RotaryParams {
  Stream q, k, v;                        // heads = 0 where absent
  const double* turns; const int32_t* axis;
  const void* positions; int64_t ps[3];
  const int32_t* start; const int32_t* counts;
  const int32_t* table; int64_t table_stride;
  int32_t tokens, rows, head_dim, rotary_dim, units, per_chunk;
  int32_t turned_chunks;                 // of the grid's y axis: q's and k's, then v's
  int32_t pages, page_size;
  int64_t capacity;
  int32_t position_type;
  bool inverse, paged;
};

// (sin, cos) of `turns` times `position` turns: what is left of an eighth of a turn either way goes
// through the power series, whose first term left out is 2e-9 at pi / 4.
__device__ __forceinline__ float2 turn(double position, double turns) {
  double u = position * turns;
  u -= rint(u);                                     // exact
  const double quarter = rint(4.0 * u);
  const float x = 6.283185307f * static_cast<float>(fma(-0.25, quarter, u)), z = x * x;
  float s = fmaf(z, 1.f / 362880.f, -1.f / 5040.f), c = fmaf(z, -1.f / 3628800.f, 1.f / 40320.f);
  s = fmaf(z, s, 1.f / 120.f);
  c = fmaf(z, c, -1.f / 720.f);
  s = fmaf(z, s, -1.f / 6.f);
  c = fmaf(z, c, 1.f / 24.f);
  c = fmaf(z, c, -0.5f);
  s = fmaf(x * z, s, x);
  c = fmaf(z, c, 1.f);
  const int q = static_cast<int>(quarter);
  const float a = (q & 1) ? c : s, b = (q & 1) ? s : c;
  // quarters 0 .. 3: (s, c), (c, -s), (-s, -c), (-c, s)
  return make_float2(__uint_as_float(__float_as_uint(a) ^ ((q & 2u) << 30)),
                     __uint_as_float(__float_as_uint(b) ^ (((q + 1) & 2u) << 30)));
}

template <int T, int V> struct Chunk {   // T: 0 f32, 1 f16, 2 bf16; V values
  static constexpr int kWords = V * (T == 0 ? 4 : 2) / 4;
  uint32_t w[kWords];
  __device__ __forceinline__ void load(const void* p) {
    if constexpr (kWords == 4) {
      const uint4 r = __ldg(static_cast<const uint4*>(p));
      w[0] = r.x; w[1] = r.y; w[2] = r.z; w[3] = r.w;
    } else {
      const uint2 r = __ldg(static_cast<const uint2*>(p));
      w[0] = r.x; w[1] = r.y;
    }
  }
  __device__ __forceinline__ void store(void* p) const {
    if constexpr (kWords == 4)
      *static_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    else
      *static_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  }
  __device__ __forceinline__ void get(float (&f)[V]) const {
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      if constexpr (T == 0) {
        f[i] = __uint_as_float(w[i]);
      } else {
        const float2 p = unpack2<T == 2>(w[i]);
        f[2 * i] = p.x;
        f[2 * i + 1] = p.y;
      }
    }
  }
  __device__ __forceinline__ void set(const float (&f)[V]) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      if constexpr (T == 0) w[i] = __float_as_uint(f[i]);
      else w[i] = pack2<T == 2>(f[2 * i], f[2 * i + 1]);
    }
  }
};

// q's and k's heads stand in a row, v's behind them; a block takes per_chunk of one kind.
template <int T, int V, bool NEIGHBOURS>
__global__ void __launch_bounds__(kThreads)
rotary_kernel(const RotaryParams p) {
  using C = Chunk<T, V>;
  constexpr int kSize = T == 0 ? 4 : 2;
  const int32_t in_block = threadIdx.x / p.units, unit = threadIdx.x - in_block * p.units;
  const int32_t per_block = kThreads / p.units;
  const int64_t token = static_cast<int64_t>(blockIdx.x) * per_block + in_block;
  if (in_block >= per_block || token >= p.tokens) return;
  const int32_t b = static_cast<int32_t>(token) / p.rows, row = static_cast<int32_t>(token) - b * p.rows;

  const bool copied = static_cast<int32_t>(blockIdx.y) >= p.turned_chunks;   // v
  const int32_t n_q = copied ? 0 : p.q.heads;
  const Stream& two = copied ? p.v : p.k;
  const int32_t h0 = (blockIdx.y - (copied ? p.turned_chunks : 0)) * p.per_chunk;
  const int32_t h1 = min(h0 + p.per_chunk, n_q + two.heads);

  // Columns of the two chunks.
  const int32_t turned = copied ? 0 : p.rotary_dim;
  const int32_t turned_units = turned / (2 * V);
  const bool turns = unit < turned_units;
  int32_t c0, c1;
  if (turns) {
    c0 = NEIGHBOURS ? 2 * V * unit : V * unit;
    c1 = NEIGHBOURS ? c0 + V : turned / 2 + c0;
  } else {
    c0 = turned + 2 * V * (unit - turned_units);
    c1 = c0 + V;
  }
  if (c0 >= p.head_dim) return;
  const bool pair = c1 < p.head_dim;

  // This thread's heads: of q, then of k (or of v alone).
  const int32_t q0 = min(h0, n_q), n0 = min(h1, n_q) - q0, two0 = max(h0, n_q) - n_q, n1 = max(h1, n_q) - n_q - two0;
  const int64_t step_q = p.q.xs[1] * kSize, step_two = two.xs[1] * kSize;
  const uint8_t* x_q = static_cast<const uint8_t*>(p.q.x) + (b * p.q.xs[0] + row * p.q.xs[2] + c0) * kSize + q0 * step_q;
  const uint8_t* x_two = static_cast<const uint8_t*>(two.x) + (b * two.xs[0] + row * two.xs[2] + c0) * kSize + two0 * step_two;
  const int32_t apart = (c1 - c0) * kSize;
  C v[kUnroll][2];
  auto fetch = [&](const uint8_t* src, int64_t step, int32_t n) {
#pragma unroll
    for (int i = 0; i < kUnroll; ++i)
      if (i < n) {
        v[i][0].load(src + i * step);
        if (pair) v[i][1].load(src + i * step + apart);
      }
  };
  if (n0 > 0)
    fetch(x_q, step_q, n0);
  else
    fetch(x_two, step_two, n1);

  const int64_t at = p.start == nullptr ? row : static_cast<int64_t>(p.start[b]) + row;
  // The row's place in the cache: its page is asked for before the angles and used after them.
  int32_t page = -1;
  uint32_t page_row = 0;
  if (p.paged && n1 > 0 && at >= 0 && at < p.capacity && (p.counts == nullptr || row < p.counts[b])) {
    const uint32_t index = static_cast<uint32_t>(at) / static_cast<uint32_t>(p.page_size);
    page = __ldg(p.table + b * p.table_stride + index);
    page_row = static_cast<uint32_t>(at) - index * static_cast<uint32_t>(p.page_size);
  }
  float2 sn[V / 2], cs[V / 2];              // of two pairs each
  if (turns) {
    double position = static_cast<double>(at);
    int32_t last = -1;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int32_t i = unit * V + e;
      if (p.position_type != kRow) {
        const int32_t axis = __ldg(p.axis + i);
        if (axis != last) {                 // neighbouring pairs mostly turn by one axis
          last = axis;
          const int64_t o = b * p.ps[0] + row * p.ps[1] + axis * p.ps[2];
          position = p.position_type == kInt32   ? static_cast<double>(static_cast<const int32_t*>(p.positions)[o])
                     : p.position_type == kInt64 ? static_cast<double>(static_cast<const int64_t*>(p.positions)[o])
                                                 : static_cast<double>(static_cast<const float*>(p.positions)[o]);
        }
      }
      const float2 r = turn(position, __ldg(p.turns + i));
      (e & 1 ? sn[e / 2].y : sn[e / 2].x) = p.inverse ? -r.x : r.x;
      (e & 1 ? cs[e / 2].y : cs[e / 2].x) = r.y;
    }
  }
  auto turn_pairs = [&](C& first, C& second) {
    float a[V], c[V];
    first.get(a);
    second.get(c);
#pragma unroll
    for (int e = 0; e < V; e += 2) {        // pairs e and e + 1
      float* f = e < V / 2 ? a : c;         // NEIGHBOURS: where they stand
      const int o = (2 * e) % V;
      const float2 one = NEIGHBOURS ? make_float2(f[o], f[o + 2]) : make_float2(a[e], a[e + 1]);
      const float2 other = NEIGHBOURS ? make_float2(f[o + 1], f[o + 3]) : make_float2(c[e], c[e + 1]);
      const float2 y1 = fma2(other, make_float2(-sn[e / 2].x, -sn[e / 2].y), mul2(one, cs[e / 2]));
      const float2 y2 = fma2(one, sn[e / 2], mul2(other, cs[e / 2]));
      if (NEIGHBOURS) {
        f[o] = y1.x;
        f[o + 1] = y2.x;
        f[o + 2] = y1.y;
        f[o + 3] = y2.y;
      } else {
        a[e] = y1.x;
        a[e + 1] = y1.y;
        c[e] = y2.x;
        c[e + 1] = y2.y;
      }
    }
    first.set(a);
    second.set(c);
  };
  // n heads, the first of which are in v.
  auto finish = [&](const uint8_t* src, int64_t step, uint8_t* dst, int64_t out_step, int32_t n) {
    while (true) {
#pragma unroll
      for (int i = 0; i < kUnroll; ++i)
        if (i < n) {
          if (turns) turn_pairs(v[i][0], v[i][1]);
          v[i][0].store(dst + i * out_step);
          if (pair) v[i][1].store(dst + i * out_step + apart);
        }
      n -= kUnroll;
      if (n <= 0) return;
      src += kUnroll * step;
      dst += kUnroll * out_step;
      fetch(src, step, n);
    }
  };
  if (n0 > 0) {
    finish(x_q, step_q, static_cast<uint8_t*>(p.q.out) + (b * p.q.os[0] + row * p.q.os[2] + c0 + q0 * p.q.os[1]) * kSize,
           p.q.os[1] * kSize, n0);
    if (n1 <= 0) return;
    fetch(x_two, step_two, n1);
  }
  uint8_t* out_two = static_cast<uint8_t*>(two.out) + (c0 + two0 * two.os[1]) * kSize;
  if (p.paged) {
    if (page < 0 || page >= p.pages) return;  // rows without a place are not written
    out_two += (page * two.os[0] + page_row * two.os[2]) * kSize;
  } else {
    out_two += (b * two.os[0] + row * two.os[2]) * kSize;
  }
  finish(x_two, step_two, out_two, two.os[1] * kSize, n1);
}

constexpr int64_t kMaxSize = int64_t(1) << 30;

// Unit stride along D, 16-byte rows, strides that are multiples of 16 bytes below 2^40 bytes; `broadcast` allows zero.
bool rows_ok(const void* x, const int64_t* stride, const int64_t* extent, int64_t size, bool broadcast) {
  if (reinterpret_cast<uintptr_t>(x) % 16 || stride[3] != 1) return false;
  for (int d = 0; d < 3; ++d)
    if (extent[d] > 1 && (stride[d] < (broadcast ? 0 : 1) || stride[d] * size % 16 || stride[d] >= (int64_t(1) << 40) / size))
      return false;
  return true;
}

void take(int64_t* dst, const int64_t* src, const int64_t* extent) {
  for (int d = 0; d < 3; ++d) dst[d] = extent[d] > 1 ? src[d] : 0;
}

template <int T, int V, bool NEIGHBOURS>
int32_t launch(RotaryParams p, cudaStream_t stream) {
  p.units = std::max((p.rotary_dim / V + 1) / 2 + ((p.head_dim - p.rotary_dim) / V + 1) / 2, (p.head_dim / V + 1) / 2);
  const int64_t per_block = kThreads / p.units;
  const int64_t blocks = (p.tokens + per_block - 1) / per_block;
  // Heads of a thread, which shares its angles among them: as many as leave four blocks an SM (eight:
  // a training step of B256 H3 N196 D64 36.3 us instead of 33.1, B16 H12 N512 in 32 bits 11.8 instead of 12.6).
  const int64_t turned = p.q.heads + p.k.heads, heads = turned + p.v.heads;
  p.per_chunk = 1;
  while (p.per_chunk < 64 && blocks * heads / (2 * p.per_chunk) >= 148 * 4) p.per_chunk *= 2;
  const int64_t of_q_k = (turned + p.per_chunk - 1) / p.per_chunk, chunks = of_q_k + (p.v.heads + p.per_chunk - 1) / p.per_chunk;
  p.turned_chunks = static_cast<int32_t>(of_q_k);
  if (blocks > INT32_MAX || chunks > 65535) return INTP_ERR_SHAPE;
  rotary_kernel<T, V, NEIGHBOURS><<<dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(chunks)), kThreads, 0, stream>>>(p);
  return cudaGetLastError() == cudaSuccess ? INTP_OK : INTP_ERR_LAUNCH;
}

template <int T, int V>
int32_t launch_pairs(const RotaryParams& p, bool neighbours, cudaStream_t stream) {
  return neighbours ? launch<T, V, true>(p, stream) : launch<T, V, false>(p, stream);
}

intp_status run(const rotary_args* a, bool paged, cudaStream_t stream) {
  if (!a) return INTP_ERR_ARGUMENT;
  for (int64_t n : {a->batch, a->heads, a->groups, a->rows, a->pages, a->page_size, a->table_width})
    if (n < 0 || n > kMaxSize) return INTP_ERR_SHAPE;
  if (a->batch * a->rows > INT32_MAX - kThreads) return INTP_ERR_SHAPE;
  if (a->head_dim < 8 || a->head_dim > 128 || a->head_dim % 8) return INTP_ERR_SHAPE;
  if (a->rotary_dim < 0 || a->rotary_dim > a->head_dim || a->rotary_dim % 8) return INTP_ERR_SHAPE;
  if (a->dtype != INTP_F16 && a->dtype != INTP_BF16 && !(a->dtype == INTP_F32 && !paged)) return INTP_ERR_DTYPE;
  if (a->position_type < kRow || a->position_type > kFloat32) return INTP_ERR_ARGUMENT;
  if (!paged && (a->v || a->page_table || a->counts || a->position_type == kRow)) return INTP_ERR_ARGUMENT;
  if (paged && a->page_size < 1) return INTP_ERR_SHAPE;
  if (a->batch == 0 || a->rows == 0) return INTP_OK;
  if (a->position_type != kRow && !a->positions) return INTP_ERR_ARGUMENT;
  if (a->rotary_dim > 0 && (!a->turns || !a->axis)) return INTP_ERR_ARGUMENT;
  if (paged && (!a->k || !a->v || !a->page_table)) return INTP_ERR_ARGUMENT;
  const int64_t size = a->dtype == INTP_F32 ? 4 : 2;
  RotaryParams p;
  std::memset(&p, 0, sizeof(p));
  const void* x[3] = {a->q, a->k, a->v};
  void* out[3] = {a->q_out, a->k_out, a->v_out};
  const int64_t* xs[3] = {a->q_stride, a->k_stride, a->v_stride};
  const int64_t* os[3] = {a->q_out_stride, a->k_out_stride, a->v_out_stride};
  bool any = false;
  for (int i = 0; i < 3; ++i) {
    const int64_t heads = i == 0 ? a->heads : a->groups;
    if (!x[i] || heads == 0) continue;
    const bool cache = paged && i > 0;
    if (cache && a->pages == 0) continue;  // nothing has a place
    const int64_t from[3] = {a->batch, heads, a->rows};
    const int64_t to[3] = {cache ? a->pages : a->batch, heads, cache ? a->page_size : a->rows};
    if (!out[i]) return INTP_ERR_ARGUMENT;
    if (!rows_ok(x[i], xs[i], from, size, true) || !rows_ok(out[i], os[i], to, size, false)) return INTP_ERR_LAYOUT;
    Stream& s = i == 0 ? p.q : i == 1 ? p.k : p.v;
    s.x = x[i];
    s.out = out[i];
    s.heads = static_cast<int32_t>(heads);
    take(s.xs, xs[i], from);
    take(s.os, os[i], to);
    any = true;
  }
  if (!any) return INTP_OK;
  int sms = 0;
  const int32_t device = current_device_facts(&sms);
  if (device != INTP_OK) return device;
  p.turns = a->turns;
  p.axis = a->axis;
  p.positions = a->positions;
  std::memcpy(p.ps, a->position_stride, sizeof(p.ps));
  p.start = a->start;
  p.counts = a->counts;
  p.table = a->page_table;
  p.table_stride = a->table_stride;
  p.tokens = static_cast<int32_t>(a->batch * a->rows);
  p.rows = static_cast<int32_t>(a->rows);
  p.head_dim = static_cast<int32_t>(a->head_dim);
  p.rotary_dim = static_cast<int32_t>(a->rotary_dim);
  p.pages = static_cast<int32_t>(a->pages);
  p.page_size = static_cast<int32_t>(std::max<int64_t>(a->page_size, 1));
  // positions past 2^31 - 1 have no place: a row number is a 32-bit one
  p.capacity = std::min<int64_t>(a->table_width * a->page_size, INT32_MAX);
  p.position_type = a->position_type;
  p.inverse = a->inverse != 0;
  p.paged = paged;
  const bool neighbours = a->interleaved != 0;
  if (a->dtype == INTP_F32) return launch_pairs<0, 4>(p, neighbours, stream);
  // 16-byte chunks hold 8 values: with 8 columns more or less than a multiple of 16 to turn, halves do
  // not start on one, and chunks are 8 bytes.
  const bool wide = a->rotary_dim % 16 == 0;
  if (a->dtype == INTP_BF16) return wide ? launch_pairs<2, 8>(p, neighbours, stream) : launch_pairs<2, 4>(p, neighbours, stream);
  return wide ? launch_pairs<1, 8>(p, neighbours, stream) : launch_pairs<1, 4>(p, neighbours, stream);
}

}  // namespace
}  // namespace intp

extern "C" {

intp_status rotary_positions(const rotary_args* a, void* stream) {
  return intp::run(a, false, static_cast<cudaStream_t>(stream));
}

intp_status paged_cache_append(const rotary_args* a, void* stream) {
  return intp::run(a, true, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
