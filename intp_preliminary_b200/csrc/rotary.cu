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
// what is left is rounded once to 32 bits (2^-24 of at most pi / 4) before sin and cos.
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
  int32_t heads, first_chunk;            // first_chunk: of the grid's y axis
};

struct RotaryParams {
  Stream s[3];                           // q, k, v; heads = 0 where absent
  const double* turns; const int32_t* axis;
  const void* positions; int64_t ps[3];
  const int32_t* start; const int32_t* counts;
  const int32_t* table; int64_t table_stride;
  int32_t tokens, rows, head_dim, rotary_dim, units, per_chunk;
  int32_t pages, page_size;
  int64_t capacity;
  int32_t position_type;
  bool inverse, paged;
};

// (sin, cos) of 2 pi times `position` turns.
__device__ __forceinline__ float2 turn(double position, double turns) {
  double u = position * turns;
  u -= rint(u);                                     // exact
  const double quarter = rint(4.0 * u);
  float s, c;
  sincospif(2.f * static_cast<float>(u - 0.25 * quarter), &s, &c);
  const int q = static_cast<int>(quarter);
  const float a = (q & 1) ? c : s, b = (q & 1) ? s : c;
  // quarters 0 .. 3: (s, c), (c, -s), (-s, -c), (-c, s)
  return make_float2((q & 2) ? -a : a, ((q + 1) & 2) ? -b : b);
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

// One unit of `n` heads, hs elements apart: two chunks, `two` elements apart (second chunk absent where `single`).
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

  const int chunk_y = blockIdx.y;
  const int which = chunk_y >= p.s[2].first_chunk ? 2 : chunk_y >= p.s[1].first_chunk ? 1 : 0;
  const Stream& s = p.s[which];
  const int32_t h0 = (chunk_y - s.first_chunk) * p.per_chunk;
  const int32_t h1 = h0 + p.per_chunk < s.heads ? h0 + p.per_chunk : s.heads;

  // Columns of the two chunks.
  const int32_t turned = which == 2 ? 0 : p.rotary_dim;
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

  const int64_t at = p.start == nullptr ? row : static_cast<int64_t>(p.start[b]) + row;
  uint8_t* out = static_cast<uint8_t*>(s.out);
  bool write = true;
  if (p.paged && which != 0) {
    // The row's place in the cache; rows without one are not written.
    write = at >= 0 && at < p.capacity && (p.counts == nullptr || row < p.counts[b]);
    if (!write) return;
    const uint32_t index = static_cast<uint32_t>(at) / static_cast<uint32_t>(p.page_size);
    const int32_t page = p.table[b * p.table_stride + index];
    if (page < 0 || page >= p.pages) return;
    out += (page * s.os[0] + (static_cast<uint32_t>(at) - index * static_cast<uint32_t>(p.page_size)) * s.os[2]) * kSize;
  } else {
    out += (b * s.os[0] + row * s.os[2]) * kSize;
  }
  const uint8_t* x = static_cast<const uint8_t*>(s.x) + (b * s.xs[0] + row * s.xs[2]) * kSize;

  C v[kUnroll][2];
  auto fetch = [&](int32_t h) {
#pragma unroll
    for (int i = 0; i < kUnroll; ++i)
      if (h + i < h1) {
        const uint8_t* src = x + (h + i) * s.xs[1] * kSize;
        v[i][0].load(src + c0 * kSize);
        if (pair) v[i][1].load(src + c1 * kSize);
      }
  };
  auto put = [&](int32_t h) {
#pragma unroll
    for (int i = 0; i < kUnroll; ++i)
      if (h + i < h1) {
        uint8_t* dst = out + (h + i) * s.os[1] * kSize;
        v[i][0].store(dst + c0 * kSize);
        if (pair) v[i][1].store(dst + c1 * kSize);
      }
  };
  fetch(h0);
  if (!turns) {
    for (int32_t h = h0;;) {
      put(h);
      h += kUnroll;
      if (h >= h1) return;
      fetch(h);
    }
  }
  float sn[V], cs[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const int32_t i = unit * V + e;
    double position = static_cast<double>(at);
    if (p.position_type != kRow) {
      const int64_t o = b * p.ps[0] + row * p.ps[1] + p.axis[i] * p.ps[2];
      position = p.position_type == kInt32   ? static_cast<double>(static_cast<const int32_t*>(p.positions)[o])
                 : p.position_type == kInt64 ? static_cast<double>(static_cast<const int64_t*>(p.positions)[o])
                                             : static_cast<double>(static_cast<const float*>(p.positions)[o]);
    }
    const float2 r = turn(position, p.turns[i]);
    sn[e] = p.inverse ? -r.x : r.x;
    cs[e] = r.y;
  }
  for (int32_t h = h0;;) {
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      if (h + i >= h1) break;
      float a[V], c[V];
      v[i][0].get(a);
      v[i][1].get(c);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float& one = NEIGHBOURS ? (e < V / 2 ? a[(2 * e) % V] : c[(2 * e) % V]) : a[e];
        float& two = NEIGHBOURS ? (e < V / 2 ? a[(2 * e + 1) % V] : c[(2 * e + 1) % V]) : c[e];
        const float y1 = one * cs[e] - two * sn[e], y2 = two * cs[e] + one * sn[e];
        one = y1;
        two = y2;
      }
      v[i][0].set(a);
      v[i][1].set(c);
    }
    put(h);
    h += kUnroll;
    if (h >= h1) return;
    fetch(h);
  }
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
  // Heads of a thread: as many as leave the GPU full (16 blocks an SM), eight at most.
  int64_t heads = 0;
  for (const Stream& s : p.s) heads += s.heads;
  p.per_chunk = 1;
  while (p.per_chunk < 8 && blocks * heads / (2 * p.per_chunk) >= 148 * 16) p.per_chunk *= 2;
  int64_t chunks = 0;
  for (Stream& s : p.s) {
    s.first_chunk = static_cast<int32_t>(chunks);
    chunks += (s.heads + p.per_chunk - 1) / p.per_chunk;
  }
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
    p.s[i].x = x[i];
    p.s[i].out = out[i];
    p.s[i].heads = static_cast<int32_t>(heads);
    take(p.s[i].xs, xs[i], from);
    take(p.s[i].os, os[i], to);
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
