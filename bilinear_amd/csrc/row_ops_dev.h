// Device helpers of the row operators (row_norm.hip, row_dropout.hip): 8-element units of a row, wave and block sums,
// and the draws of the regenerated dropout mask.
//
// Unit: 8 consecutive columns of one row, owned by one lane in every kernel and every type — one 16-byte access for
// bf16 / fp16, two for fp32 — and exactly the elements one Philox call draws for.  A row may start at any multiple of
// the element size (odd widths, rows that are slices of a wider tensor): units are copied with the element's own
// alignment, which gfx950 serves as ordinary 16-byte accesses.
#pragma once
#include <type_traits>

#include "common.h"
#include "philox.h"

namespace blh {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;
static constexpr int ROW_UNIT = 8;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// a unit as it lies in memory: 4 registers for 16-bit types, 8 for fp32
template <typename T> struct RawUnit {
  typedef u32x4 vec __attribute__((aligned(2)));
  u32x4 q;
  __device__ __forceinline__ void load(const T* p) { q = *reinterpret_cast<const vec*>(p); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<vec*>(p) = q; }
  __device__ __forceinline__ void zero() { q = u32x4{0, 0, 0, 0}; }
  // drop the first k elements (1 .. 7), zeros enter behind
  __device__ __forceinline__ void shift(int k) {
    uint64_t lo = (uint64_t)q[1] << 32 | q[0], hi = (uint64_t)q[3] << 32 | q[2];
    const int s = 16 * k;
    lo = s < 64 ? lo >> s | hi << (64 - s) : hi >> (s - 64);
    hi = s < 64 ? hi >> s : 0;
    q = u32x4{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
  }
  // the same, the dropped elements enter behind
  __device__ __forceinline__ void rotate(int k) {
    if (k & 4) q = u32x4{q[2], q[3], q[0], q[1]};
    if (k & 2) q = u32x4{q[1], q[2], q[3], q[0]};
    if (k & 1)
      q = u32x4{q[0] >> 16 | q[1] << 16, q[1] >> 16 | q[2] << 16, q[2] >> 16 | q[3] << 16, q[3] >> 16 | q[0] << 16};
  }
  // the first n elements (1 .. 7)
  __device__ __forceinline__ void store_some(T* p, int n) const {
    typedef uint64_t w4 __attribute__((aligned(2)));
    typedef uint32_t w2 __attribute__((aligned(2)));
    uint64_t v = (uint64_t)q[1] << 32 | q[0];
    if (n & 4) {
      *reinterpret_cast<w4*>(p) = v;
      p += 4;
      v = (uint64_t)q[3] << 32 | q[2];
    }
    if (n & 2) {
      *reinterpret_cast<w2*>(p) = (uint32_t)v;
      p += 2;
      v >>= 32;
    }
    if (n & 1) *reinterpret_cast<uint16_t*>(p) = (uint16_t)v;
  }
  __device__ __forceinline__ float get(int e) const {
    const uint32_t w = q[e >> 1];
    if constexpr (std::is_same<T, bf16_t>::value) return __uint_as_float((e & 1) ? w & 0xffff0000u : w << 16);
    return (float)__builtin_bit_cast(f16_t, (uint16_t)((e & 1) ? w >> 16 : w));
  }
  __device__ __forceinline__ void set(const float (&f)[ROW_UNIT]) {
    typedef T pair __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int k = 0; k < 4; ++k) q[k] = __builtin_bit_cast(uint32_t, pair{(T)f[2 * k], (T)f[2 * k + 1]});
  }
};
template <> struct RawUnit<float> {
  typedef f32x4 vec __attribute__((aligned(4)));
  f32x4 q[2];
  __device__ __forceinline__ void load(const float* p) {
    q[0] = *reinterpret_cast<const vec*>(p);
    q[1] = *reinterpret_cast<const vec*>(p + 4);
  }
  __device__ __forceinline__ void store(float* p) const {
    *reinterpret_cast<vec*>(p) = q[0];
    *reinterpret_cast<vec*>(p + 4) = q[1];
  }
  __device__ __forceinline__ void zero() { q[0] = q[1] = f32x4{0.f, 0.f, 0.f, 0.f}; }
  __device__ __forceinline__ void shift(int k) {
    if (k & 4) { q[0] = q[1]; q[1] = f32x4{0.f, 0.f, 0.f, 0.f}; }
    if (k & 2) { q[0] = f32x4{q[0][2], q[0][3], q[1][0], q[1][1]}; q[1] = f32x4{q[1][2], q[1][3], 0.f, 0.f}; }
    if (k & 1) { q[0] = f32x4{q[0][1], q[0][2], q[0][3], q[1][0]}; q[1] = f32x4{q[1][1], q[1][2], q[1][3], 0.f}; }
  }
  __device__ __forceinline__ void rotate(int k) {
    const f32x4 a = q[0], b = q[1];
    if (k & 4) { q[0] = b; q[1] = a; }
    const f32x4 c = q[0], d = q[1];
    if (k & 2) { q[0] = f32x4{c[2], c[3], d[0], d[1]}; q[1] = f32x4{d[2], d[3], c[0], c[1]}; }
    const f32x4 u = q[0], v = q[1];
    if (k & 1) { q[0] = f32x4{u[1], u[2], u[3], v[0]}; q[1] = f32x4{v[1], v[2], v[3], u[0]}; }
  }
  __device__ __forceinline__ void store_some(float* p, int n) const {
    typedef float pair __attribute__((ext_vector_type(2)));
    typedef pair pair4 __attribute__((aligned(4)));
    f32x4 v = q[0];
    if (n & 4) {
      *reinterpret_cast<vec*>(p) = v;
      p += 4;
      v = q[1];
    }
    if (n & 2) {
      *reinterpret_cast<pair4*>(p) = pair{v[0], v[1]};
      p += 2;
      v[0] = v[2];
    }
    if (n & 1) *p = v[0];
  }
  __device__ __forceinline__ float get(int e) const { return q[e >> 2][e & 3]; }
  __device__ __forceinline__ void set(const float (&f)[ROW_UNIT]) {
#pragma unroll
    for (int e = 0; e < ROW_UNIT; ++e) q[e >> 2][e & 3] = f[e];
  }
};

// The unit row[c .. c + 8) of a row of `width` elements, in two steps so that no load waits for another:
//   load_raw  reads 16 (32) bytes without a branch — a unit that crosses the row's end, or lies behind it, reads the row's
//             last 8 elements instead, which lie inside the row (SHORT: rows of fewer than 8 elements, element by element to
//             the same places);
//   settle    moves such a unit down and leaves zeros behind the row's end; `width` 0 makes it all zeros;
//   settle2   settles a gradient and, beside it, what is normalised, with elements of the same row (of the last one, in a group
//             without a row) behind the row's end: (0 - mean) rstd may pass the largest number, whose product with the gradient's
//             0 is NaN, where a row's own elements make NaN only if the row's results are.
// (16384 x 1001 fp16: layer norm 12.2 us, backward 24.7; with the shift inside the load 18.9 and 29.9, with a branch around
// element loads 14.7 and 27.0; 16384 x 1000 takes 12.0 and 23.4.)
template <bool SHORT, typename T> __device__ __forceinline__ RawUnit<T> load_raw(const T* row, int c, int width) {
  RawUnit<T> r;
  if constexpr (!SHORT) {
    r.load(row + min(c, width - ROW_UNIT));
  } else {
    float f[ROW_UNIT];
#pragma unroll
    for (int e = 0; e < ROW_UNIT; ++e) f[e] = (float)row[max(0, e - (ROW_UNIT - width))];
    r.set(f);
  }
  return r;
}
template <typename T> __device__ __forceinline__ void settle(RawUnit<T>& r, int c, int width) {
  if (c + ROW_UNIT > width) {
    if (c < width) r.shift(c + ROW_UNIT - width);
    else r.zero();
  }
}
template <typename T, typename R> __device__ __forceinline__ void settle2(RawUnit<T>& d, RawUnit<R>& f, int c, int width) {
  if (c + ROW_UNIT > width) {
    if (c < width) {
      f.rotate(c + ROW_UNIT - width);
      d.shift(c + ROW_UNIT - width);
    } else {
      d.zero();
    }
  }
}

template <bool SHORT, typename T>
__device__ __forceinline__ void load_unit(const T* row, int c, int width, float (&f)[ROW_UNIT]) {
  RawUnit<T> r = load_raw<SHORT>(row, c, width);
  settle(r, c, width);
#pragma unroll
  for (int e = 0; e < ROW_UNIT; ++e) f[e] = r.get(e);
}

// row[c .. c + 8) = f, nothing at or behind `width`
template <typename T>
__device__ __forceinline__ void store_unit(T* row, int c, int width, const float (&f)[ROW_UNIT]) {
  RawUnit<T> r;
  r.set(f);
  if (c + ROW_UNIT <= width) r.store(row + c);
  else if (c < width) r.store_some(row + c, width - c);
}

// weight / bias: fp32 or the activations' type (`same`), or absent (nullptr: `absent` everywhere)
template <bool SHORT, typename T>
__device__ __forceinline__ void load_param_unit(const void* p, bool same, int c, int width, float absent,
                                                float (&f)[ROW_UNIT]) {
  if (!p) {
#pragma unroll
    for (int e = 0; e < ROW_UNIT; ++e) f[e] = absent;
  } else if (same) {
    load_unit<SHORT>(static_cast<const T*>(p), c, width, f);
  } else {
    load_unit<SHORT>(static_cast<const float*>(p), c, width, f);
  }
}

template <int CTRL, int ROWS = 0xf> __device__ __forceinline__ float dpp_add(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, ROWS, 0xf, false));
}

// sum over groups of LANES consecutive lanes (8, 16, 32 or 64), in every lane; all 64 lanes take part.  Each step pairs
// lanes that hold the same partial sum's two halves, so a group's lanes agree bit for bit; whole waves join their rows of 16
// by the two row broadcasts and read the last lane.
template <int LANES> __device__ __forceinline__ float lanes_sum(float v) {
  if constexpr (LANES == 8) {
    v = dpp_add<0xB1>(v);        // quad_perm 1 0 3 2
    v = dpp_add<0x4E>(v);        // quad_perm 2 3 0 1
    return dpp_add<0x141>(v);    // row_half_mirror: the other quad
  }
  v = dpp_add<0x128>(v);         // row_ror:8, 4, 2, 1
  v = dpp_add<0x124>(v);
  v = dpp_add<0x122>(v);
  v = dpp_add<0x121>(v);
  if constexpr (LANES == 32) v += __shfl_xor(v, 16);
  if constexpr (LANES == 64) {
    v = dpp_add<0x142, 0xa>(v);    // row_bcast:15 into rows 1 and 3
    v = dpp_add<0x143, 0xc>(v);    // row_bcast:31 into rows 2 and 3
    v = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
  }
  return v;
}

// ---- dropout of rows (row_dropout.hip has the definition) ----------------------------------------------------------
struct RowDrop {
  uint64_t seed, step;
  const uint64_t* step_dev;   // optional: added to `step` (a replayed graph draws another mask each time)
  uint64_t* step_used;        // optional: the sum, for the backward
  int64_t row_offset;
  uint32_t layer;             // bit 31 set: apart from the stages' counters (philox.h: dropout_patch)
  uint32_t threshold;         // 0: nothing is dropped; 65536: everything
  float scale;
};

struct RowKey { uint32_t k0, k1, c2, c3; };

__device__ __forceinline__ RowKey row_key(const RowDrop& d) {
  const uint64_t step = d.step + (d.step_dev ? *d.step_dev : 0ull);
  if (d.step_used && blockIdx.x == 0 && threadIdx.x == 0) *d.step_used = step;
  return RowKey{(uint32_t)d.seed ^ (uint32_t)(step >> 32), (uint32_t)(d.seed >> 32), d.layer, (uint32_t)step};
}

// Philox4x32-10 with each round's two products as 32 x 32 -> 64 bit multiplies (one v_mad_u64_u32 each where philox.h's
// high and low halves are two quarter-rate multiplies: 16384 x 2048 bf16 dropout 22.6 against 23.6 us)
__device__ __forceinline__ Philox128 philox_row(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, uint32_t k0, uint32_t k1) {
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = (uint64_t)0xD2511F53u * c0, p1 = (uint64_t)0xCD9E8D57u * c2;
    c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0;
    c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
    c1 = (uint32_t)p1;
    c3 = (uint32_t)p0;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return Philox128{{c0, c1, c2, c3}};
}

// the 16-bit draws of the unit at columns 8 unit .. 8 unit + 7 of global row `row`: an element is kept where
// its draw reaches the threshold
__device__ __forceinline__ void draw_unit(const RowKey& k, int64_t row, int64_t unit, uint32_t (&u)[ROW_UNIT]) {
  const Philox128 q = philox_row((uint32_t)row, (uint32_t)unit | ((uint32_t)(row >> 32) << 21), k.c2, k.c3, k.k0, k.k1);
#pragma unroll
  for (int e = 0; e < ROW_UNIT; ++e) u[e] = (e & 1) ? q.w[e >> 1] >> 16 : q.w[e >> 1] & 0xFFFFu;
}

// f = dropout(f) of that unit (a select: what is dropped is zero whatever it held)
__device__ __forceinline__ void drop_unit(const RowKey& k, const RowDrop& d, int64_t row, int64_t unit,
                                          float (&f)[ROW_UNIT]) {
  uint32_t u[ROW_UNIT];
  draw_unit(k, row, unit, u);
#pragma unroll
  for (int e = 0; e < ROW_UNIT; ++e) f[e] = u[e] >= d.threshold ? f[e] * d.scale : 0.f;
}

// f = dropout(f) + r with one rounding
__device__ __forceinline__ void drop_add_unit(const RowKey& k, const RowDrop& d, int64_t row, int64_t unit,
                                              const float (&r)[ROW_UNIT], float (&f)[ROW_UNIT]) {
  if (d.threshold) {
    uint32_t u[ROW_UNIT];
    draw_unit(k, row, unit, u);
#pragma unroll
    for (int e = 0; e < ROW_UNIT; ++e) f[e] = u[e] >= d.threshold ? fmaf(f[e], d.scale, r[e]) : r[e];
  } else {
#pragma unroll
    for (int e = 0; e < ROW_UNIT; ++e) f[e] += r[e];
  }
}

}  // namespace blh
