// Device helpers of the row operators (row_norm.hip, row_dropout.hip): 8-element units of a row, wave and block sums,
// and the draws of the regenerated dropout mask.
//
// Unit: 8 consecutive columns of one row, owned by one lane in every kernel and every type — one 16-byte access for
// bf16 / fp16, two for fp32 — and exactly the elements one Philox call draws for.  A row may start at any multiple of
// the element size (odd widths, rows that are slices of a wider tensor): units are copied with the element's own
// alignment, which gfx950 serves as ordinary 16-byte accesses; only the unit that crosses the end of a row goes element
// by element.
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
  __device__ __forceinline__ float get(int e) const { return q[e >> 2][e & 3]; }
  __device__ __forceinline__ void set(const float (&f)[ROW_UNIT]) {
#pragma unroll
    for (int e = 0; e < ROW_UNIT; ++e) q[e >> 2][e & 3] = f[e];
  }
};

// the unit p[0 .. n), zeros behind it (n <= 0: nothing is read)
template <typename T> __device__ __forceinline__ RawUnit<T> load_raw(const T* p, int64_t n) {
  RawUnit<T> r;
  if (n >= ROW_UNIT) {
    r.load(p);
  } else {
    float f[ROW_UNIT];
#pragma unroll
    for (int e = 0; e < ROW_UNIT; ++e) f[e] = e < n ? (float)p[e] : 0.f;
    r.set(f);
  }
  return r;
}

template <typename T>
__device__ __forceinline__ void load_unit(const T* p, int64_t n, float (&f)[ROW_UNIT]) {
  const RawUnit<T> r = load_raw(p, n);
#pragma unroll
  for (int e = 0; e < ROW_UNIT; ++e) f[e] = r.get(e);
}

template <typename T>
__device__ __forceinline__ void store_unit(T* p, int64_t n, const float (&f)[ROW_UNIT]) {
  RawUnit<T> r;
  r.set(f);
  if (n >= ROW_UNIT) {
    r.store(p);
  } else {
#pragma unroll
    for (int e = 0; e < ROW_UNIT; ++e)
      if (e < n) p[e] = (T)f[e];
  }
}

// weight / bias: fp32 or the activations' type (`same`), or absent (nullptr: `absent` everywhere)
template <typename T>
__device__ __forceinline__ void load_param_unit(const void* p, bool same, int64_t col, int64_t n, float absent,
                                                float (&f)[ROW_UNIT]) {
  if (!p) {
#pragma unroll
    for (int e = 0; e < ROW_UNIT; ++e) f[e] = absent;
  } else if (same) {
    load_unit(static_cast<const T*>(p) + col, n, f);
  } else {
    load_unit(static_cast<const float*>(p) + col, n, f);
  }
}

template <int CTRL, int ROWS = 0xf> __device__ __forceinline__ float dpp_add(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, ROWS, 0xf, false));
}

// sum over groups of LANES consecutive lanes (16, 32 or 64), in every lane; all 64 lanes take part.  Rotations inside
// rows of 16 lanes pair equal partial sums, so a group's lanes agree bit for bit; whole waves join their rows by the two
// row broadcasts and read the last lane.
template <int LANES> __device__ __forceinline__ float lanes_sum(float v) {
  v = dpp_add<0x128>(v);       // row_ror:8, 4, 2, 1
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

// the 16-bit draws of the unit at columns 8 unit .. 8 unit + 7 of global row `row`: an element is kept where
// its draw reaches the threshold
__device__ __forceinline__ void draw_unit(const RowKey& k, int64_t row, int64_t unit, uint32_t (&u)[ROW_UNIT]) {
  const Philox128 q = philox4x32_10((uint32_t)row, (uint32_t)unit | ((uint32_t)(row >> 32) << 21), k.c2, k.c3, k.k0, k.k1);
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
