// Device helpers of the row operators (row_norm.hip, row_dropout.hip): 8-element units of a row, wave and block sums,
// and the draws of the regenerated dropout mask.
//
// Unit: 8 consecutive columns of one row, owned by one lane in every kernel and every type — one 16-byte access for
// bf16 / fp16, two for fp32 — and exactly the elements one Philox call draws for.  A row may start at any multiple of
// the element size (odd widths, rows that are slices of a wider tensor): units are copied with the element's own
// alignment, which gfx950 serves as ordinary 16-byte accesses; only the unit that crosses the end of a row goes element
// by element.
#pragma once
#include "common.h"
#include "philox.h"

namespace blh {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;
static constexpr int ROW_UNIT = 8;

template <typename T> struct alignas(alignof(T)) RawUnit { T v[ROW_UNIT]; };

// f = p[0 .. n) as fp32, zeros behind it (n <= 0: nothing is read)
template <typename T>
__device__ __forceinline__ void load_unit(const T* p, int64_t n, float (&f)[ROW_UNIT]) {
  if (n >= ROW_UNIT) {
    RawUnit<T> r;
    __builtin_memcpy(&r, p, sizeof(r));
#pragma unroll
    for (int e = 0; e < ROW_UNIT; ++e) f[e] = (float)r.v[e];
  } else {
#pragma unroll
    for (int e = 0; e < ROW_UNIT; ++e) f[e] = e < n ? (float)p[e] : 0.f;
  }
}

template <typename T>
__device__ __forceinline__ void store_unit(T* p, int64_t n, const float (&f)[ROW_UNIT]) {
  if (n >= ROW_UNIT) {
    RawUnit<T> r;
#pragma unroll
    for (int e = 0; e < ROW_UNIT; ++e) r.v[e] = (T)f[e];
    __builtin_memcpy(p, &r, sizeof(r));
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

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o);
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
