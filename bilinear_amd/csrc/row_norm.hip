// Layer norm and residual norm over rows, forward and backward.
//
//   h = x                                    (layer norm)
//   h = residual + dropout(x), rounded to the stream's type R   (residual norm; row_dropout.hip defines the mask)
//   mean = sum_j h / W,  rstd = 1 / sqrt(sum_j (h - mean)^2 / W + eps),  hat = (h - mean) rstd,  y = hat g + b
//   backward, t = dy g:  dh' = dh + rstd (t - mean_j t - hat mean_j (t hat)),  dx = dropout(dh'),  dresidual = dh'
//                        dg_j = sum_i dy hat,  db_j = sum_i dy
//
// The variance is taken about the mean in a second pass (no difference of large squares); all sums are fp32, the
// weight gradients' row sums are joined in a fixed order, so results do not change from run to run.
#include "row_ops.h"
#include "row_ops_dev.h"

namespace blh {

struct NormFwd {
  const void *x, *res, *gamma, *beta;
  void *y, *h;
  float *mean, *rstd;
  int64_t ldx, ldr, rows, width;
  float eps;
  bool same;            // weight and bias have the activations' type (else fp32)
  RowDrop drop;
};

struct NormBwd {
  const void *dy, *dh, *h, *gamma;
  const float *mean, *rstd;
  void *dx, *dres, *dgamma, *dbeta;
  float* part;          // [chunks][2][stride]: partial column sums of dy hat and dy
  int64_t lddy, lddh, ldh, rows, width, chunk, stride;
  int chunks;
  bool same;
  RowDrop drop;
};

// sums over the block's 4 waves; `sh` may be reused after the next barrier
__device__ __forceinline__ float block_sum(float v, float* sh) {
  v = lanes_sum<64>(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  return (sh[0] + sh[1]) + (sh[2] + sh[3]);
}

// One block per row, the row read again from cache in each pass: any width.
template <typename T, typename R, bool RESID>
__global__ __launch_bounds__(256) void norm_fwd_kernel(NormFwd p) {
  __shared__ float sh[4];
  const RowKey key = RESID && p.drop.threshold ? row_key(p.drop) : RowKey{};
  const int64_t W = p.width, units = (W + ROW_UNIT - 1) / ROW_UNIT;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(p.x) + row * p.ldx;
    T* y = static_cast<T*>(p.y) + row * W;
    R* h = RESID ? static_cast<R*>(p.h) + row * W : nullptr;
    float sum = 0.f;
    for (int64_t u = threadIdx.x; u < units; u += 256) {
      float f[ROW_UNIT];
      const int64_t c = u * ROW_UNIT;
      load_unit(x + c, W - c, f);
      if (RESID) {
        float r[ROW_UNIT];
        load_unit(static_cast<const R*>(p.res) + row * p.ldr + c, W - c, r);
        drop_add_unit(key, p.drop, p.drop.row_offset + row, u, r, f);
#pragma unroll
        for (int e = 0; e < ROW_UNIT; ++e) f[e] = (float)(R)f[e];      // (what the stream holds is what is normalised)
        store_unit(h + c, W - c, f);
      }
#pragma unroll
      for (int e = 0; e < ROW_UNIT; ++e) sum += f[e];
    }
    const float mean = block_sum(sum, sh) / (float)W;
    float sq = 0.f;
    for (int64_t u = threadIdx.x; u < units; u += 256) {
      float f[ROW_UNIT];
      const int64_t c = u * ROW_UNIT;
      if (RESID) load_unit(h + c, W - c, f); else load_unit(x + c, W - c, f);
#pragma unroll
      for (int e = 0; e < ROW_UNIT; ++e) {
        const float d = c + e < W ? f[e] - mean : 0.f;
        sq = fmaf(d, d, sq);
      }
    }
    const float rstd = 1.f / sqrtf(block_sum(sq, sh) / (float)W + p.eps);
    if (threadIdx.x == 0 && p.mean) { p.mean[row] = mean; p.rstd[row] = rstd; }
    for (int64_t u = threadIdx.x; u < units; u += 256) {
      float f[ROW_UNIT], g[ROW_UNIT], b[ROW_UNIT];
      const int64_t c = u * ROW_UNIT;
      if (RESID) load_unit(h + c, W - c, f); else load_unit(x + c, W - c, f);
      load_param_unit<T>(p.gamma, p.same, c, W - c, 1.f, g);
      load_param_unit<T>(p.beta, p.same, c, W - c, 0.f, b);
#pragma unroll
      for (int e = 0; e < ROW_UNIT; ++e) f[e] = fmaf((f[e] - mean) * rstd, g[e], b[e]);
      store_unit(y + c, W - c, f);
    }
  }
}

// dh' (and dx): one block per row, two passes
template <typename T, typename R, bool RESID>
__global__ __launch_bounds__(256) void norm_bwd_rows_kernel(NormBwd p) {
  __shared__ float sh[4];
  const RowKey key = RESID && p.drop.threshold ? row_key(p.drop) : RowKey{};
  const int64_t W = p.width, units = (W + ROW_UNIT - 1) / ROW_UNIT;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* dy = static_cast<const T*>(p.dy) + row * p.lddy;
    const R* h = static_cast<const R*>(p.h) + row * p.ldh;
    const float mean = p.mean[row], rstd = p.rstd[row];
    float s1 = 0.f, s2 = 0.f;
    for (int64_t u = threadIdx.x; u < units; u += 256) {
      float d[ROW_UNIT], f[ROW_UNIT], g[ROW_UNIT];
      const int64_t c = u * ROW_UNIT;
      load_unit(dy + c, W - c, d);
      load_unit(h + c, W - c, f);
      load_param_unit<T>(p.gamma, p.same, c, W - c, 1.f, g);
#pragma unroll
      for (int e = 0; e < ROW_UNIT; ++e) {
        const float t = d[e] * g[e];          // (zero behind the row's end: dy is)
        s1 += t;
        s2 = fmaf(t, (f[e] - mean) * rstd, s2);
      }
    }
    const float c1 = block_sum(s1, sh) / (float)W;
    const float c2 = block_sum(s2, sh) / (float)W;
    for (int64_t u = threadIdx.x; u < units; u += 256) {
      float d[ROW_UNIT], f[ROW_UNIT], g[ROW_UNIT];
      const int64_t c = u * ROW_UNIT;
      load_unit(dy + c, W - c, d);
      load_unit(h + c, W - c, f);
      load_param_unit<T>(p.gamma, p.same, c, W - c, 1.f, g);
#pragma unroll
      for (int e = 0; e < ROW_UNIT; ++e)
        f[e] = rstd * (d[e] * g[e] - c1 - (f[e] - mean) * rstd * c2);
      if (RESID) {
        if (p.dh) {
          load_unit(static_cast<const R*>(p.dh) + row * p.lddh + c, W - c, g);
#pragma unroll
          for (int e = 0; e < ROW_UNIT; ++e) f[e] += g[e];
        }
        if (p.dres) store_unit(static_cast<R*>(p.dres) + row * W + c, W - c, f);
        if (p.drop.threshold) drop_unit(key, p.drop, p.drop.row_offset + row, u, f);
      }
      if (p.dx) store_unit(static_cast<T*>(p.dx) + row * W + c, W - c, f);
    }
  }
}

// column sums of dy hat and dy over one chunk of rows: a lane owns a unit, the block's 4 waves share the rows
template <typename T, typename R>
__global__ __launch_bounds__(256) void norm_bwd_cols_kernel(NormBwd p) {
  __shared__ float sh[4][2][64 * ROW_UNIT];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t W = p.width, c0 = (int64_t)blockIdx.x * 64 * ROW_UNIT, c = c0 + lane * ROW_UNIT;
  const int64_t r0 = blockIdx.y * p.chunk, r1 = min(p.rows, r0 + p.chunk);
  float ag[ROW_UNIT] = {}, ab[ROW_UNIT] = {};
  for (int64_t row = r0 + wave; row < r1; row += 4) {
    float d[ROW_UNIT], f[ROW_UNIT];
    load_unit(static_cast<const T*>(p.dy) + row * p.lddy + c, W - c, d);
    load_unit(static_cast<const R*>(p.h) + row * p.ldh + c, W - c, f);
    const float mean = p.mean[row], rstd = p.rstd[row];
#pragma unroll
    for (int e = 0; e < ROW_UNIT; ++e) {
      ag[e] = fmaf(d[e], (f[e] - mean) * rstd, ag[e]);
      ab[e] += d[e];
    }
  }
#pragma unroll
  for (int e = 0; e < ROW_UNIT; ++e) { sh[wave][0][lane * ROW_UNIT + e] = ag[e]; sh[wave][1][lane * ROW_UNIT + e] = ab[e]; }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * 64 * ROW_UNIT; i += 256) {
    const int which = i / (64 * ROW_UNIT), j = i % (64 * ROW_UNIT);
    if (c0 + j < W)
      p.part[(blockIdx.y * 2 + which) * p.stride + c0 + j] =
          (sh[0][which][j] + sh[1][which][j]) + (sh[2][which][j] + sh[3][which][j]);
  }
}

// dgamma, dbeta = sums of the chunks' partials, in the parameters' type (chunks == 0: zeros).  A block owns 32 columns:
// 8 lanes x 4 columns, 128 slices of the chunks, so that 512 partial rows are one round trip of four loads.
template <typename T>
__global__ __launch_bounds__(1024) void norm_bwd_finish_kernel(NormBwd p) {
  __shared__ f32x4 sh[128][8];
  const int lane = threadIdx.x & 7, slice = threadIdx.x >> 3;
  const int which = blockIdx.y;
  void* out = which ? p.dbeta : p.dgamma;
  if (!out) return;
  const int64_t c = blockIdx.x * 32ll + lane * 4;
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
  if (c < p.stride) {
#pragma unroll 4
    for (int k = slice; k < p.chunks; k += 128)
      s += *reinterpret_cast<const f32x4*>(p.part + ((int64_t)k * 2 + which) * p.stride + c);
  }
  sh[slice][lane] = s;
#pragma unroll
  for (int half = 64; half >= 1; half >>= 1) {
    __syncthreads();
    if (slice < half) sh[slice][lane] += sh[slice + half][lane];
  }
  if (slice == 0) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (c + e < p.width) {
        const float v = sh[0][lane][e];
        if (p.same) static_cast<T*>(out)[c + e] = (T)v;
        else static_cast<float*>(out)[c + e] = v;
      }
  }
}

// ---- rows that stay in registers --------------------------------------------------------------------------------------
// LANES lanes own a row, NV units each: one read of every input.  Up to 64 lanes a wave needs no barrier; a row of 256
// or 1024 lanes joins its waves' sums through LDS, two buffers in turn (one barrier per sum).

template <int LANES> struct RowGroup {
  static constexpr int WAVES = LANES > 64 ? LANES / 64 : 1;
  int turn = 0;
  // sums of a and b over the row, in every lane; every thread of the block takes part
  __device__ __forceinline__ void sum2(float& a, float& b, float2 (*sh)[16]) {
    constexpr int L = LANES > 64 ? 64 : LANES;
    a = lanes_sum<L>(a);
    b = lanes_sum<L>(b);
    if constexpr (WAVES > 1) {
      const int wave = threadIdx.x >> 6;
      if ((threadIdx.x & 63) == 0) sh[turn][wave] = make_float2(a, b);
      __syncthreads();
      a = b = 0.f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) { const float2 v = sh[turn][w]; a += v.x; b += v.y; }
      turn ^= 1;
    }
  }
  __device__ __forceinline__ float sum(float a, float2 (*sh)[16]) {
    constexpr int L = LANES > 64 ? 64 : LANES;
    a = lanes_sum<L>(a);
    if constexpr (WAVES > 1) {
      const int wave = threadIdx.x >> 6;
      if ((threadIdx.x & 63) == 0) sh[turn][wave].x = a;
      __syncthreads();
      a = 0.f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) a += sh[turn][w].x;
      turn ^= 1;
    }
    return a;
  }
};

template <int LANES> constexpr int fwd_block() { return LANES > 256 ? LANES : 256; }

template <typename T, typename R, bool RESID, int LANES, int NV>
__global__ __launch_bounds__(fwd_block<LANES>()) void norm_fwd_rows_kernel(NormFwd p) {
  constexpr int BLOCK = fwd_block<LANES>(), GROUPS = BLOCK / LANES;
  __shared__ float2 sh[2][16];
  RowGroup<LANES> group;
  const RowKey key = RESID && p.drop.threshold ? row_key(p.drop) : RowKey{};
  const int W = (int)p.width, lane = threadIdx.x % LANES;
  int g = threadIdx.x / LANES;
  if constexpr (LANES == 64) g = __builtin_amdgcn_readfirstlane(g);
  for (int64_t base = (int64_t)blockIdx.x * GROUPS; base < p.rows; base += (int64_t)gridDim.x * GROUPS) {
    const int64_t row = base + g;
    const int width = row < p.rows ? W : 0;        // (a group behind the last row: nothing is read or written)
    const T* x = static_cast<const T*>(p.x) + row * p.ldx;
    float f[NV][ROW_UNIT];
    RawUnit<T> xr[NV];
    RawUnit<R> rr[RESID ? NV : 1];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * LANES + lane) * ROW_UNIT;
      xr[i] = load_raw(x + c, width - c);
      if constexpr (RESID) rr[i] = load_raw(static_cast<const R*>(p.res) + row * p.ldr + c, width - c);
    }
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int u = i * LANES + lane, c = u * ROW_UNIT;
#pragma unroll
      for (int e = 0; e < ROW_UNIT; ++e) f[i][e] = xr[i].get(e);
      if constexpr (RESID) {
        float r[ROW_UNIT];
#pragma unroll
        for (int e = 0; e < ROW_UNIT; ++e) r[e] = rr[i].get(e);
        drop_add_unit(key, p.drop, p.drop.row_offset + row, u, r, f[i]);
#pragma unroll
        for (int e = 0; e < ROW_UNIT; ++e) f[i][e] = (float)(R)f[i][e];      // (what the stream holds is what is normalised)
        store_unit(static_cast<R*>(p.h) + row * p.width + c, width - c, f[i]);
      }
#pragma unroll
      for (int e = 0; e < ROW_UNIT; ++e) sum += f[i][e];
    }
    const float mean = group.sum(sum, sh) / (float)W;
    float sq = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int n = width - (i * LANES + lane) * ROW_UNIT;
#pragma unroll
      for (int e = 0; e < ROW_UNIT; ++e) {
        f[i][e] = e < n ? f[i][e] - mean : 0.f;
        sq = fmaf(f[i][e], f[i][e], sq);
      }
    }
    const float rstd = 1.f / sqrtf(group.sum(sq, sh) / (float)W + p.eps);
    if (lane == 0 && width && p.mean) { p.mean[row] = mean; p.rstd[row] = rstd; }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * LANES + lane) * ROW_UNIT;
      float gm[ROW_UNIT], bt[ROW_UNIT];
      load_param_unit<T>(p.gamma, p.same, c, width - c, 1.f, gm);
      load_param_unit<T>(p.beta, p.same, c, width - c, 0.f, bt);
#pragma unroll
      for (int e = 0; e < ROW_UNIT; ++e) f[i][e] = fmaf(f[i][e] * rstd, gm[e], bt[e]);
      store_unit(static_cast<T*>(p.y) + row * p.width + c, width - c, f[i]);
    }
  }
}

// One block's rows: dh' (and dx), and the block's partial column sums.
template <typename T, typename R, bool RESID, int LANES, int NV, int BLOCK>
__global__ __launch_bounds__(BLOCK) void norm_bwd_kernel(NormBwd p) {
  constexpr int GROUPS = BLOCK / LANES;
  __shared__ float2 sh[2][16];
  extern __shared__ float cols[];          // [2][stride]
  RowGroup<LANES> group;
  const RowKey key = RESID && p.drop.threshold ? row_key(p.drop) : RowKey{};
  const int W = (int)p.width, lane = threadIdx.x % LANES;
  int g = threadIdx.x / LANES;
  if constexpr (LANES == 64) g = __builtin_amdgcn_readfirstlane(g);
  float gm[NV][ROW_UNIT], ag[NV][ROW_UNIT], ab[NV][ROW_UNIT];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * LANES + lane) * ROW_UNIT;
    load_param_unit<T>(p.gamma, p.same, c, W - c, 1.f, gm[i]);
#pragma unroll
    for (int e = 0; e < ROW_UNIT; ++e) ag[i][e] = ab[i][e] = 0.f;
  }
  for (int64_t base = (int64_t)blockIdx.x * GROUPS; base < p.rows; base += (int64_t)gridDim.x * GROUPS) {
    const int64_t row = base + g;
    const bool live = row < p.rows;
    const int width = live ? W : 0;
    const T* dy = static_cast<const T*>(p.dy) + row * p.lddy;
    const R* h = static_cast<const R*>(p.h) + row * p.ldh;
    RawUnit<T> d[NV];
    RawUnit<R> f[NV], dh[RESID ? NV : 1];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * LANES + lane) * ROW_UNIT;
      d[i] = load_raw(dy + c, width - c);
      f[i] = load_raw(h + c, width - c);
    }
    if constexpr (RESID) {
      if (p.dh) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int c = (i * LANES + lane) * ROW_UNIT;
          dh[i] = load_raw(static_cast<const R*>(p.dh) + row * p.lddh + c, width - c);
        }
      }
    }
    const float mean = live ? p.mean[row] : 0.f, rstd = live ? p.rstd[row] : 0.f;
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int e = 0; e < ROW_UNIT; ++e) {
        const float v = d[i].get(e), hat = (f[i].get(e) - mean) * rstd, t = v * gm[i][e];     // (v = 0 behind the row's end)
        s1 += t;
        s2 = fmaf(t, hat, s2);
        ag[i][e] = fmaf(v, hat, ag[i][e]);
        ab[i][e] += v;
      }
    }
    group.sum2(s1, s2, sh);
    const float c1 = s1 / (float)W, c2 = s2 / (float)W;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int u = i * LANES + lane, c = u * ROW_UNIT;
      float o[ROW_UNIT];
#pragma unroll
      for (int e = 0; e < ROW_UNIT; ++e) {
        const float hat = (f[i].get(e) - mean) * rstd;
        o[e] = rstd * (fmaf(d[i].get(e), gm[i][e], -c1) - hat * c2);
      }
      if constexpr (RESID) {
        if (p.dh) {
#pragma unroll
          for (int e = 0; e < ROW_UNIT; ++e) o[e] += dh[i].get(e);
        }
        if (p.dres) store_unit(static_cast<R*>(p.dres) + row * p.width + c, width - c, o);
        if (p.dx && p.drop.threshold) drop_unit(key, p.drop, p.drop.row_offset + row, u, o);
      }
      if (p.dx) store_unit(static_cast<T*>(p.dx) + row * p.width + c, width - c, o);
    }
  }
  if (!p.part) return;
  // the block's groups add their columns up one after the other
#pragma unroll 1
  for (int k = 0; k < GROUPS; ++k) {
    if (k == threadIdx.x / LANES) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (i * LANES + lane) * ROW_UNIT;
        if (c < W) {
#pragma unroll
          for (int e = 0; e < ROW_UNIT; ++e) {
            cols[c + e] = k ? cols[c + e] + ag[i][e] : ag[i][e];
            cols[p.stride + c + e] = k ? cols[p.stride + c + e] + ab[i][e] : ab[i][e];
          }
        }
      }
    }
    __syncthreads();
  }
  float* out = p.part + (int64_t)blockIdx.x * 2 * p.stride;
  for (int j = threadIdx.x * 4; j < 2 * p.stride; j += BLOCK * 4)
    *reinterpret_cast<f32x4*>(out + j) = *reinterpret_cast<const f32x4*>(cols + j);
}

// rows of one partial sum of the wide form: whole groups of 16 rows, at most 256 chunks
static int64_t norm_chunk(int64_t rows) { return round_up(std::max<int64_t>(1, ceil_div(rows, 256)), 16); }
static int64_t norm_stride(int64_t width) { return round_up(width, ROW_UNIT); }
static constexpr int64_t ROW_RESIDENT = 8192;      // widest row that stays in registers
#ifndef ROW_BWD_BLOCKS
#define ROW_BWD_BLOCKS 512
#endif
#ifndef ROW_FWD_BLOCKS
#define ROW_FWD_BLOCKS 2048
#endif
static constexpr int BWD_BLOCKS = ROW_BWD_BLOCKS;      // partial rows the backward leaves at most
static int norm_partials(int64_t rows, int64_t width) {
  return width <= ROW_RESIDENT ? (int)std::min<int64_t>(rows, BWD_BLOCKS) : (int)ceil_div(rows, norm_chunk(rows));
}

template <typename T, typename R, bool RESID, int LANES, int NV>
static int launch_fwd_rows(hipStream_t s, const NormFwd& p) {
  constexpr int BLOCK = fwd_block<LANES>();
  const unsigned blocks = (unsigned)std::min<int64_t>(ceil_div(p.rows, BLOCK / LANES), ROW_FWD_BLOCKS);
  hipLaunchKernelGGL((norm_fwd_rows_kernel<T, R, RESID, LANES, NV>), dim3(blocks), dim3(BLOCK), 0, s, p);
  BLH_HIP_TRY(hipGetLastError());
  return BLH_OK;
}

template <typename T, typename R, bool RESID>
static int launch_norm_fwd(hipStream_t s, const NormFwd& p) {
  if (p.width <= 128) return launch_fwd_rows<T, R, RESID, 16, 1>(s, p);
  if (p.width <= 256) return launch_fwd_rows<T, R, RESID, 32, 1>(s, p);
  if (p.width <= 512) return launch_fwd_rows<T, R, RESID, 64, 1>(s, p);
  if (p.width <= 1024) return launch_fwd_rows<T, R, RESID, 64, 2>(s, p);
  if (p.width <= 2048) return launch_fwd_rows<T, R, RESID, 64, 4>(s, p);
  if (p.width <= 4096) return launch_fwd_rows<T, R, RESID, 256, 2>(s, p);
  if (p.width <= ROW_RESIDENT) return launch_fwd_rows<T, R, RESID, 256, 4>(s, p);
  const unsigned blocks = (unsigned)std::min<int64_t>(p.rows, 1 << 16);
  hipLaunchKernelGGL((norm_fwd_kernel<T, R, RESID>), dim3(blocks), dim3(256), 0, s, p);
  BLH_HIP_TRY(hipGetLastError());
  return BLH_OK;
}

template <typename T, typename R, bool RESID, int LANES, int NV, int BLOCK>
static int launch_bwd_rows(hipStream_t s, NormBwd& p) {
  const unsigned blocks = (unsigned)std::min<int64_t>(ceil_div(p.rows, BLOCK / LANES), BWD_BLOCKS);
  p.chunks = (int)blocks;
  const size_t lds = p.part ? 2 * p.stride * sizeof(float) : 0;
  auto kern = norm_bwd_kernel<T, R, RESID, LANES, NV, BLOCK>;
  if (lds > 65536 - 1024) BLH_HIP_TRY(hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
  hipLaunchKernelGGL(kern, dim3(blocks), dim3(BLOCK), lds, s, p);
  BLH_HIP_TRY(hipGetLastError());
  return BLH_OK;
}

template <typename T, typename R, bool RESID>
static int launch_norm_bwd(hipStream_t s, NormBwd p) {
  const bool grads = p.dgamma || p.dbeta;
  p.stride = norm_stride(p.width);
  if (!grads) p.part = nullptr;
  if (p.rows > 0 && p.width <= ROW_RESIDENT) {
    if (p.width <= 128) BLH_TRY((launch_bwd_rows<T, R, RESID, 16, 1, 256>(s, p)));
    else if (p.width <= 256) BLH_TRY((launch_bwd_rows<T, R, RESID, 32, 1, 256>(s, p)));
    else if (p.width <= 512) BLH_TRY((launch_bwd_rows<T, R, RESID, 64, 1, 512>(s, p)));
    else if (p.width <= 1024) BLH_TRY((launch_bwd_rows<T, R, RESID, 64, 2, 512>(s, p)));
    else if (p.width <= 2048) BLH_TRY((launch_bwd_rows<T, R, RESID, 64, 4, 512>(s, p)));
    else if (p.width <= 4096) BLH_TRY((launch_bwd_rows<T, R, RESID, 256, 2, 256>(s, p)));
    else BLH_TRY((launch_bwd_rows<T, R, RESID, 256, 4, 256>(s, p)));
  } else if (p.rows > 0) {
    if (p.dx || p.dres) {
      const unsigned blocks = (unsigned)std::min<int64_t>(p.rows, 1 << 16);
      hipLaunchKernelGGL((norm_bwd_rows_kernel<T, R, RESID>), dim3(blocks), dim3(256), 0, s, p);
      BLH_HIP_TRY(hipGetLastError());
    }
    if (grads) {
      p.chunk = norm_chunk(p.rows);
      p.chunks = norm_partials(p.rows, p.width);
      const dim3 grid((unsigned)ceil_div(p.width, 64 * ROW_UNIT), (unsigned)p.chunks);
      hipLaunchKernelGGL((norm_bwd_cols_kernel<T, R>), grid, dim3(256), 0, s, p);
      BLH_HIP_TRY(hipGetLastError());
    }
  }
  if (grads) {
    hipLaunchKernelGGL((norm_bwd_finish_kernel<T>), dim3((unsigned)ceil_div(p.stride, 32), 2), dim3(1024), 0, s, p);
    BLH_HIP_TRY(hipGetLastError());
  }
  return BLH_OK;
}

// the type combinations: activations T, residual stream R = T or fp32
#define BLH_NORM_DISPATCH(dtype, rtype, resid, fn, ...)                                        \
  switch (dtype) {                                                                             \
    case BLH_F32: return fn<float, float, resid>(__VA_ARGS__);                                 \
    case BLH_BF16:                                                                             \
      if (rtype == BLH_F32) return fn<bf16_t, float, resid>(__VA_ARGS__);                      \
      return fn<bf16_t, bf16_t, resid>(__VA_ARGS__);                                           \
    default:                                                                                   \
      if (rtype == BLH_F32) return fn<f16_t, float, resid>(__VA_ARGS__);                       \
      return fn<f16_t, f16_t, resid>(__VA_ARGS__);                                             \
  }

static int norm_fwd(hipStream_t s, const NormFwd& p, int32_t dtype) {
  switch (dtype) {
    case BLH_F32: return launch_norm_fwd<float, float, false>(s, p);
    case BLH_BF16: return launch_norm_fwd<bf16_t, bf16_t, false>(s, p);
    default: return launch_norm_fwd<f16_t, f16_t, false>(s, p);
  }
}
static int norm_bwd(hipStream_t s, const NormBwd& p, int32_t dtype) {
  switch (dtype) {
    case BLH_F32: return launch_norm_bwd<float, float, false>(s, p);
    case BLH_BF16: return launch_norm_bwd<bf16_t, bf16_t, false>(s, p);
    default: return launch_norm_bwd<f16_t, f16_t, false>(s, p);
  }
}
static int resid_fwd(hipStream_t s, const NormFwd& p, int32_t dtype, int32_t rtype) {
  BLH_NORM_DISPATCH(dtype, rtype, true, launch_norm_fwd, s, p)
}
static int resid_bwd(hipStream_t s, const NormBwd& p, int32_t dtype, int32_t rtype) {
  BLH_NORM_DISPATCH(dtype, rtype, true, launch_norm_bwd, s, p)
}

static int check_types(int32_t dtype, int32_t rtype, int32_t param_dtype) {
  if (!row_dtype_ok(dtype) || !row_dtype_ok(rtype) || !row_dtype_ok(param_dtype)) return BLH_ERR_INVALID_ARGUMENT;
  if (rtype != dtype && rtype != BLH_F32) return BLH_ERR_INVALID_ARGUMENT;
  if (param_dtype != dtype && param_dtype != BLH_F32) return BLH_ERR_INVALID_ARGUMENT;
  return BLH_OK;
}

static const RowDrop NO_DROP = {0, 0, nullptr, nullptr, 0, 0, 0, 1.f};

}  // namespace blh

using namespace blh;

extern "C" {

int blh_layer_norm_forward(void* stream, const void* x, int64_t ldx, const void* weight, const void* bias, double eps,
                           void* y, float* mean, float* rstd, int64_t rows, int64_t width, int32_t dtype,
                           int32_t param_dtype) {
  BLH_TRY(check_types(dtype, dtype, param_dtype));
  if (!(eps >= 0.0) || ldx < 0 || !mean != !rstd) return BLH_ERR_INVALID_ARGUMENT;
  BLH_TRY(row_check_shape(rows, width));
  if (rows == 0) return BLH_OK;
  if (!x || !y || !row_aligned(x, dtype) || !row_aligned(y, dtype) || !row_aligned(weight, param_dtype) ||
      !row_aligned(bias, param_dtype))
    return BLH_ERR_INVALID_ARGUMENT;
  const NormFwd p{x, nullptr, weight, bias, y, nullptr, mean, rstd, ldx, 0, rows, width, (float)eps,
                  param_dtype == dtype, NO_DROP};
  return norm_fwd((hipStream_t)stream, p, dtype);
}

int blh_residual_norm_forward(void* stream, const void* x, int64_t ldx, const void* residual, int64_t ldr,
                              const void* weight, const void* bias, double eps, const blh_row_drop* drop, void* y,
                              void* h, float* mean, float* rstd, int64_t rows, int64_t width, int32_t dtype,
                              int32_t stream_dtype, int32_t param_dtype) {
  BLH_TRY(check_types(dtype, stream_dtype, param_dtype));
  if (!(eps >= 0.0) || ldx < 0 || ldr < 0 || !mean != !rstd) return BLH_ERR_INVALID_ARGUMENT;
  BLH_TRY(row_check_shape(rows, width));
  RowDrop d = NO_DROP;
  if (drop) BLH_TRY(row_make_drop(drop, rows, &d));
  if (rows == 0) return BLH_OK;
  if (!x || !residual || !y || !h || !row_aligned(x, dtype) || !row_aligned(y, dtype) ||
      !row_aligned(residual, stream_dtype) || !row_aligned(h, stream_dtype) || !row_aligned(weight, param_dtype) ||
      !row_aligned(bias, param_dtype))
    return BLH_ERR_INVALID_ARGUMENT;
  const NormFwd p{x, residual, weight, bias, y, h, mean, rstd, ldx, ldr, rows, width, (float)eps,
                  param_dtype == dtype, d};
  return resid_fwd((hipStream_t)stream, p, dtype, stream_dtype);
}

int64_t blh_row_norm_workspace_bytes(int64_t rows, int64_t width) {
  BLH_TRY(row_check_shape(rows, width));
  return std::max<int64_t>(256, (int64_t)norm_partials(rows, width) * 2 * norm_stride(width) * (int64_t)sizeof(float));
}

int blh_layer_norm_backward(void* stream, const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* weight,
                            const float* mean, const float* rstd, void* dx, void* dweight, void* dbias,
                            void* workspace, int64_t workspace_bytes, int64_t rows, int64_t width, int32_t dtype,
                            int32_t param_dtype) {
  BLH_TRY(check_types(dtype, dtype, param_dtype));
  if (lddy < 0 || ldx < 0) return BLH_ERR_INVALID_ARGUMENT;
  BLH_TRY(row_check_shape(rows, width));
  if (rows > 0 && (!dy || !x || !mean || !rstd)) return BLH_ERR_INVALID_ARGUMENT;
  if (!row_aligned(dy, dtype) || !row_aligned(x, dtype) || !row_aligned(dx, dtype) || !row_aligned(weight, param_dtype) ||
      !row_aligned(dweight, param_dtype) || !row_aligned(dbias, param_dtype))
    return BLH_ERR_INVALID_ARGUMENT;
  if (dweight || dbias) {
    if (!workspace || (uintptr_t)workspace % 16 != 0) return BLH_ERR_INVALID_ARGUMENT;
    if (workspace_bytes < blh_row_norm_workspace_bytes(rows, width)) return BLH_ERR_WORKSPACE;
  }
  const NormBwd p{dy, nullptr, x, weight, mean, rstd, dx, nullptr, dweight, dbias, static_cast<float*>(workspace),
                  lddy, 0, ldx, rows, width, 0, 0, 0, param_dtype == dtype, NO_DROP};
  return norm_bwd((hipStream_t)stream, p, dtype);
}

int blh_residual_norm_backward(void* stream, const void* dy, int64_t lddy, const void* dh, int64_t lddh, const void* h,
                               int64_t ldh, const void* weight, const float* mean, const float* rstd,
                               const blh_row_drop* drop, void* dx, void* dresidual, void* dweight, void* dbias,
                               void* workspace, int64_t workspace_bytes, int64_t rows, int64_t width, int32_t dtype,
                               int32_t stream_dtype, int32_t param_dtype) {
  BLH_TRY(check_types(dtype, stream_dtype, param_dtype));
  if (lddy < 0 || lddh < 0 || ldh < 0) return BLH_ERR_INVALID_ARGUMENT;
  BLH_TRY(row_check_shape(rows, width));
  RowDrop d = NO_DROP;
  if (drop) BLH_TRY(row_make_drop(drop, rows, &d));
  d.step_used = nullptr;
  if (rows > 0 && (!dy || !h || !mean || !rstd)) return BLH_ERR_INVALID_ARGUMENT;
  if (!row_aligned(dy, dtype) || !row_aligned(dx, dtype) || !row_aligned(dh, stream_dtype) ||
      !row_aligned(h, stream_dtype) || !row_aligned(dresidual, stream_dtype) || !row_aligned(weight, param_dtype) ||
      !row_aligned(dweight, param_dtype) || !row_aligned(dbias, param_dtype))
    return BLH_ERR_INVALID_ARGUMENT;
  if (dweight || dbias) {
    if (!workspace || (uintptr_t)workspace % 16 != 0) return BLH_ERR_INVALID_ARGUMENT;
    if (workspace_bytes < blh_row_norm_workspace_bytes(rows, width)) return BLH_ERR_WORKSPACE;
  }
  const NormBwd p{dy, dh, h, weight, mean, rstd, dx, dresidual, dweight, dbias, static_cast<float*>(workspace),
                  lddy, lddh, ldh, rows, width, 0, 0, 0, param_dtype == dtype, d};
  return resid_bwd((hipStream_t)stream, p, dtype, stream_dtype);
}

}  // extern "C"
