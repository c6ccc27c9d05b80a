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
  int row_blocks;       // few rows: blocks of the launch that take rows, those behind them take columns
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

// ---- rows that are read again in each pass: any width ---------------------------------------------------------------------
// (over 16384 columns; 512 x 32768 bf16: layer norm forward 24 us = 2.8 TB/s of its bytes, backward 51 us = 2.0)

template <typename T, typename R, bool RESID>
__global__ __launch_bounds__(256) void norm_fwd_kernel(NormFwd p) {
  __shared__ float sh[4];
  const RowKey key = RESID && p.drop.threshold ? row_key(p.drop) : RowKey{};
  const int W = (int)p.width, units = (W + ROW_UNIT - 1) / ROW_UNIT;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(p.x) + row * p.ldx;
    T* y = static_cast<T*>(p.y) + row * p.width;
    R* h = RESID ? static_cast<R*>(p.h) + row * p.width : nullptr;
    float sum = 0.f;
    for (int u = threadIdx.x; u < units; u += 256) {
      float f[ROW_UNIT];
      const int c = u * ROW_UNIT;
      load_unit<false>(x, c, W, f);
      if (RESID) {
        float r[ROW_UNIT];
        load_unit<false>(static_cast<const R*>(p.res) + row * p.ldr, c, W, r);
        drop_add_unit(key, p.drop, p.drop.row_offset + row, u, r, f);
#pragma unroll
        for (int e = 0; e < ROW_UNIT; ++e) f[e] = (float)(R)f[e];      // (what the stream holds is what is normalised)
        store_unit(h, c, W, f);
      }
#pragma unroll
      for (int e = 0; e < ROW_UNIT; ++e) sum += f[e];
    }
    const float mean = block_sum(sum, sh) / (float)W;
    float sq = 0.f;
    for (int u = threadIdx.x; u < units; u += 256) {
      float f[ROW_UNIT];
      const int c = u * ROW_UNIT;
      if (RESID) load_unit<false>(h, c, W, f); else load_unit<false>(x, c, W, f);
#pragma unroll
      for (int e = 0; e < ROW_UNIT; ++e) {
        const float d = c + e < W ? f[e] - mean : 0.f;
        sq = fmaf(d, d, sq);
      }
    }
    const float rstd = 1.f / sqrtf(block_sum(sq, sh) / (float)W + p.eps);
    if (threadIdx.x == 0 && p.mean) { p.mean[row] = mean; p.rstd[row] = rstd; }
    for (int u = threadIdx.x; u < units; u += 256) {
      float f[ROW_UNIT], g[ROW_UNIT], b[ROW_UNIT];
      const int c = u * ROW_UNIT;
      if (RESID) load_unit<false>(h, c, W, f); else load_unit<false>(x, c, W, f);
      load_param_unit<false, T>(p.gamma, p.same, c, W, 1.f, g);
      load_param_unit<false, T>(p.beta, p.same, c, W, 0.f, b);
#pragma unroll
      for (int e = 0; e < ROW_UNIT; ++e) f[e] = fmaf((f[e] - mean) * rstd, g[e], b[e]);
      store_unit(y, c, W, f);
    }
  }
}

// dh' (and dx): one block per row, two passes
template <typename T, typename R, bool RESID>
__global__ __launch_bounds__(256) void norm_bwd_rows_kernel(NormBwd p) {
  __shared__ float sh[4];
  const RowKey key = RESID && p.drop.threshold ? row_key(p.drop) : RowKey{};
  const int W = (int)p.width, units = (W + ROW_UNIT - 1) / ROW_UNIT;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* dy = static_cast<const T*>(p.dy) + row * p.lddy;
    const R* h = static_cast<const R*>(p.h) + row * p.ldh;
    const float mean = p.mean[row], rstd = p.rstd[row];
    float s1 = 0.f, s2 = 0.f;
    for (int u = threadIdx.x; u < units; u += 256) {
      float g[ROW_UNIT];
      const int c = u * ROW_UNIT;
      RawUnit<T> d = load_raw<false>(dy, c, W);
      RawUnit<R> f = load_raw<false>(h, c, W);
      settle2(d, f, c, W);
      load_param_unit<false, T>(p.gamma, p.same, c, W, 1.f, g);
#pragma unroll
      for (int e = 0; e < ROW_UNIT; ++e) {
        const float t = d.get(e) * g[e];          // (zero behind the row's end: dy is)
        s1 += t;
        s2 = fmaf(t, (f.get(e) - mean) * rstd, s2);
      }
    }
    const float c1 = block_sum(s1, sh) / (float)W;
    const float c2 = block_sum(s2, sh) / (float)W;
    for (int u = threadIdx.x; u < units; u += 256) {
      float d[ROW_UNIT], f[ROW_UNIT], g[ROW_UNIT];
      const int c = u * ROW_UNIT;
      load_unit<false>(dy, c, W, d);
      load_unit<false>(h, c, W, f);
      load_param_unit<false, T>(p.gamma, p.same, c, W, 1.f, g);
#pragma unroll
      for (int e = 0; e < ROW_UNIT; ++e)
        f[e] = rstd * (d[e] * g[e] - c1 - (f[e] - mean) * rstd * c2);
      if (RESID) {
        if (p.dh) {
          load_unit<false>(static_cast<const R*>(p.dh) + row * p.lddh, c, W, g);
#pragma unroll
          for (int e = 0; e < ROW_UNIT; ++e) f[e] += g[e];
        }
        if (p.dres) store_unit(static_cast<R*>(p.dres) + row * p.width, c, W, f);
        if (p.drop.threshold) drop_unit(key, p.drop, p.drop.row_offset + row, u, f);
      }
      if (p.dx) store_unit(static_cast<T*>(p.dx) + row * p.width, c, W, f);
    }
  }
}

// column sums of dy hat and dy over one chunk of rows: a lane owns a unit, the block's 4 waves share the rows
template <typename T, typename R>
__global__ __launch_bounds__(256) void norm_bwd_cols_kernel(NormBwd p) {
  __shared__ float sh[4][2][64 * ROW_UNIT];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int W = (int)p.width, c0 = blockIdx.x * 64 * ROW_UNIT, c = c0 + lane * ROW_UNIT;
  const int64_t r0 = blockIdx.y * p.chunk, r1 = min(p.rows, r0 + p.chunk);
  float ag[ROW_UNIT] = {}, ab[ROW_UNIT] = {};
  for (int64_t row = r0 + wave; row < r1; row += 4) {
    float d[ROW_UNIT], f[ROW_UNIT];
    load_unit<false>(static_cast<const T*>(p.dy) + row * p.lddy, c, W, d);
    load_unit<false>(static_cast<const R*>(p.h) + row * p.ldh, c, W, f);
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
// 8 lanes x 4 columns, 128 slices of the chunks, so that 512 partial rows are one round trip of four loads (4 us for 512 rows
// of 1024 or 256 of 2048 columns: a launch and that round trip).
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
// LANES lanes own a row, NV units each: one read of every input, one write of every output, so what bounds these kernels is
// memory (16384 x 2048 bf16, one operation over and over on three inputs in turn: layer norm forward 22.9 us, backward with its
// finish 39 us, on an fp32 stream residual norm 76 and 104 us; a copy of as many bytes in the same loop 19.5, 35, 74 and 100).
// One kernel does not fit: the residual norm's backward of 8193 to 16384 columns on an fp32 stream spills 10 to 14 registers
// a lane (1024 x 16384 fp32 96 us = 3.5 TB/s of its bytes).  Up to 64 lanes a row needs no barrier; a longer one joins its waves' sums through LDS, two
// buffers in turn (one barrier per sum).

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
      for (int w = 0; w < WAVES; ++w) { const float2 v = sh[turn][(wave & ~(WAVES - 1)) + w]; a += v.x; b += v.y; }
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
      for (int w = 0; w < WAVES; ++w) a += sh[turn][(wave & ~(WAVES - 1)) + w].x;
      turn ^= 1;
    }
    return a;
  }
};

template <typename T, typename R, bool RESID, int LANES, int NV, int BLOCK, bool SHORT>
__global__ __launch_bounds__(BLOCK) void norm_fwd_rows_kernel(NormFwd p) {
  constexpr int GROUPS = BLOCK / LANES;
  __shared__ float2 sh[2][16];
  RowGroup<LANES> group;
  const RowKey key = RESID && p.drop.threshold ? row_key(p.drop) : RowKey{};
  const int W = (int)p.width, lane = threadIdx.x % LANES;
  int g = threadIdx.x / LANES;
  if constexpr (LANES == 64) g = __builtin_amdgcn_readfirstlane(g);
  // the parameters first: in the epilogue each would be a round trip of its own, behind the sums
  float gm[NV][ROW_UNIT], bt[NV][ROW_UNIT];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * LANES + lane) * ROW_UNIT;
    load_param_unit<SHORT, T>(p.gamma, p.same, c, W, 1.f, gm[i]);
    load_param_unit<SHORT, T>(p.beta, p.same, c, W, 0.f, bt[i]);
  }
  struct In { RawUnit<T> x[NV]; RawUnit<R> r[RESID ? NV : 1]; };
  auto load = [&](int64_t row, In& q) {
    row = min(row, p.rows - 1);                    // (a group behind the last row reads that one and writes nothing)
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * LANES + lane) * ROW_UNIT;
      q.x[i] = load_raw<SHORT>(static_cast<const T*>(p.x) + row * p.ldx, c, W);
      if constexpr (RESID) q.r[i] = load_raw<SHORT>(static_cast<const R*>(p.res) + row * p.ldr, c, W);
    }
  };
  for (int64_t base = (int64_t)blockIdx.x * GROUPS; base < p.rows; base += (int64_t)gridDim.x * GROUPS) {
    const int64_t row = base + g;
    const int width = row < p.rows ? W : 0;
    In in;
    load(row, in);
    float f[NV][ROW_UNIT];
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int u = i * LANES + lane, c = u * ROW_UNIT;
      settle(in.x[i], c, width);
#pragma unroll
      for (int e = 0; e < ROW_UNIT; ++e) f[i][e] = in.x[i].get(e);
      if constexpr (RESID) {
        float r[ROW_UNIT];
        settle(in.r[i], c, width);
#pragma unroll
        for (int e = 0; e < ROW_UNIT; ++e) r[e] = in.r[i].get(e);
        drop_add_unit(key, p.drop, p.drop.row_offset + row, u, r, f[i]);
#pragma unroll
        for (int e = 0; e < ROW_UNIT; ++e) f[i][e] = (float)(R)f[i][e];      // (what the stream holds is what is normalised)
        store_unit(static_cast<R*>(p.h) + row * p.width, c, width, f[i]);
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
#pragma unroll
      for (int e = 0; e < ROW_UNIT; ++e) f[i][e] = fmaf(f[i][e] * rstd, gm[i][e], bt[i][e]);
      store_unit(static_cast<T*>(p.y) + row * p.width, c, width, f[i]);
    }
  }
}

// Few rows: dg and db of 64 columns by one block of 512 threads that reads all rows itself (8 lanes of a unit, 64 slices of
// the rows), so that the backward is one launch without partial sums.
template <typename T, typename R, bool SHORT>
__device__ __forceinline__ void norm_few_cols(const NormBwd& p, int block) {
  __shared__ float sh[8][8][2 * ROW_UNIT];
  const int lane = threadIdx.x & 7, wave = threadIdx.x >> 6, W = (int)p.width, c0 = block * 64, c = c0 + lane * ROW_UNIT;
  float a[2 * ROW_UNIT] = {};
  for (int row = threadIdx.x >> 3; row < (int)p.rows; row += 64) {
    RawUnit<T> d = load_raw<SHORT>(static_cast<const T*>(p.dy) + row * p.lddy, c, W);
    RawUnit<R> h = load_raw<SHORT>(static_cast<const R*>(p.h) + row * p.ldh, c, W);
    const float mean = p.mean[row], rstd = p.rstd[row];
    settle(d, c, W);
    settle(h, c, W);
#pragma unroll
    for (int e = 0; e < ROW_UNIT; ++e) {
      a[e] = fmaf(d.get(e), (h.get(e) - mean) * rstd, a[e]);
      a[ROW_UNIT + e] += d.get(e);
    }
  }
#pragma unroll
  for (int e = 0; e < 2 * ROW_UNIT; ++e) {
#pragma unroll
    for (int o = 8; o < 64; o <<= 1) a[e] += __shfl_xor(a[e], o);
    if ((threadIdx.x & 63) < 8) sh[wave][lane][e] = a[e];
  }
  __syncthreads();
  const int which = threadIdx.x >> 6, j = threadIdx.x & 63;
  void* out = which ? p.dbeta : p.dgamma;
  if (which < 2 && out && c0 + j < W) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) v += sh[w][j / ROW_UNIT][which * ROW_UNIT + j % ROW_UNIT];
    if (p.same) static_cast<T*>(out)[c0 + j] = (T)v;
    else static_cast<float*>(out)[c0 + j] = v;
  }
}

// partial rows a block of the backward holds in LDS: one for each wave (groups inside a wave join by shuffles) or for each
// group of waves, but the first, which stays in registers
template <int LANES, int BLOCK> constexpr int bwd_shares() { return LANES < 64 ? BLOCK / 64 : BLOCK / LANES; }

// One block's rows, NV units a lane (one; two in rows of over 8192 columns: 1024 x 16384 bf16 33 us, read again in each pass
// 48): dh' (and dx), and the block's partial column sums in its row of p.part.
template <typename T, typename R, bool RESID, int LANES, int NV, int BLOCK, bool SHORT, bool FEW>
__global__ __launch_bounds__(BLOCK) void norm_bwd_kernel(NormBwd p) {
  constexpr int GROUPS = BLOCK / LANES, SHARES = bwd_shares<LANES, BLOCK>();
  if constexpr (FEW) {
    if ((int)blockIdx.x >= p.row_blocks) {
      norm_few_cols<T, R, SHORT>(p, blockIdx.x - p.row_blocks);
      return;
    }
  }
  __shared__ float2 sh[2][16];
  extern __shared__ f32x4 cols4[];         // [SHARES - 1][2][stride]
  RowGroup<LANES> group;
  const RowKey key = RESID && p.drop.threshold ? row_key(p.drop) : RowKey{};
  const int W = (int)p.width, lane = threadIdx.x % LANES;
  int g = threadIdx.x / LANES;
  if constexpr (LANES == 64) g = __builtin_amdgcn_readfirstlane(g);
  float gm[NV][ROW_UNIT], ag[NV][ROW_UNIT], ab[NV][ROW_UNIT];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    load_param_unit<SHORT, T>(p.gamma, p.same, (i * LANES + lane) * ROW_UNIT, W, 1.f, gm[i]);
#pragma unroll
    for (int e = 0; e < ROW_UNIT; ++e) ag[i][e] = ab[i][e] = 0.f;
  }
  struct In { RawUnit<T> d[NV]; RawUnit<R> f[NV], dh[NV]; float mean, rstd; };
  auto load = [&](int64_t row, In& q) {
    row = min(row, p.rows - 1);                    // (a group behind the last row reads that one and writes nothing)
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * LANES + lane) * ROW_UNIT;
      q.d[i] = load_raw<SHORT>(static_cast<const T*>(p.dy) + row * p.lddy, c, W);
      q.f[i] = load_raw<SHORT>(static_cast<const R*>(p.h) + row * p.ldh, c, W);
      if (RESID && p.dh) q.dh[i] = load_raw<SHORT>(static_cast<const R*>(p.dh) + row * p.lddh, c, W);
    }
    q.mean = p.mean[row];
    q.rstd = p.rstd[row];
  };
  // the next row's loads go out in front of this row's sums where that costs at most 12 registers (16384 x 1024 bf16: 21.9
  // against 22.9 us; with an fp32 stream the registers cost more waves than the loads bring: 8192 x 1024 36.3 against 35.2)
  constexpr bool AHEAD = NV * (sizeof(T) + (RESID ? 2 : 1) * sizeof(R)) <= 6;
  const int64_t step = (int64_t)gridDim.x * GROUPS;
  In next;
  if constexpr (AHEAD) load((int64_t)blockIdx.x * GROUPS + g, next);
  for (int64_t base = (int64_t)blockIdx.x * GROUPS; base < p.rows; base += step) {
    const int64_t row = base + g;
    const int width = row < p.rows ? W : 0;
    In in;
    if constexpr (AHEAD) {
      in = next;
      if (base + step < p.rows) load(row + step, next);
    } else {
      load(row, in);
    }
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * LANES + lane) * ROW_UNIT;
      settle2(in.d[i], in.f[i], c, width);         // (dy is 0 behind the row's end and in a group without a row)
#pragma unroll
      for (int e = 0; e < ROW_UNIT; ++e) {
        const float v = in.d[i].get(e), hat = (in.f[i].get(e) - in.mean) * in.rstd, t = v * gm[i][e];
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
        const float hat = (in.f[i].get(e) - in.mean) * in.rstd;
        o[e] = in.rstd * (fmaf(in.d[i].get(e), gm[i][e], -c1) - hat * c2);
      }
      if constexpr (RESID) {
        if (p.dh) {
          settle(in.dh[i], c, width);
#pragma unroll
          for (int e = 0; e < ROW_UNIT; ++e) o[e] += in.dh[i].get(e);
        }
        if (p.dres) store_unit(static_cast<R*>(p.dres) + row * p.width, c, width, o);
        if (p.dx && p.drop.threshold) drop_unit(key, p.drop, p.drop.row_offset + row, u, o);
      }
      if (p.dx) store_unit(static_cast<T*>(p.dx) + row * p.width, c, width, o);
    }
  }
  if (FEW || !p.part) return;
  const int share = LANES < 64 ? threadIdx.x >> 6 : threadIdx.x / LANES;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * LANES + lane) * ROW_UNIT;
    if constexpr (LANES < 64) {
#pragma unroll
      for (int e = 0; e < ROW_UNIT; ++e)
#pragma unroll
        for (int o = LANES; o < 64; o <<= 1) {
          ag[i][e] += __shfl_xor(ag[i][e], o);
          ab[i][e] += __shfl_xor(ab[i][e], o);
        }
    }
    const bool mine = (LANES >= 64 || (threadIdx.x & 63) < LANES) && c < W;
    f32x4 a[4] = {{ag[i][0], ag[i][1], ag[i][2], ag[i][3]}, {ag[i][4], ag[i][5], ag[i][6], ag[i][7]},
                  {ab[i][0], ab[i][1], ab[i][2], ab[i][3]}, {ab[i][4], ab[i][5], ab[i][6], ab[i][7]}};
    const int64_t at[4] = {c / 4, c / 4 + 1, (p.stride + c) / 4, (p.stride + c) / 4 + 1};
    if constexpr (SHARES > 1) {
      static_assert(NV == 1 || SHARES == 1, "one unit a lane where shares meet in LDS");
      if (mine && share > 0) {
#pragma unroll
        for (int k = 0; k < 4; ++k) cols4[(share - 1) * (p.stride / 2) + at[k]] = a[k];
      }
      __syncthreads();
    }
    if (mine && share == 0) {
      f32x4* out = reinterpret_cast<f32x4*>(p.part + (int64_t)blockIdx.x * 2 * p.stride);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
#pragma unroll
        for (int n = 1; n < SHARES; ++n) a[k] += cols4[(n - 1) * (p.stride / 2) + at[k]];
        out[at[k]] = a[k];
      }
    }
  }
}

// rows of one partial sum of the wide form: whole groups of 16 rows, at most 256 chunks
static int64_t norm_chunk(int64_t rows) { return round_up(std::max<int64_t>(1, ceil_div(rows, 256)), 16); }
static int64_t norm_stride(int64_t width) { return round_up(width, ROW_UNIT); }
static constexpr int64_t ROW_RESIDENT = 16384;     // widest row that stays in registers
// Blocks of the resident backward: 16 waves a CU, in two blocks of 512 threads, or in one of 1024 where a row is over 1024
// columns and its partial sums are the larger cost (16384 x 2048 bf16 residual norm 65.3 against 68.4 us, 8192 x 4096 67.2
// against 72.8; 1024 blocks of 256 threads 73).
static constexpr int64_t ROW_TWO_BLOCKS = 1024;
static int norm_blocks(int64_t width) { return width <= ROW_TWO_BLOCKS ? 512 : 256; }
// One launch without partial sums (norm_few_cols) for few rows.  Kernel time, first launch's start to last one's end, on the
// same tensors again and again (on others in turn 12.5 us for 1024 rows of 1024), of 64 / 512 / 1024 / 2048 rows of 1024 bf16: 4.3 / 6.3 / 9.1 / 14.1 us, by the two launches 15.8 / 16.3 / 15.1 / 15.2 (2048
// columns: 4.3 / 6.8 / 10.0 / 22.8 against 15.9 / 15.3 / 16.8 / 16.4).
static bool norm_few(int64_t rows, int64_t width) { return rows > 0 && rows <= 1024 && width <= 4096; }
static int norm_partials(int64_t rows, int64_t width) {
  if (norm_few(rows, width)) return 0;
  return (int)(width <= ROW_RESIDENT ? std::min<int64_t>(rows, norm_blocks(width)) : ceil_div(rows, norm_chunk(rows)));
}

template <typename T, typename R, bool RESID, int LANES, int NV, bool SHORT = false>
static int launch_fwd_rows(hipStream_t s, const NormFwd& p) {
  constexpr int BLOCK = LANES > 256 ? LANES : 256;
  // at most 8 blocks of 256 threads a CU, which walk the rows with the parameters in registers: 16384 x 2048 bf16 layer
  // norm 22.4 us, one group of rows a block (parameters read for each) 27.6.  The layer norm of rows of 1 to 4 KiB runs
  // better in 6 a CU (4096 x 1024 fp32 8.4 against 9.5 us, 16384 x 1001 fp16 12.2 against 13.3, 16384 x 1024 bf16 11.6
  // against 12.0); shorter rows (65536 x 256 bf16 13.7 against 12.8) and the residual norm (16384 x 2048 bf16 47.0 against
  // 44.3) do not.
  constexpr int bytes = LANES * NV * ROW_UNIT * (int)sizeof(T);
  constexpr int most = (!RESID && NV <= 2 && bytes >= 1024 && bytes <= 4096 ? 6 : 8) * 256;
  const unsigned blocks = (unsigned)std::min<int64_t>(ceil_div(p.rows, BLOCK / LANES), most * 256 / BLOCK);
  hipLaunchKernelGGL((norm_fwd_rows_kernel<T, R, RESID, LANES, NV, BLOCK, SHORT>), dim3(blocks), dim3(BLOCK), 0, s, p);
  BLH_HIP_TRY(hipGetLastError());
  return BLH_OK;
}

// Lanes a row.  16-bit rows of up to 2048 columns belong to one wave (two for the residual norm, which holds two streams) of
// 2 or 4 units a lane: no barrier, and the parameters' registers are spent once per row in flight (16384 x 2048 bf16:
// 22.4 us, spread over four waves 25.0).  fp32 rows are twice the bytes and go to twice the lanes (8192 x 1024: 12.6 against
// 14.0 us).  Few rows — at most eight a CU — are spread too, one unit a lane: nothing else hides a row's latency (1 x 2048
// residual norm 5.3 us, by one wave 8.3).
template <typename T, typename R, bool RESID>
static int launch_norm_fwd(hipStream_t s, const NormFwd& p) {
  constexpr bool wide = sizeof(T) == 4;
  const bool few = p.rows <= 2048;
  if (p.width < ROW_UNIT) return launch_fwd_rows<T, R, RESID, 8, 1, true>(s, p);
  if (p.width <= 64) return launch_fwd_rows<T, R, RESID, 8, 1>(s, p);
  if (p.width <= 128) return launch_fwd_rows<T, R, RESID, 16, 1>(s, p);
  if (p.width <= 256) return launch_fwd_rows<T, R, RESID, 32, 1>(s, p);
  if (p.width <= 512) return launch_fwd_rows<T, R, RESID, 64, 1>(s, p);
  if (p.width <= 1024) {
    if (wide || few) return launch_fwd_rows<T, R, RESID, 128, 1>(s, p);
    if constexpr (!wide) return launch_fwd_rows<T, R, RESID, 64, 2>(s, p);
  }
  if (p.width <= 2048) {
    if (wide || few) return launch_fwd_rows<T, R, RESID, 256, 1>(s, p);
    if constexpr (!wide) return launch_fwd_rows<T, R, RESID, RESID ? 128 : 64, RESID ? 2 : 4>(s, p);
  }
  if (p.width <= 4096) return launch_fwd_rows<T, R, RESID, wide ? 512 : 256, wide ? 1 : 2>(s, p);
  if (p.width <= 8192) return launch_fwd_rows<T, R, RESID, wide ? 512 : 256, wide ? 2 : 4>(s, p);
  if (p.width <= ROW_RESIDENT) return launch_fwd_rows<T, R, RESID, 1024, 2>(s, p);
  const unsigned blocks = (unsigned)std::min<int64_t>(p.rows, 1 << 16);
  hipLaunchKernelGGL((norm_fwd_kernel<T, R, RESID>), dim3(blocks), dim3(256), 0, s, p);
  BLH_HIP_TRY(hipGetLastError());
  return BLH_OK;
}

template <typename T, typename R, bool RESID, int LANES, int NV, int BLOCK, bool SHORT = false>
static int launch_bwd_rows(hipStream_t s, NormBwd& p) {
  p.chunks = (int)std::min<int64_t>(ceil_div(p.rows, BLOCK / LANES), norm_blocks(p.width));
  const size_t lds = p.part ? (bwd_shares<LANES, BLOCK>() - 1) * 2 * p.stride * sizeof(float) : 0;    // at most 48 KiB
  hipLaunchKernelGGL((norm_bwd_kernel<T, R, RESID, LANES, NV, BLOCK, SHORT, false>), dim3((unsigned)p.chunks), dim3(BLOCK), lds, s,
                     p);
  BLH_HIP_TRY(hipGetLastError());
  return BLH_OK;
}

template <typename T, typename R, bool RESID, int LANES, bool SHORT = false>
static int launch_bwd_few(hipStream_t s, NormBwd p) {
  p.row_blocks = p.dx || p.dres ? (int)ceil_div(p.rows, 512 / LANES) : 0;
  const unsigned blocks = (unsigned)(p.row_blocks + ceil_div(p.width, 64));
  hipLaunchKernelGGL((norm_bwd_kernel<T, R, RESID, LANES, 1, 512, SHORT, true>), dim3(blocks), dim3(512), 0, s, p);
  BLH_HIP_TRY(hipGetLastError());
  return BLH_OK;
}

template <typename T, typename R, bool RESID>
static int launch_norm_bwd(hipStream_t s, NormBwd p) {
  const bool grads = p.dgamma || p.dbeta;
  p.stride = norm_stride(p.width);
  if (!grads) p.part = nullptr;
  if (grads && norm_few(p.rows, p.width)) {
    if (p.width < ROW_UNIT) return launch_bwd_few<T, R, RESID, 8, true>(s, p);
    if (p.width <= 64) return launch_bwd_few<T, R, RESID, 8>(s, p);
    if (p.width <= 128) return launch_bwd_few<T, R, RESID, 16>(s, p);
    if (p.width <= 512) return launch_bwd_few<T, R, RESID, 64>(s, p);
    if (p.width <= 1024) return launch_bwd_few<T, R, RESID, 128>(s, p);
    if (p.width <= 2048) return launch_bwd_few<T, R, RESID, 256>(s, p);
    return launch_bwd_few<T, R, RESID, 512>(s, p);
  }
  if (p.rows > 0 && p.width <= ROW_RESIDENT) {
    if (p.width < ROW_UNIT) BLH_TRY((launch_bwd_rows<T, R, RESID, 8, 1, 512, true>(s, p)));
    else if (p.width <= 64) BLH_TRY((launch_bwd_rows<T, R, RESID, 8, 1, 512>(s, p)));
    else if (p.width <= 128) BLH_TRY((launch_bwd_rows<T, R, RESID, 16, 1, 512>(s, p)));
    else if (p.width <= 256) BLH_TRY((launch_bwd_rows<T, R, RESID, 32, 1, 512>(s, p)));
    else if (p.width <= 512) BLH_TRY((launch_bwd_rows<T, R, RESID, 64, 1, 512>(s, p)));
    else if (p.width <= 1024) BLH_TRY((launch_bwd_rows<T, R, RESID, 128, 1, 512>(s, p)));
    else if (p.width <= 2048) BLH_TRY((launch_bwd_rows<T, R, RESID, 256, 1, 1024>(s, p)));
    else if (p.width <= 4096) BLH_TRY((launch_bwd_rows<T, R, RESID, 512, 1, 1024>(s, p)));
    else if (p.width <= 8192) BLH_TRY((launch_bwd_rows<T, R, RESID, 1024, 1, 1024>(s, p)));
    else BLH_TRY((launch_bwd_rows<T, R, RESID, 1024, 2, 1024>(s, p)));
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
  switch (dtype) {
    case BLH_F32: return launch_norm_fwd<float, float, true>(s, p);
    case BLH_BF16:
      return rtype == BLH_F32 ? launch_norm_fwd<bf16_t, float, true>(s, p) : launch_norm_fwd<bf16_t, bf16_t, true>(s, p);
    default:
      return rtype == BLH_F32 ? launch_norm_fwd<f16_t, float, true>(s, p) : launch_norm_fwd<f16_t, f16_t, true>(s, p);
  }
}
static int resid_bwd(hipStream_t s, const NormBwd& p, int32_t dtype, int32_t rtype) {
  switch (dtype) {
    case BLH_F32: return launch_norm_bwd<float, float, true>(s, p);
    case BLH_BF16:
      return rtype == BLH_F32 ? launch_norm_bwd<bf16_t, float, true>(s, p) : launch_norm_bwd<bf16_t, bf16_t, true>(s, p);
    default:
      return rtype == BLH_F32 ? launch_norm_bwd<f16_t, float, true>(s, p) : launch_norm_bwd<f16_t, f16_t, true>(s, p);
  }
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
  if (d.step_used && !d.threshold) BLH_TRY(row_write_step((hipStream_t)stream, d));
  return resid_fwd((hipStream_t)stream, p, dtype, stream_dtype);
}

int64_t blh_row_norm_workspace_bytes(int64_t rows, int64_t width) {
  BLH_TRY(row_check_shape(rows, width));
  return (int64_t)norm_partials(rows, width) * 2 * norm_stride(width) * (int64_t)sizeof(float);
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
  const int64_t need = dweight || dbias ? blh_row_norm_workspace_bytes(rows, width) : 0;
  if (need > 0 && (!workspace || (uintptr_t)workspace % 16 != 0)) return BLH_ERR_INVALID_ARGUMENT;
  if (need > workspace_bytes) return BLH_ERR_WORKSPACE;
  const NormBwd p{dy, nullptr, x, weight, mean, rstd, dx, nullptr, dweight, dbias, static_cast<float*>(workspace),
                  lddy, 0, ldx, rows, width, 0, 0, 0, 0, param_dtype == dtype, NO_DROP};
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
  const int64_t need = dweight || dbias ? blh_row_norm_workspace_bytes(rows, width) : 0;
  if (need > 0 && (!workspace || (uintptr_t)workspace % 16 != 0)) return BLH_ERR_INVALID_ARGUMENT;
  if (need > workspace_bytes) return BLH_ERR_WORKSPACE;
  const NormBwd p{dy, dh, h, weight, mean, rstd, dx, dresidual, dweight, dbias, static_cast<float*>(workspace),
                  lddy, lddh, ldh, rows, width, 0, 0, 0, 0, param_dtype == dtype, d};
  return resid_bwd((hipStream_t)stream, p, dtype, stream_dtype);
}

}  // extern "C"
