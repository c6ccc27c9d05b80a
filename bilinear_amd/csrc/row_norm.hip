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
  float* part;          // [chunks][2][width]
  int64_t lddy, lddh, ldh, rows, width, chunk;
  int chunks;
  bool same;
  RowDrop drop;
};

// sums over the block's 4 waves; `sh` may be reused after the next barrier
__device__ __forceinline__ float block_sum(float v, float* sh) {
  v = wave_sum(v);
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
      p.part[(blockIdx.y * 2 + which) * W + c0 + j] =
          (sh[0][which][j] + sh[1][which][j]) + (sh[2][which][j] + sh[3][which][j]);
  }
}

// dgamma, dbeta = sums of the chunks' partials, in the parameters' type (chunks == 0: zeros)
template <typename T>
__global__ __launch_bounds__(256) void norm_bwd_finish_kernel(NormBwd p) {
  const int64_t W = p.width, j = blockIdx.x * 256ll + threadIdx.x;
  if (j >= W) return;
  const int which = blockIdx.y;
  void* out = which ? p.dbeta : p.dgamma;
  if (!out) return;
  float s = 0.f;
  for (int k = 0; k < p.chunks; ++k) s += p.part[((int64_t)k * 2 + which) * W + j];
  if (p.same) static_cast<T*>(out)[j] = (T)s;
  else static_cast<float*>(out)[j] = s;
}

// rows of one partial sum: whole groups of 16 rows, at most 256 chunks
static int64_t norm_chunk(int64_t rows) { return round_up(std::max<int64_t>(1, ceil_div(rows, 256)), 16); }
static int norm_chunks(int64_t rows) { return (int)ceil_div(rows, norm_chunk(rows)); }

template <typename T, typename R, bool RESID>
static int launch_norm_fwd(hipStream_t s, const NormFwd& p) {
  const unsigned blocks = (unsigned)std::min<int64_t>(p.rows, 1 << 16);
  hipLaunchKernelGGL((norm_fwd_kernel<T, R, RESID>), dim3(blocks), dim3(256), 0, s, p);
  BLH_HIP_TRY(hipGetLastError());
  return BLH_OK;
}

template <typename T, typename R, bool RESID>
static int launch_norm_bwd(hipStream_t s, NormBwd p) {
  if (p.rows > 0 && (p.dx || p.dres)) {
    const unsigned blocks = (unsigned)std::min<int64_t>(p.rows, 1 << 16);
    hipLaunchKernelGGL((norm_bwd_rows_kernel<T, R, RESID>), dim3(blocks), dim3(256), 0, s, p);
    BLH_HIP_TRY(hipGetLastError());
  }
  if (p.dgamma || p.dbeta) {
    p.chunk = norm_chunk(p.rows);
    p.chunks = norm_chunks(p.rows);
    if (p.chunks > 0) {
      const dim3 grid((unsigned)ceil_div(p.width, 64 * ROW_UNIT), (unsigned)p.chunks);
      hipLaunchKernelGGL((norm_bwd_cols_kernel<T, R>), grid, dim3(256), 0, s, p);
      BLH_HIP_TRY(hipGetLastError());
    }
    hipLaunchKernelGGL((norm_bwd_finish_kernel<T>), dim3((unsigned)ceil_div(p.width, 256), 2), dim3(256), 0, s, p);
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
  return std::max<int64_t>(256, (int64_t)norm_chunks(rows) * 2 * width * (int64_t)sizeof(float));
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
                  lddy, 0, ldx, rows, width, 0, 0, param_dtype == dtype, NO_DROP};
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
                  lddy, lddh, ldh, rows, width, 0, 0, param_dtype == dtype, d};
  return resid_bwd((hipStream_t)stream, p, dtype, stream_dtype);
}

}  // extern "C"
