// Dropout of rows with a mask that is regenerated, never stored.
//
//   y[i][j] = u(i, j) >= t ? s x[i][j] : 0,    t = floor(65536 p + 1/2),  s = 65536 / (65536 - t)
//
// u(i, j): 16 bits of Philox4x32-10, one call for 8 columns of one GLOBAL row (row_offset + i):
//   counter (row lo, j / 8 | row hi << 21, layer | 2^31, step lo), key (seed lo ^ step hi, seed hi),
//   element e = j % 8 takes the half e & 1 of word e / 2.
// The mask depends on (seed, step, layer, global row, column) alone: not on the type, the launch or how rows are spread
// over devices.  p is rounded to a multiple of 2^-16 and s is the exact inverse of the rounded keep probability, so the
// expectation of y is x.  The backward pass is the same map on dy: there is nothing to save.
//
// Bound by memory: 16384 x 2048 bf16 22.4 us = 6.0 TB/s of its bytes over and over on three inputs in turn (a copy in the same
// loop 19.5), 25 us = 5.3 among the other operators on 800 MB (a copy of 537 MB: 5.4); a stored mask of one bit would add 3 % to a 16-bit type's bytes
// each way.  A draw takes 16 bits so that a call, 20 multiplies, serves 8 elements.
#include "row_ops.h"
#include "row_ops_dev.h"

namespace blh {

int row_make_drop(const blh_row_drop* d, int64_t rows, RowDrop* out) {
  if (!(d->p >= 0.0 && d->p <= 1.0) || d->layer < 0 || d->row_offset < 0 ||
      (d->step_used && d->step_used == d->step_dev))
    return BLH_ERR_INVALID_ARGUMENT;
  if (d->row_offset > ROW_MAX_ROWS - rows) return BLH_ERR_SHAPE;
  const uint32_t t = (uint32_t)(d->p * 65536.0 + 0.5);
  *out = RowDrop{d->seed, d->step, d->step_dev, d->step_used, d->row_offset, (uint32_t)d->layer | 0x80000000u, t,
                 t < 65536u ? (float)(65536.0 / (double)(65536u - t)) : 0.f};
  return BLH_OK;
}

__global__ void row_write_step_kernel(RowDrop drop) { row_key(drop); }

int row_write_step(hipStream_t s, const RowDrop& drop) {
  hipLaunchKernelGGL(row_write_step_kernel, dim3(1), dim3(1), 0, s, drop);
  BLH_HIP_TRY(hipGetLastError());
  return BLH_OK;
}

// I: the type that counts units: 32 bits wherever they fit, since the index costs a division by `units` (65536 x 64 bf16 5.4
// against 5.8 us)
template <typename T, typename I, bool SHORT>
__global__ __launch_bounds__(256) void row_dropout_kernel(const T* x, int64_t ldx, T* y, RowDrop drop, I total, I units,
                                                          int width) {
  const RowKey key = row_key(drop);
  for (I i = (I)blockIdx.x * 256 + threadIdx.x; i < total; i += (I)gridDim.x * 256) {
    const I row = i / units;
    const int unit = (int)(i - row * units), c = unit * ROW_UNIT;
    float f[ROW_UNIT];
    load_unit<SHORT>(x + (int64_t)row * ldx, c, width, f);
    drop_unit(key, drop, drop.row_offset + (int64_t)row, unit, f);
    store_unit(y + (int64_t)row * width, c, width, f);
  }
}

template <typename T>
static int launch_row_dropout(hipStream_t s, const void* x, int64_t ldx, void* y, const RowDrop& drop, int64_t rows,
                              int64_t width) {
  const int64_t units = ceil_div(width, ROW_UNIT), total = rows * units;
  const unsigned blocks = (unsigned)std::min<int64_t>(ceil_div(total, 256), 4096);
  const T* in = static_cast<const T*>(x);
  T* out = static_cast<T*>(y);
  // (32 bits: the loop's index passes `total` by at most one grid)
  if (width < ROW_UNIT)
    hipLaunchKernelGGL((row_dropout_kernel<T, uint64_t, true>), dim3(blocks), dim3(256), 0, s, in, ldx, out, drop,
                       (uint64_t)total, (uint64_t)units, (int)width);
  else if (total < (int64_t)1 << 31)
    hipLaunchKernelGGL((row_dropout_kernel<T, uint32_t, false>), dim3(blocks), dim3(256), 0, s, in, ldx, out, drop,
                       (uint32_t)total, (uint32_t)units, (int)width);
  else
    hipLaunchKernelGGL((row_dropout_kernel<T, uint64_t, false>), dim3(blocks), dim3(256), 0, s, in, ldx, out, drop,
                       (uint64_t)total, (uint64_t)units, (int)width);
  BLH_HIP_TRY(hipGetLastError());
  return BLH_OK;
}

}  // namespace blh

using namespace blh;

extern "C" {

int blh_row_dropout(void* stream, const void* x, int64_t ldx, void* y, const blh_row_drop* drop, int64_t rows,
                    int64_t width, int32_t dtype) {
  if (!drop || !row_dtype_ok(dtype) || ldx < 0) return BLH_ERR_INVALID_ARGUMENT;
  BLH_TRY(row_check_shape(rows, width));
  RowDrop d;
  BLH_TRY(row_make_drop(drop, rows, &d));
  if (rows == 0) return BLH_OK;
  if (!x || !y || !row_aligned(x, dtype) || !row_aligned(y, dtype)) return BLH_ERR_INVALID_ARGUMENT;
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case BLH_F32: return launch_row_dropout<float>(s, x, ldx, y, d, rows, width);
    case BLH_BF16: return launch_row_dropout<bf16_t>(s, x, ldx, y, d, rows, width);
    default: return launch_row_dropout<f16_t>(s, x, ldx, y, d, rows, width);
  }
}

}  // extern "C"
