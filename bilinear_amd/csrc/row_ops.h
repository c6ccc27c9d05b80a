// Host-side arithmetic and launchers of the row operators (row_norm.hip, row_dropout.hip).
#pragma once
#include "common.h"

namespace blh {

static constexpr int64_t ROW_MAX_WIDTH = (int64_t)1 << 24;   // a unit's index keeps 21 bits of its Philox counter word
static constexpr int64_t ROW_MAX_ROWS = (int64_t)1 << 43;    // ... and a global row 32 + 11 bits

static inline bool row_dtype_ok(int32_t t) { return t == BLH_F32 || t == BLH_BF16 || t == BLH_F16; }
static inline int row_dtype_bytes(int32_t t) { return t == BLH_F32 ? 4 : 2; }
static inline bool row_aligned(const void* p, int32_t t) { return (uintptr_t)p % row_dtype_bytes(t) == 0; }

// BLH_ERR_SHAPE for sizes the counters cannot hold; rows == 0 is an empty call
static inline int row_check_shape(int64_t rows, int64_t width) {
  if (rows < 0 || width < 1) return BLH_ERR_INVALID_ARGUMENT;
  if (rows > ROW_MAX_ROWS || width > ROW_MAX_WIDTH) return BLH_ERR_SHAPE;
  return BLH_OK;
}

struct RowDrop;
// threshold = floor(65536 p + 1/2), scale = 65536 / (65536 - threshold); refuses p outside [0, 1] and rows past 2^43
int row_make_drop(const blh_row_drop* d, int64_t rows, RowDrop* out);
// *step_used = step + *step_dev, for a call whose kernel drops nothing and so does not look (in that kernel the write costs
// registers: 4096 x 5000 fp16 residual norm on an fp32 stream 51.1 against 48.5 us)
int row_write_step(hipStream_t s, const RowDrop& drop);

}  // namespace blh
