// Helpers shared by the library's translation units (not part of the C ABI): the calling
// thread's last-error message behind tabby_last_error(), and a HIP status check.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <string>

#include "tabby_sampler.h"

namespace tabby {

// Records `msg` as the calling thread's last error and returns `status`.
int record_failure(int status, const std::string &msg);

inline int record_hip_failure(hipError_t e, const char *what) {
  return record_failure(TABBY_EHIP, std::string(what) + ": " + hipGetErrorString(e));
}

// The device's compute-unit count (cached per device).
int device_cus(int device, int *cus);

// What the library's other kernels may use of a sampler handle: its device, its limits, and
// its candidate region as scratch (rows_max * vocab_max composites of 8 bytes). The scratch
// is shared with the sampling kernels; calls on one handle are stream-ordered and must not
// overlap, as for every entry point that takes a handle.
struct HandleView {
  int device;
  int cus;
  int32_t vocab_max, rows_max, k_max;
  void *scratch;
  size_t scratch_bytes;
};
int handle_view(const tabby_sampler *h, HandleView *out);

// The int4 lm_head's shape rules (hidden and block_size multiples of 32, block_size dividing
// hidden); TABBY_EINVAL with a message otherwise.
int check_q4_shape(int32_t vocab, int32_t hidden, int32_t block);

// Rows in memory: `rows` of `row_bytes` each, `stride` bytes apart.
struct RowSpan {
  const void *base;
  int64_t rows, row_bytes, stride;
  int64_t bytes() const { return (rows - 1) * stride + row_bytes; }
};

// Rows of `cols` elements of `size` bytes, `stride` elements apart. (One row has no stride, and what lies further
// apart than an address space is as good as that.)
inline RowSpan row_span(const void *base, int64_t rows, int64_t cols, int64_t stride, int64_t size) {
  const int64_t far = INT64_MAX / (8 * (rows < 1 ? 1 : rows));
  return {base, rows, cols * size, rows > 1 ? (stride < far ? stride : far) * size : 0};
}

// Whether `bytes` at `at` meet one of the rows.
inline bool rows_meet(const RowSpan &s, const void *at, int64_t bytes) {
  const int64_t from = (int64_t)(uintptr_t)at - (int64_t)(uintptr_t)s.base;
  const int64_t row = from < s.row_bytes ? 0 : s.rows > 1 ? (from - s.row_bytes) / s.stride + 1 : 1;  // the first that ends after `at`
  return row < s.rows && row * s.stride < from + bytes;
}

// MXFP4 matrices: the sizes a matrix may have, the pointers of one, and the conversion itself
// (arguments checked by the caller).
int check_mx4_shape(int32_t rows, int32_t cols);
int check_mx4_operand(const void *codes, const void *scales);
// What a call writes must not lie on what it reads: TABBY_EINVAL if the rows meet the matrix.
int check_mx4_apart(const RowSpan &rows, const void *codes, const void *scales, int32_t m_rows, int32_t m_cols);
int mx4_quantize(const void *x, int32_t dtype, int32_t rows, int32_t cols, int64_t stride, uint8_t *codes,
                 uint8_t *scales, hipStream_t s);

// FP8 matrices, likewise; block_rows 1 or 128.
int check_fp8_shape(int32_t rows, int32_t cols, int32_t block_rows);
void fp8_sizes(int32_t rows, int32_t cols, int32_t block_rows, int64_t *code_bytes, int64_t *scale_bytes);
int check_fp8_operand(const void *codes, const void *scales);
int check_fp8_apart(const RowSpan &rows, const void *codes, const void *scales, int32_t m_rows, int32_t m_cols, int32_t block_rows);
int fp8_quantize(const void *x, int32_t dtype, int32_t rows, int32_t cols, int64_t stride, int32_t block_rows, uint8_t *codes,
                 float *scales, hipStream_t s);

}  // namespace tabby

#define TABBY_HIP_CHECK(expr)                                            \
  do {                                                                   \
    hipError_t e_ = (expr);                                              \
    if (e_ != hipSuccess) return ::tabby::record_hip_failure(e_, #expr); \
  } while (0)
