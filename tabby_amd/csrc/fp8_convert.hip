// FP8 conversions: a matrix to codes and scales (fp8.h has the layout), the way back, and the repacking of a
// checkpoint's row-major codes.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <string>

#include "abi_internal.h"
#include "elem.h"
#include "fp8.h"

namespace tabby {
namespace {

constexpr unsigned kConvertGrid = 1u << 20;

// Both directions are bound by HBM. A workgroup takes a panel, or the two panels of a square block, along the
// rows, 16 bytes to a lane; the codes change places in LDS, so that either side moves whole lines.
template <int DT, int BR>
struct BlockWalk {
  using E = Elem<DT>;
  static constexpr int kThreads = BR == 1 ? 256 : 512;
  static constexpr int kPanels = BR == 1 ? 1 : kF8Block / kF8PanelRows;  // of a workgroup's step
  static constexpr int kRows = kPanels * kF8PanelRows;
  static constexpr int kRowLanes = kF8PanelCols / E::kVec;       // lanes to a row
  static constexpr int kRowStep = kThreads / kRowLanes;
  static constexpr int kSteps = kRows / kRowStep;                // rows of a thread
  int row, col;  // the first row; its column in the panel
  __device__ __forceinline__ BlockWalk()
      : row((int)threadIdx.x / kRowLanes), col((int)threadIdx.x % kRowLanes * E::kVec) {}
};

// 151,936 x 896 f16 to square blocks: 62 us, 408 MB at 6.5 TB/s, and 59 us back; 1,531 x 4,850 bf16, whose rows lie off
// 16 bytes: 8.4 us; one row of 896 f32: 3.6 us, a launch's latency.
template <int DT, int BR, bool WHOLE>
__global__ __launch_bounds__(BR == 1 ? 256 : 512) void fp8_quantize_kernel(const typename Elem<DT>::Bits *x, int rows, int cols,
                                                                           int64_t stride, uint8_t *codes, float *scales) {
  using Walk = BlockWalk<DT, BR>;
  __shared__ __align__(16) uint8_t held[Walk::kPanels * kF8PanelBytes];
  __shared__ float row_scales[kF8PanelRows];
  __shared__ uint32_t wave_top[Walk::kThreads / 64];
  const Walk walk;
  const int t = (int)threadIdx.x;
  const int64_t col_panels = f8_parts(cols, kF8PanelCols), blocks = f8_parts(rows, Walk::kRows) * col_panels;
  const int64_t row_panels = f8_parts(rows, kF8PanelRows);
  for (int64_t block = blockIdx.x; block < blocks; block += gridDim.x) {
    const int64_t block_row = block / col_panels, block_col = block - block_row * col_panels;
    const int64_t row0 = block_row * Walk::kRows;
    const int col0 = (int)block_col * kF8PanelCols;
    u32x4 raw[Walk::kSteps];
#pragma unroll
    for (int i = 0; i < Walk::kSteps; ++i) {
      const int64_t row = row0 + walk.row + i * Walk::kRowStep;
      raw[i] = row < rows ? load_values<DT, WHOLE>(x + row * stride, col0 + walk.col, cols) : u32x4{0, 0, 0, 0};
    }
    if constexpr (BR == 1) {
#pragma unroll
      for (int i = 0; i < Walk::kSteps; ++i) {
        const int r = walk.row + i * Walk::kRowStep;
        uint32_t top = f8_largest<DT>(raw[i]);
#pragma unroll
        for (int lanes = 1; lanes < Walk::kRowLanes; lanes *= 2) top = max(top, xor_lane_by(top, lanes));
        float scale, inverse;
        f8_scale(top, scale, inverse);
        f8_encode<DT>(&held[f8_code_byte(r, walk.col)], raw[i], inverse);
        if (walk.col == 0) row_scales[r] = scale;
      }
    } else {
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < Walk::kSteps; ++i) top = max(top, f8_largest<DT>(raw[i]));
      top = wave_max_u32(top);
      if ((t & 63) == 0) wave_top[t >> 6] = top;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < Walk::kThreads / 64; ++w) top = max(top, wave_top[w]);
      float scale, inverse;
      f8_scale(top, scale, inverse);
#pragma unroll
      for (int i = 0; i < Walk::kSteps; ++i) {
        const int r = walk.row + i * Walk::kRowStep;
        f8_encode<DT>(&held[r / kF8PanelRows * kF8PanelBytes + f8_code_byte(r % kF8PanelRows, walk.col)], raw[i], inverse);
      }
      if (t == 0) scales[block] = scale;
    }
    __syncthreads();
#pragma unroll
    for (int p = 0; p < Walk::kPanels; ++p) {
      const int64_t panel_row = block_row * Walk::kPanels + p;
      if (panel_row >= row_panels) break;
      u32x4 *to = reinterpret_cast<u32x4 *>(codes + (panel_row * col_panels + block_col) * kF8PanelBytes);
      const u32x4 *from = reinterpret_cast<const u32x4 *>(held + p * kF8PanelBytes);
#pragma unroll
      for (int i = t; i < kF8PanelBytes / 16; i += Walk::kThreads) to[i] = from[i];
    }
    if constexpr (BR == 1) {
      if (t < kF8PanelRows) scales[block * kF8PanelRows + t] = row_scales[t];
    }
    __syncthreads();
  }
}

template <int DT>
__global__ __launch_bounds__(256) void fp8_dequantize_kernel(Fp8Matrix m, int block_rows, typename Elem<DT>::Bits *out,
                                                             int64_t stride, bool whole) {
  using E = Elem<DT>;
  using Walk = BlockWalk<DT, 1>;
  __shared__ __align__(16) uint8_t held[kF8PanelBytes];
  const Walk walk;
  const int t = (int)threadIdx.x;
  const int64_t col_panels = m.col_panels(), panels = f8_parts(m.rows, kF8PanelRows) * col_panels;
  for (int64_t panel = blockIdx.x; panel < panels; panel += gridDim.x) {
    const int64_t panel_row = panel / col_panels, panel_col = panel - panel_row * col_panels;
    const int64_t row0 = panel_row * kF8PanelRows;
    const int col = (int)panel_col * kF8PanelCols + walk.col;
    const u32x4 *from = reinterpret_cast<const u32x4 *>(m.codes + panel * kF8PanelBytes);
#pragma unroll
    for (int i = 0; i < kF8PanelBytes / 16 / Walk::kThreads; ++i)
      reinterpret_cast<u32x4 *>(held)[t + i * Walk::kThreads] = from[t + i * Walk::kThreads];
    // Two panels of rows to a square block.
    const float *scales = block_rows == 1 ? m.scales + panel * kF8PanelRows : m.scales + (panel_row >> 1) * col_panels + panel_col;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < Walk::kSteps; ++i) {
      const int r = walk.row + i * Walk::kRowStep;
      const int64_t row = row0 + r;
      if (row >= m.rows || col >= m.cols) continue;
      const float scale = scales[block_rows == 1 ? r : 0];
      float v[E::kVec];
      const uint32_t *word = reinterpret_cast<const uint32_t *>(&held[f8_code_byte(r, walk.col)]);
#pragma unroll
      for (int j = 0; j < E::kVec / 4; ++j) f8_decode4(word[j], v + 4 * j);
#pragma unroll
      for (int j = 0; j < E::kVec; ++j) v[j] *= scale;
      typename E::Bits *to = out + row * stride + col;
      if (col + E::kVec <= m.cols) {
        u32x4 u;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if constexpr (E::kVec == 4) u[j] = E::narrow(v[j]);
          else u[j] = (uint32_t)E::narrow(v[2 * j]) | ((uint32_t)E::narrow(v[2 * j + 1]) << 16);
        }
        if (whole) __builtin_nontemporal_store(u, reinterpret_cast<u32x4 *>(to));
        else *reinterpret_cast<u32x4_any *>(to) = u;
      } else {
#pragma unroll
        for (int j = 0; j < E::kVec; ++j)
          if (col + j < m.cols) to[j] = E::narrow(v[j]);
      }
    }
    __syncthreads();
  }
}

// A checkpoint's codes [rows][cols] to panels; what lies past the last row or column becomes code 0. The scales
// of square blocks are held in the order in which they come.
__global__ __launch_bounds__(256) void fp8_pack_kernel(const uint8_t *src, const float *src_scales, int rows, int cols,
                                                       uint8_t *codes, float *scales) {
  const int64_t col_panels = f8_parts(cols, kF8PanelCols), panels = f8_parts(rows, kF8PanelRows) * col_panels;
  const int t = (int)threadIdx.x;
  for (int64_t panel = blockIdx.x; panel < panels; panel += gridDim.x) {
    const int64_t panel_row = panel / col_panels, panel_col = panel - panel_row * col_panels;
#pragma unroll
    for (int i = 0; i < kF8PanelBytes / 16 / 256; ++i) {
      // The 16 bytes that go to place `at` of the panel.
      const int at = t + i * 256, tile = at >> 7, half = (at >> 6) & 1, lane = at & 63;
      const int64_t row = panel_row * kF8PanelRows + tile * kF8TileRows + (lane & 15);
      const int col = (int)panel_col * kF8PanelCols + 32 * (lane >> 4) + 16 * half;
      u32x4 w = {0, 0, 0, 0};
      if (row < rows && col < cols) {
        const uint8_t *from = src + row * cols + col;
        if (col + 16 <= cols) {
          w = *reinterpret_cast<const u32x4_any *>(from);
        } else {
#pragma unroll
          for (int j = 0; j < 15; ++j)
            if (col + j < cols) w[j / 4] |= (uint32_t)from[j] << (8 * (j % 4));
        }
      }
      reinterpret_cast<u32x4 *>(codes + panel * kF8PanelBytes)[at] = w;
    }
    if (t == 0 && (panel_row & 1) == 0) {
      const int64_t block = (panel_row >> 1) * col_panels + panel_col;
      scales[block] = src_scales[block];
    }
  }
}

dim3 convert_grid(int64_t steps) { return dim3((unsigned)std::min<int64_t>(steps, kConvertGrid)); }

// Whether no two lanes share 16 bytes of memory.
template <int DT>
bool whole_rows(const void *rows, int64_t stride) {
  return (uintptr_t)rows % 16 == 0 && stride % Elem<DT>::kVec == 0;
}

template <int DT, int BR>
int launch_quantize(const void *x, int rows, int cols, int64_t stride, uint8_t *codes, float *scales, hipStream_t s) {
  using Walk = BlockWalk<DT, BR>;
  const auto *from = (const typename Elem<DT>::Bits *)x;
  const dim3 grid = convert_grid(f8_parts(rows, Walk::kRows) * f8_parts(cols, kF8PanelCols)), block(Walk::kThreads);
  if (whole_rows<DT>(x, stride))
    hipLaunchKernelGGL((fp8_quantize_kernel<DT, BR, true>), grid, block, 0, s, from, rows, cols, stride, codes, scales);
  else
    hipLaunchKernelGGL((fp8_quantize_kernel<DT, BR, false>), grid, block, 0, s, from, rows, cols, stride, codes, scales);
  TABBY_HIP_CHECK(hipGetLastError());
  return TABBY_OK;
}

template <int DT>
int launch_quantize(const void *x, int rows, int cols, int64_t stride, int block_rows, uint8_t *codes, float *scales, hipStream_t s) {
  return block_rows == 1 ? launch_quantize<DT, 1>(x, rows, cols, stride, codes, scales, s)
                         : launch_quantize<DT, kF8Block>(x, rows, cols, stride, codes, scales, s);
}

template <int DT>
int launch_dequantize(const Fp8Matrix &m, int block_rows, void *out, int64_t stride, hipStream_t s) {
  const dim3 grid = convert_grid(f8_parts(m.rows, kF8PanelRows) * m.col_panels());
  hipLaunchKernelGGL(fp8_dequantize_kernel<DT>, grid, dim3(256), 0, s, m, block_rows, (typename Elem<DT>::Bits *)out, stride,
                     whole_rows<DT>(out, stride));
  TABBY_HIP_CHECK(hipGetLastError());
  return TABBY_OK;
}

int check_rows(const void *rows_at, int32_t dtype, int32_t rows, int32_t cols, int64_t stride, const char *what) {
  if (!rows_at) return record_failure(TABBY_EINVAL, "null pointer");
  if (!known_dtype(dtype)) return record_failure(TABBY_EINVAL, "dtype must be TABBY_F32, TABBY_F16 or TABBY_BF16");
  if (rows > 1 && stride < cols) return record_failure(TABBY_EINVAL, "row_stride must be at least cols");
  if ((uintptr_t)rows_at % dtype_size(dtype) != 0)
    return record_failure(TABBY_EINVAL, std::string(what) + " must be aligned to its elements");
  return TABBY_OK;
}

}  // namespace

int check_fp8_shape(int32_t rows, int32_t cols, int32_t block_rows) {
  if (rows < 1 || cols < 1) return record_failure(TABBY_EINVAL, "rows and cols must be >= 1");
  if (cols > INT32_MAX - kF8Block || rows > INT32_MAX - kF8Block)
    return record_failure(TABBY_EINVAL, "rows and cols must leave room for their padding in 32 bits");
  if (block_rows != 1 && block_rows != kF8Block)
    return record_failure(TABBY_EINVAL, "block_rows must be 1 or 128, got " + std::to_string(block_rows));
  return TABBY_OK;
}

void fp8_sizes(int32_t rows, int32_t cols, int32_t block_rows, int64_t *code_bytes, int64_t *scale_bytes) {
  const int64_t col_panels = f8_parts(cols, kF8PanelCols), panels = f8_parts(rows, kF8PanelRows) * col_panels;
  *code_bytes = panels * kF8PanelBytes;
  // A multiple of 256 as well, so that arrays may lie one after another.
  *scale_bytes = block_rows == 1 ? panels * kF8PanelScales : f8_parts(f8_parts(rows, kF8Block) * col_panels * 4, 256) * 256;
}

int check_fp8_operand(const void *codes, const void *scales) {
  if (!codes || !scales) return record_failure(TABBY_EINVAL, "null pointer");
  if ((uintptr_t)codes % 16 != 0 || (uintptr_t)scales % 4 != 0)
    return record_failure(TABBY_EINVAL, "codes must be 16-byte aligned and scales 4-byte aligned");
  return TABBY_OK;
}

int check_fp8_apart(const RowSpan &rows, const void *codes, const void *scales, int32_t m_rows, int32_t m_cols, int32_t block_rows) {
  int64_t code_bytes, scale_bytes;
  fp8_sizes(m_rows, m_cols, block_rows, &code_bytes, &scale_bytes);
  if (rows_meet(rows, codes, code_bytes) || rows_meet(rows, scales, scale_bytes))
    return record_failure(TABBY_EINVAL, "what a call writes must not overlap what it reads");
  return TABBY_OK;
}

int fp8_quantize(const void *x, int32_t dtype, int32_t rows, int32_t cols, int64_t stride, int32_t block_rows, uint8_t *codes,
                 float *scales, hipStream_t s) {
  switch (dtype) {
    case TABBY_F32: return launch_quantize<TABBY_F32>(x, rows, cols, stride, block_rows, codes, scales, s);
    case TABBY_F16: return launch_quantize<TABBY_F16>(x, rows, cols, stride, block_rows, codes, scales, s);
    default: return launch_quantize<TABBY_BF16>(x, rows, cols, stride, block_rows, codes, scales, s);
  }
}

}  // namespace tabby

using namespace tabby;

extern "C" int tabby_fp8_bytes(int32_t rows, int32_t cols, int32_t block_rows, int64_t *code_bytes, int64_t *scale_bytes) {
  if (!code_bytes || !scale_bytes) return record_failure(TABBY_EINVAL, "null pointer");
  const int rc = check_fp8_shape(rows, cols, block_rows);
  if (rc) return rc;
  fp8_sizes(rows, cols, block_rows, code_bytes, scale_bytes);
  return TABBY_OK;
}

extern "C" int tabby_fp8_quantize_device(const void *x_dev, int32_t dtype, int32_t rows, int32_t cols, int64_t row_stride,
                                         int32_t block_rows, void *codes_dev, void *scales_dev, void *stream) {
  int rc = check_fp8_shape(rows, cols, block_rows);
  if (!rc) rc = check_rows(x_dev, dtype, rows, cols, row_stride, "x");
  if (!rc) rc = check_fp8_operand(codes_dev, scales_dev);
  if (rc) return rc;
  rc = check_fp8_apart(row_span(x_dev, rows, cols, row_stride, dtype_size(dtype)), codes_dev, scales_dev, rows, cols, block_rows);
  if (rc) return rc;
  return fp8_quantize(x_dev, dtype, rows, cols, row_stride, block_rows, (uint8_t *)codes_dev, (float *)scales_dev,
                      (hipStream_t)stream);
}

extern "C" int tabby_fp8_dequantize_device(const void *codes_dev, const void *scales_dev, int32_t rows, int32_t cols,
                                           int32_t block_rows, void *out_dev, int32_t dtype, int64_t row_stride, void *stream) {
  int rc = check_fp8_shape(rows, cols, block_rows);
  if (!rc) rc = check_rows(out_dev, dtype, rows, cols, row_stride, "out");
  if (!rc) rc = check_fp8_operand(codes_dev, scales_dev);
  if (rc) return rc;
  rc = check_fp8_apart(row_span(out_dev, rows, cols, row_stride, dtype_size(dtype)), codes_dev, scales_dev, rows, cols, block_rows);
  if (rc) return rc;
  const Fp8Matrix m{(const uint8_t *)codes_dev, (const float *)scales_dev, rows, cols};
  const hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case TABBY_F32: return launch_dequantize<TABBY_F32>(m, block_rows, out_dev, row_stride, s);
    case TABBY_F16: return launch_dequantize<TABBY_F16>(m, block_rows, out_dev, row_stride, s);
    default: return launch_dequantize<TABBY_BF16>(m, block_rows, out_dev, row_stride, s);
  }
}

extern "C" int tabby_fp8_pack_device(const void *row_codes_dev, const float *block_scales_dev, int32_t rows, int32_t cols,
                                     void *codes_dev, void *scales_dev, void *stream) {
  if (!row_codes_dev || !block_scales_dev) return record_failure(TABBY_EINVAL, "null pointer");
  int rc = check_fp8_shape(rows, cols, kF8Block);
  if (!rc) rc = check_fp8_operand(codes_dev, scales_dev);
  if (rc) return rc;
  if ((uintptr_t)block_scales_dev % 4 != 0) return record_failure(TABBY_EINVAL, "block_scales must be 4-byte aligned");
  const int64_t blocks = f8_parts(rows, kF8Block) * f8_parts(cols, kF8Block);
  rc = check_fp8_apart(row_span(row_codes_dev, 1, (int64_t)rows * cols, 0, 1), codes_dev, scales_dev, rows, cols, kF8Block);
  if (!rc) rc = check_fp8_apart(row_span(block_scales_dev, 1, blocks, 0, 4), codes_dev, scales_dev, rows, cols, kF8Block);
  if (rc) return rc;
  hipLaunchKernelGGL(fp8_pack_kernel, convert_grid(f8_parts(rows, kF8PanelRows) * f8_parts(cols, kF8PanelCols)), dim3(256), 0,
                     (hipStream_t)stream, (const uint8_t *)row_codes_dev, block_scales_dev, rows, cols, (uint8_t *)codes_dev,
                     (float *)scales_dev);
  TABBY_HIP_CHECK(hipGetLastError());
  return TABBY_OK;
}
