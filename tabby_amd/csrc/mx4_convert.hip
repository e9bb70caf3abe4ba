// MXFP4 conversions: a matrix to codes and scales (mx4.h has the layout), the way back, and the
// repacking of a checkpoint's row-major codes.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <string>

#include "abi_internal.h"
#include "elem.h"
#include "mx4.h"

namespace tabby {
namespace {

constexpr int kConvertBlock = 256;  // 16 rows x 16 blocks: one tile to a wave

template <int DT, bool VEC>
__global__ __launch_bounds__(kConvertBlock) void mx4_quantize_kernel(const typename Elem<DT>::Bits *x, int rows, int cols,
                                                                     int64_t stride, uint8_t *codes, uint8_t *scales) {
  const int col_panels = (cols + kMxPanelCols - 1) / kMxPanelCols;
  const int panel_col = (int)blockIdx.x * 4 + (int)(threadIdx.x >> 6);  // one tile to a wave
  if (panel_col >= col_panels) return;
  const int lane = (int)threadIdx.x & 63;
  for (int tile = (int)blockIdx.y; tile * kMxTileRows < rows; tile += (int)gridDim.y) {
    const int row = tile * kMxTileRows + (lane & 15);
    const int col = panel_col * kMxPanelCols + (lane >> 4) * kMxBlock;
    if (row >= rows) continue;
    float v[kMxBlock];
    load_block<DT, VEC>(x + (int64_t)row * stride, col, cols, v);
    u32x4 word;
    const uint32_t s = encode_block(v, word);
    const int64_t panel = (int64_t)(tile >> 2) * col_panels + panel_col;
    *reinterpret_cast<u32x4 *>(codes + panel * kMxPanelBytes + (tile & 3) * kMxTileBytes + lane * 16) = word;
    scales[panel * kMxPanelScales + lane * 4 + (tile & 3)] = (uint8_t)(col < cols ? s : kMxScaleOne);
  }
}

template <int DT, bool VEC>
__global__ __launch_bounds__(kConvertBlock) void mx4_dequantize_kernel(Mx4Matrix m, typename Elem<DT>::Bits *out,
                                                                       int64_t stride) {
  using E = Elem<DT>;
  const int col_panels = m.col_panels();
  const int panel_col = (int)blockIdx.x * 4 + (int)(threadIdx.x >> 6);
  if (panel_col >= col_panels) return;
  const int lane = (int)threadIdx.x & 63;
  for (int tile = (int)blockIdx.y; tile * kMxTileRows < m.rows; tile += (int)gridDim.y) {
    const int row = tile * kMxTileRows + (lane & 15);
    const int col = panel_col * kMxPanelCols + (lane >> 4) * kMxBlock;
    if (row >= m.rows || col >= m.cols) continue;
    const int64_t panel = (int64_t)(tile >> 2) * col_panels + panel_col;
    const u32x4 w = *reinterpret_cast<const u32x4 *>(m.codes + panel * kMxPanelBytes + (tile & 3) * kMxTileBytes + lane * 16);
    const uint32_t s = m.scales[panel * kMxPanelScales + lane * 4 + (tile & 3)];
    const float scale = s == kMxScaleNan ? __uint_as_float(0x7fc00000u) : __uint_as_float(s << 23);
    float v[kMxBlock];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const auto a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], scale, 0);
      const auto b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], scale, 1);
      const auto c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], scale, 2);
      const auto d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], scale, 3);
      v[8 * i] = a[0];
      v[8 * i + 1] = a[1];
      v[8 * i + 2] = b[0];
      v[8 * i + 3] = b[1];
      v[8 * i + 4] = c[0];
      v[8 * i + 5] = c[1];
      v[8 * i + 6] = d[0];
      v[8 * i + 7] = d[1];
    }
    if (s == kMxScaleNan) {
#pragma unroll
      for (int i = 0; i < kMxBlock; ++i) v[i] = scale;
    }
    typename E::Bits *dst = out + (int64_t)row * stride + col;
    if (VEC && col + kMxBlock <= m.cols) {
#pragma unroll
      for (int i = 0; i < kMxBlock; i += E::kVec) {
        u32x4 u;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if constexpr (E::kVec == 4) u[j] = E::narrow(v[i + j]);
          else u[j] = (uint32_t)E::narrow(v[i + 2 * j]) | ((uint32_t)E::narrow(v[i + 2 * j + 1]) << 16);
        }
        *reinterpret_cast<u32x4 *>(dst + i) = u;
      }
    } else {
#pragma unroll
      for (int i = 0; i < kMxBlock; ++i)
        if (col + i < m.cols) dst[i] = E::narrow(v[i]);
    }
  }
}

// A checkpoint's codes [rows][blocks * 16] and exponents [rows][blocks] to panels. What lies past the
// last column becomes code 0.
__global__ __launch_bounds__(kConvertBlock) void mx4_pack_kernel(const uint8_t *src, const uint8_t *src_scales, int rows,
                                                                 int cols, uint8_t *codes, uint8_t *scales) {
  const int col_panels = (cols + kMxPanelCols - 1) / kMxPanelCols;
  const int blocks = (cols + kMxBlock - 1) / kMxBlock;
  const int panel_col = (int)blockIdx.x * 4 + (int)(threadIdx.x >> 6);
  if (panel_col >= col_panels) return;
  const int lane = (int)threadIdx.x & 63;
  for (int tile = (int)blockIdx.y; tile * kMxTileRows < rows; tile += (int)gridDim.y) {
    const int row = tile * kMxTileRows + (lane & 15);
    const int block = panel_col * (kMxPanelCols / kMxBlock) + (lane >> 4);
    if (row >= rows) continue;
    u32x4 w = {0, 0, 0, 0};
    uint32_t s = kMxScaleOne;
    if (block < blocks) {
      const uint8_t *from = src + ((int64_t)row * blocks + block) * 16;
      s = src_scales[(int64_t)row * blocks + block];
      if ((uintptr_t)src % 16 == 0) {
        w = *reinterpret_cast<const u32x4 *>(from);
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) w[i / 4] |= (uint32_t)from[i] << (8 * (i % 4));
      }
      const int left = cols - block * kMxBlock;  // columns of this block that exist
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int n = left - 8 * i;
        if (n < 8) w[i] &= n <= 0 ? 0u : (1u << (4 * n)) - 1u;
      }
    }
    const int64_t panel = (int64_t)(tile >> 2) * col_panels + panel_col;
    *reinterpret_cast<u32x4 *>(codes + panel * kMxPanelBytes + (tile & 3) * kMxTileBytes + lane * 16) = w;
    scales[panel * kMxPanelScales + lane * 4 + (tile & 3)] = (uint8_t)s;
  }
}

dim3 convert_grid(int rows, int cols) {
  const int64_t tiles = mx_panels(rows, kMxTileRows);
  return dim3((unsigned)mx_panels(mx_panels(cols, kMxPanelCols), 4), (unsigned)std::min<int64_t>(tiles, 65535));
}

template <int DT>
int launch_quantize(const void *x, int rows, int cols, int64_t stride, uint8_t *codes, uint8_t *scales, hipStream_t s) {
  using E = Elem<DT>;
  const auto *src = (const typename E::Bits *)x;
  const bool vec = (uintptr_t)x % 16 == 0 && stride % E::kVec == 0;
  const dim3 grid = convert_grid(rows, cols);
  if (vec)
    hipLaunchKernelGGL((mx4_quantize_kernel<DT, true>), grid, dim3(kConvertBlock), 0, s, src, rows, cols, stride, codes, scales);
  else
    hipLaunchKernelGGL((mx4_quantize_kernel<DT, false>), grid, dim3(kConvertBlock), 0, s, src, rows, cols, stride, codes, scales);
  TABBY_HIP_CHECK(hipGetLastError());
  return TABBY_OK;
}

template <int DT>
int launch_dequantize(const Mx4Matrix &m, void *out, int64_t stride, hipStream_t s) {
  using E = Elem<DT>;
  auto *dst = (typename E::Bits *)out;
  const bool vec = (uintptr_t)out % 16 == 0 && stride % E::kVec == 0;
  const dim3 grid = convert_grid(m.rows, m.cols);
  if (vec) hipLaunchKernelGGL((mx4_dequantize_kernel<DT, true>), grid, dim3(kConvertBlock), 0, s, m, dst, stride);
  else hipLaunchKernelGGL((mx4_dequantize_kernel<DT, false>), grid, dim3(kConvertBlock), 0, s, m, dst, stride);
  TABBY_HIP_CHECK(hipGetLastError());
  return TABBY_OK;
}

}  // namespace

int check_mx4_shape(int32_t rows, int32_t cols) {
  if (rows < 1 || cols < 1) return record_failure(TABBY_EINVAL, "rows and cols must be >= 1");
  if (cols > INT32_MAX - kMxPanelCols || rows > INT32_MAX - kMxPanelRows)
    return record_failure(TABBY_EINVAL, "rows and cols must leave room for their padding in 32 bits");
  return TABBY_OK;
}

int check_mx4_operand(const void *codes, const void *scales) {
  if (!codes || !scales) return record_failure(TABBY_EINVAL, "null pointer");
  if ((uintptr_t)codes % 16 != 0 || (uintptr_t)scales % 4 != 0)
    return record_failure(TABBY_EINVAL, "codes must be 16-byte aligned and scales 4-byte aligned");
  return TABBY_OK;
}

int mx4_quantize(const void *x, int32_t dtype, int32_t rows, int32_t cols, int64_t stride, uint8_t *codes,
                 uint8_t *scales, hipStream_t s) {
  switch (dtype) {
    case TABBY_F32: return launch_quantize<TABBY_F32>(x, rows, cols, stride, codes, scales, s);
    case TABBY_F16: return launch_quantize<TABBY_F16>(x, rows, cols, stride, codes, scales, s);
    default: return launch_quantize<TABBY_BF16>(x, rows, cols, stride, codes, scales, s);
  }
}

}  // namespace tabby

using namespace tabby;

extern "C" int tabby_mx4_bytes(int32_t rows, int32_t cols, int64_t *code_bytes, int64_t *scale_bytes) {
  if (!code_bytes || !scale_bytes) return record_failure(TABBY_EINVAL, "null pointer");
  const int rc = check_mx4_shape(rows, cols);
  if (rc) return rc;
  const int64_t panels = mx_panels(rows, kMxPanelRows) * mx_panels(cols, kMxPanelCols);
  *code_bytes = panels * kMxPanelBytes;
  *scale_bytes = panels * kMxPanelScales;
  return TABBY_OK;
}

extern "C" int tabby_mx4_quantize_device(const void *x_dev, int32_t dtype, int32_t rows, int32_t cols,
                                         int64_t row_stride, void *codes_dev, void *scales_dev, void *stream) {
  if (!x_dev) return record_failure(TABBY_EINVAL, "null pointer");
  int rc = check_mx4_operand(codes_dev, scales_dev);
  if (rc) return rc;
  rc = check_mx4_shape(rows, cols);
  if (rc) return rc;
  if (!known_dtype(dtype)) return record_failure(TABBY_EINVAL, "dtype must be TABBY_F32, TABBY_F16 or TABBY_BF16");
  if (rows > 1 && row_stride < cols) return record_failure(TABBY_EINVAL, "row_stride must be at least cols");
  if ((uintptr_t)x_dev % dtype_size(dtype) != 0) return record_failure(TABBY_EINVAL, "x must be aligned to its elements");
  return mx4_quantize(x_dev, dtype, rows, cols, row_stride, (uint8_t *)codes_dev, (uint8_t *)scales_dev,
                      (hipStream_t)stream);
}

extern "C" int tabby_mx4_dequantize_device(const void *codes_dev, const void *scales_dev, int32_t rows, int32_t cols,
                                           void *out_dev, int32_t dtype, int64_t row_stride, void *stream) {
  if (!out_dev) return record_failure(TABBY_EINVAL, "null pointer");
  int rc = check_mx4_operand(codes_dev, scales_dev);
  if (rc) return rc;
  rc = check_mx4_shape(rows, cols);
  if (rc) return rc;
  if (!known_dtype(dtype)) return record_failure(TABBY_EINVAL, "dtype must be TABBY_F32, TABBY_F16 or TABBY_BF16");
  if (rows > 1 && row_stride < cols) return record_failure(TABBY_EINVAL, "row_stride must be at least cols");
  if ((uintptr_t)out_dev % dtype_size(dtype) != 0) return record_failure(TABBY_EINVAL, "out must be aligned to its elements");
  const Mx4Matrix m{(const uint8_t *)codes_dev, (const uint8_t *)scales_dev, rows, cols};
  const hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case TABBY_F32: return launch_dequantize<TABBY_F32>(m, out_dev, row_stride, s);
    case TABBY_F16: return launch_dequantize<TABBY_F16>(m, out_dev, row_stride, s);
    default: return launch_dequantize<TABBY_BF16>(m, out_dev, row_stride, s);
  }
}

extern "C" int tabby_mx4_pack_device(const void *row_codes_dev, const void *row_scales_dev, int32_t rows, int32_t cols,
                                     void *codes_dev, void *scales_dev, void *stream) {
  if (!row_codes_dev || !row_scales_dev) return record_failure(TABBY_EINVAL, "null pointer");
  int rc = check_mx4_operand(codes_dev, scales_dev);
  if (rc) return rc;
  rc = check_mx4_shape(rows, cols);
  if (rc) return rc;
  hipLaunchKernelGGL(mx4_pack_kernel, convert_grid(rows, cols), dim3(kConvertBlock), 0, (hipStream_t)stream,
                     (const uint8_t *)row_codes_dev, (const uint8_t *)row_scales_dev, rows, cols, (uint8_t *)codes_dev,
                     (uint8_t *)scales_dev);
  TABBY_HIP_CHECK(hipGetLastError());
  return TABBY_OK;
}
