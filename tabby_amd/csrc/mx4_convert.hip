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

constexpr int kConvertBlock = 256;
constexpr unsigned kConvertGrid = 1u << 20;

// Both directions take a workgroup to a panel and are bound by HBM. Memory is read and written along the
// rows, 256 bytes (f16, bf16) or 512 at a time, 16 to a lane, and the codes change places in LDS, so that
// either side moves whole lines; a lane that held a block of its own would touch a line in four separate
// instructions. What is read or written once bypasses the caches, but not where rows start off 16 bytes, whose
// lines two loads or stores share. 151936 x 896 f16 there and back: 104 us (6.6 TB/s); cached, 142; a block to a lane, 193.
// 1531 x 4850 bf16, whose rows lie off 16 bytes: 14 us; a block to a lane, 63.
template <int DT>
struct PanelWalk {
  using E = Elem<DT>;
  static constexpr int kRowLanes = kMxPanelCols / E::kVec;               // lanes to a row
  static constexpr int kBlockLanes = kMxBlock / E::kVec;                 // lanes to a block
  static constexpr int kSteps = kMxPanelRows * kRowLanes / kConvertBlock;  // rows of a thread
  static constexpr int kRowStep = kConvertBlock / kRowLanes;
  int row, at;  // the first row; the place in it, in lanes
  __device__ __forceinline__ PanelWalk() : row((int)threadIdx.x / kRowLanes), at((int)threadIdx.x % kRowLanes) {}
  __device__ __forceinline__ int col() const { return at * E::kVec; }
  __device__ __forceinline__ int block() const { return at / kBlockLanes; }
  // Where a row's codes of this lane lie in the panel, and their block's scale.
  __device__ __forceinline__ int code_byte(int r) const {
    return (r >> 4) * kMxTileBytes + ((r & 15) + 16 * block()) * 16 + at % kBlockLanes * (E::kVec / 2);
  }
  __device__ __forceinline__ int scale_byte(int r) const { return 4 * ((r & 15) + 16 * block()) + (r >> 4); }
};

template <int DT, bool WHOLE>
__global__ __launch_bounds__(kConvertBlock) void mx4_quantize_kernel(const typename Elem<DT>::Bits *x, int rows, int cols,
                                                                     int64_t stride, uint8_t *codes, uint8_t *scales) {
  using E = Elem<DT>;
  using Walk = PanelWalk<DT>;
  __shared__ __align__(16) uint8_t panel_codes[kMxPanelBytes];
  __shared__ __align__(4) uint8_t panel_scales[kMxPanelScales];
  const Walk walk;
  const int64_t col_panels = mx_panels(cols, kMxPanelCols), panels = mx_panels(rows, kMxPanelRows) * col_panels;
  for (int64_t panel = blockIdx.x; panel < panels; panel += gridDim.x) {
    const int row0 = (int)(panel / col_panels) * kMxPanelRows, col0 = (int)(panel % col_panels) * kMxPanelCols;
    const int col = col0 + walk.col();
    u32x4 raw[Walk::kSteps];
#pragma unroll
    for (int i = 0; i < Walk::kSteps; ++i) {
      const int row = row0 + walk.row + i * Walk::kRowStep;
      raw[i] = row < rows ? load_values<DT, WHOLE>(x + (int64_t)row * stride, col, cols) : u32x4{0, 0, 0, 0};
    }
#pragma unroll
    for (int i = 0; i < Walk::kSteps; ++i) {
      const int r = walk.row + i * Walk::kRowStep;
      uint32_t word, s = encode_lane<DT>(raw[i], word);
      store_codes<E::kVec>(&panel_codes[walk.code_byte(r)], word);
      if (col0 + walk.block() * kMxBlock >= cols) s = kMxScaleOne;
      if (walk.at % Walk::kBlockLanes == 0) panel_scales[walk.scale_byte(r)] = (uint8_t)s;
    }
    __syncthreads();
    const int t = (int)threadIdx.x;
    reinterpret_cast<u32x4 *>(codes + panel * kMxPanelBytes)[t] = reinterpret_cast<const u32x4 *>(panel_codes)[t];
    if (t < kMxPanelScales / 4)
      reinterpret_cast<uint32_t *>(scales + panel * kMxPanelScales)[t] = reinterpret_cast<const uint32_t *>(panel_scales)[t];
    __syncthreads();
  }
}

template <int DT>
__global__ __launch_bounds__(kConvertBlock) void mx4_dequantize_kernel(Mx4Matrix m, typename Elem<DT>::Bits *out, int64_t stride,
                                                                       bool whole) {
  using E = Elem<DT>;
  using Walk = PanelWalk<DT>;
  __shared__ __align__(16) uint8_t panel_codes[kMxPanelBytes];
  __shared__ __align__(4) uint8_t panel_scales[kMxPanelScales];
  const Walk walk;
  const int64_t col_panels = m.col_panels(), panels = mx_panels(m.rows, kMxPanelRows) * col_panels;
  for (int64_t panel = blockIdx.x; panel < panels; panel += gridDim.x) {
    const int row0 = (int)(panel / col_panels) * kMxPanelRows, col0 = (int)(panel % col_panels) * kMxPanelCols;
    const int t = (int)threadIdx.x;
    reinterpret_cast<u32x4 *>(panel_codes)[t] = reinterpret_cast<const u32x4 *>(m.codes + panel * kMxPanelBytes)[t];
    if (t < kMxPanelScales / 4)
      reinterpret_cast<uint32_t *>(panel_scales)[t] = reinterpret_cast<const uint32_t *>(m.scales + panel * kMxPanelScales)[t];
    __syncthreads();
    const int col = col0 + walk.col();
#pragma unroll
    for (int i = 0; i < Walk::kSteps; ++i) {
      const int r = walk.row + i * Walk::kRowStep, row = row0 + r;
      if (row >= m.rows || col >= m.cols) continue;
      uint32_t word;
      if constexpr (E::kVec == 4) word = *reinterpret_cast<const uint16_t *>(&panel_codes[walk.code_byte(r)]);
      else word = *reinterpret_cast<const uint32_t *>(&panel_codes[walk.code_byte(r)]);
      const uint32_t s = panel_scales[walk.scale_byte(r)];
      float v[E::kVec];
      decode_values<E::kVec>(word, s, v);
      typename E::Bits *to = out + (int64_t)row * stride + col;
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

dim3 pack_grid(int rows, int cols) {
  const int64_t tiles = mx_panels(rows, kMxTileRows);
  return dim3((unsigned)mx_panels(mx_panels(cols, kMxPanelCols), 4), (unsigned)std::min<int64_t>(tiles, 65535));
}

dim3 convert_grid(int rows, int cols) {
  return dim3((unsigned)std::min<int64_t>(mx_panels(rows, kMxPanelRows) * mx_panels(cols, kMxPanelCols), kConvertGrid));
}

// Whether no two lanes share 16 bytes of memory.
template <int DT>
bool whole_rows(const void *rows, int64_t stride) {
  return (uintptr_t)rows % 16 == 0 && stride % Elem<DT>::kVec == 0;
}

template <int DT>
int launch_quantize(const void *x, int rows, int cols, int64_t stride, uint8_t *codes, uint8_t *scales, hipStream_t s) {
  const auto *from = (const typename Elem<DT>::Bits *)x;
  const dim3 grid = convert_grid(rows, cols);
  if (whole_rows<DT>(x, stride))
    hipLaunchKernelGGL((mx4_quantize_kernel<DT, true>), grid, dim3(kConvertBlock), 0, s, from, rows, cols, stride, codes, scales);
  else
    hipLaunchKernelGGL((mx4_quantize_kernel<DT, false>), grid, dim3(kConvertBlock), 0, s, from, rows, cols, stride, codes, scales);
  TABBY_HIP_CHECK(hipGetLastError());
  return TABBY_OK;
}

template <int DT>
int launch_dequantize(const Mx4Matrix &m, void *out, int64_t stride, hipStream_t s) {
  hipLaunchKernelGGL(mx4_dequantize_kernel<DT>, convert_grid(m.rows, m.cols), dim3(kConvertBlock), 0, s, m,
                     (typename Elem<DT>::Bits *)out, stride, whole_rows<DT>(out, stride));
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

int check_mx4_apart(const RowSpan &rows, const void *codes, const void *scales, int32_t m_rows, int32_t m_cols) {
  const int64_t panels = mx_panels(m_rows, kMxPanelRows) * mx_panels(m_cols, kMxPanelCols);
  if (rows_meet(rows, codes, panels * kMxPanelBytes) || rows_meet(rows, scales, panels * kMxPanelScales))
    return record_failure(TABBY_EINVAL, "what a call writes must not overlap what it reads");
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
  rc = check_mx4_apart(row_span(x_dev, rows, cols, row_stride, dtype_size(dtype)), codes_dev, scales_dev, rows, cols);
  if (rc) return rc;
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
  rc = check_mx4_apart(row_span(out_dev, rows, cols, row_stride, dtype_size(dtype)), codes_dev, scales_dev, rows, cols);
  if (rc) return rc;
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
  const int64_t blocks = mx_panels(cols, kMxBlock);
  rc = check_mx4_apart(row_span(row_codes_dev, 1, rows * blocks * (kMxBlock / 2), 0, 1), codes_dev, scales_dev, rows, cols);
  if (!rc) rc = check_mx4_apart(row_span(row_scales_dev, 1, rows * blocks, 0, 1), codes_dev, scales_dev, rows, cols);
  if (rc) return rc;
  hipLaunchKernelGGL(mx4_pack_kernel, pack_grid(rows, cols), dim3(kConvertBlock), 0, (hipStream_t)stream,
                     (const uint8_t *)row_codes_dev, (const uint8_t *)row_scales_dev, rows, cols, (uint8_t *)codes_dev,
                     (uint8_t *)scales_dev);
  TABBY_HIP_CHECK(hipGetLastError());
  return TABBY_OK;
}
