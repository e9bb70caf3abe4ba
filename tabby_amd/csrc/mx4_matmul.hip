// Y = X W^T (+ bias) with both operands in MXFP4 (mx4.h has the layout): rows x n, reduced over k.
//
// Each block of 32 products of a row of X and a row of W shares the power 2^(ex + ew), and the scaled
// matrix instruction (16 x 16 x 128, f32 accumulation) applies both exponents itself: a product of two
// codes is exact, so all rounding is the accumulation's. W's rows are the instruction's rows and X's its
// columns, so that a lane ends with four consecutive columns of Y.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <string>

#include "abi_internal.h"
#include "elem.h"
#include "mx4.h"

namespace tabby {
namespace {

typedef int32_t i32x8 __attribute__((ext_vector_type(8)));

// acc += the 16 x 16 product of one tile of each side; IW and IX pick the tiles' bytes of the scales.
template <int IW, int IX>
__device__ __forceinline__ f32x4 mx4_mfma(u32x4 w, u32x4 x, f32x4 acc, uint32_t sw, uint32_t sx) {
  const i32x8 a = {(int)w.x, (int)w.y, (int)w.z, (int)w.w, 0, 0, 0, 0};
  const i32x8 b = {(int)x.x, (int)x.y, (int)x.z, (int)x.w, 0, 0, 0, 0};
  constexpr int kFp4 = 4;
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, kFp4, kFp4, IW, (int)sw, IX, (int)sx);
}

struct Mx4Product {
  Mx4Matrix w, x;
  const float *bias;  // [n] or null
  void *out;
  int64_t out_stride;
};

// Four consecutive columns of one row of Y.
template <int DT>
__device__ __forceinline__ void store4(const Mx4Product &p, int row, int col, f32x4 v) {
  using E = Elem<DT>;
  using Bits = typename E::Bits;
  const int n = p.w.rows;
  if (row >= p.x.rows || col >= n) return;
  if (p.bias) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] += col + i < n ? p.bias[col + i] : 0.0f;
  }
  Bits *dst = (Bits *)p.out + (int64_t)row * p.out_stride + col;
  if (col + 4 <= n && (uintptr_t)dst % (4 * sizeof(Bits)) == 0) {
    typedef Bits vec4 __attribute__((ext_vector_type(4)));
    *reinterpret_cast<vec4 *>(dst) = vec4{E::narrow(v[0]), E::narrow(v[1]), E::narrow(v[2]), E::narrow(v[3])};
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (col + i < n) dst[i] = E::narrow(v[i]);
  }
}

// One wave to 64 columns and 16 rows of Y.
template <int DT>
__global__ __launch_bounds__(64) void mx4_panel_kernel(Mx4Product p) {
  const int lane = (int)threadIdx.x;
  const int kp = p.w.col_panels();
  const int64_t wp = (int64_t)blockIdx.x * kp;
  for (int tile = (int)blockIdx.y; tile * kMxTileRows < p.x.rows; tile += (int)gridDim.y) {
    const int64_t xp = (int64_t)(tile >> 2) * kp;
    f32x4 acc[4] = {};
    for (int k = 0; k < kp; ++k) {
      const uint8_t *wc = p.w.codes + (wp + k) * kMxPanelBytes + lane * 16;
      const uint8_t *xc = p.x.codes + (xp + k) * kMxPanelBytes + (tile & 3) * kMxTileBytes + lane * 16;
      const uint32_t sw = *reinterpret_cast<const uint32_t *>(p.w.scales + (wp + k) * kMxPanelScales + lane * 4);
      const uint32_t sx = *reinterpret_cast<const uint32_t *>(p.x.scales + (xp + k) * kMxPanelScales + lane * 4) >> (8 * (tile & 3));
      const u32x4 b = *reinterpret_cast<const u32x4 *>(xc);
      u32x4 a[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) a[t] = *reinterpret_cast<const u32x4 *>(wc + t * kMxTileBytes);
      acc[0] = mx4_mfma<0, 0>(a[0], b, acc[0], sw, sx);
      acc[1] = mx4_mfma<1, 0>(a[1], b, acc[1], sw, sx);
      acc[2] = mx4_mfma<2, 0>(a[2], b, acc[2], sw, sx);
      acc[3] = mx4_mfma<3, 0>(a[3], b, acc[3], sw, sx);
    }
#pragma unroll
    for (int t = 0; t < 4; ++t)
      store4<DT>(p, tile * kMxTileRows + (lane & 15), (int)blockIdx.x * kMxPanelRows + t * kMxTileRows + (lane >> 4) * 4, acc[t]);
  }
}

template <int DT>
int launch_product(const Mx4Product &p, hipStream_t s) {
  const int64_t tiles = mx_panels(p.x.rows, kMxTileRows);
  hipLaunchKernelGGL(mx4_panel_kernel<DT>, dim3((unsigned)mx_panels(p.w.rows, kMxPanelRows), (unsigned)std::min<int64_t>(tiles, 65535)),
                     dim3(64), 0, s, p);
  TABBY_HIP_CHECK(hipGetLastError());
  return TABBY_OK;
}

int product(const Mx4Product &p, int32_t out_dtype, hipStream_t s) {
  switch (out_dtype) {
    case TABBY_F32: return launch_product<TABBY_F32>(p, s);
    case TABBY_F16: return launch_product<TABBY_F16>(p, s);
    default: return launch_product<TABBY_BF16>(p, s);
  }
}

int check_output(const void *out, int32_t dtype, int32_t rows, int32_t n, int64_t stride) {
  if (!out) return record_failure(TABBY_EINVAL, "null pointer");
  if (!known_dtype(dtype)) return record_failure(TABBY_EINVAL, "dtype must be TABBY_F32, TABBY_F16 or TABBY_BF16");
  if (rows > 1 && stride < n) return record_failure(TABBY_EINVAL, "out_stride must be at least n");
  if ((uintptr_t)out % dtype_size(dtype) != 0) return record_failure(TABBY_EINVAL, "out must be aligned to its elements");
  return TABBY_OK;
}

}  // namespace
}  // namespace tabby

using namespace tabby;

extern "C" int tabby_mx4_matmul_device(const void *x_codes_dev, const void *x_scales_dev, int32_t rows,
                                       const void *w_codes_dev, const void *w_scales_dev, const float *bias_dev,
                                       int32_t n, int32_t k, void *out_dev, int32_t out_dtype, int64_t out_stride,
                                       void *stream) {
  int rc = check_mx4_operand(x_codes_dev, x_scales_dev);
  if (!rc) rc = check_mx4_operand(w_codes_dev, w_scales_dev);
  if (!rc) rc = check_mx4_shape(rows, k);
  if (!rc) rc = check_mx4_shape(n, k);
  if (!rc) rc = check_output(out_dev, out_dtype, rows, n, out_stride);
  if (rc) return rc;
  const Mx4Product p{{(const uint8_t *)w_codes_dev, (const uint8_t *)w_scales_dev, n, k},
                     {(const uint8_t *)x_codes_dev, (const uint8_t *)x_scales_dev, rows, k},
                     bias_dev, out_dev, out_stride};
  return product(p, out_dtype, (hipStream_t)stream);
}

extern "C" int tabby_mx4_linear_device(const void *x_dev, int32_t x_dtype, int64_t x_stride, int32_t rows,
                                       const void *w_codes_dev, const void *w_scales_dev, const float *bias_dev,
                                       int32_t n, int32_t k, void *out_dev, int32_t out_dtype, int64_t out_stride,
                                       void *workspace_dev, int64_t workspace_bytes, void *stream) {
  if (!x_dev || !workspace_dev) return record_failure(TABBY_EINVAL, "null pointer");
  int rc = check_mx4_operand(w_codes_dev, w_scales_dev);
  if (!rc) rc = check_mx4_shape(rows, k);
  if (!rc) rc = check_mx4_shape(n, k);
  if (!rc) rc = check_output(out_dev, out_dtype, rows, n, out_stride);
  if (rc) return rc;
  if (!known_dtype(x_dtype)) return record_failure(TABBY_EINVAL, "dtype must be TABBY_F32, TABBY_F16 or TABBY_BF16");
  if (rows > 1 && x_stride < k) return record_failure(TABBY_EINVAL, "x_stride must be at least k");
  if ((uintptr_t)x_dev % dtype_size(x_dtype) != 0) return record_failure(TABBY_EINVAL, "x must be aligned to its elements");
  int64_t code_bytes, scale_bytes;
  rc = tabby_mx4_bytes(rows, k, &code_bytes, &scale_bytes);
  if (rc) return rc;
  if ((uintptr_t)workspace_dev % 16 != 0 || workspace_bytes < code_bytes + scale_bytes)
    return record_failure(TABBY_EINVAL, "workspace must be 16-byte aligned and hold the quantised x (tabby_mx4_bytes)");
  uint8_t *codes = (uint8_t *)workspace_dev, *scales = codes + code_bytes;
  rc = mx4_quantize(x_dev, x_dtype, rows, k, x_stride, codes, scales, (hipStream_t)stream);
  if (rc) return rc;
  const Mx4Product p{{(const uint8_t *)w_codes_dev, (const uint8_t *)w_scales_dev, n, k},
                     {codes, scales, rows, k}, bias_dev, out_dev, out_stride};
  return product(p, out_dtype, (hipStream_t)stream);
}
