// Y = X W^T (+ bias) with both operands in FP8 (fp8.h has the layout): rows x n, reduced over k.
//
//   y[m, n] = sum over blocks b of k of  sx[m, b] * sw[n / 128, b] * sum over the block of x w
//
// The inner sum, 128 products of codes, comes from the matrix cores, started from zero; the vector units scale it and add
// it up in f32, so scales may be any f32. W's rows are the instruction's rows and X's its columns, so that a lane
// ends with four consecutive columns of Y, of one row: one scale to its four results.
//
// Two ways to the inner sum. Codes converted to f16, where all of them are exact, and four 16 x 16 x 32 f16
// instructions: their products are exact and their sums f32's (measured: within 2^-22 of the sum of the magnitudes).
// Or one 16 x 16 x 128 instruction on the codes themselves, at twice the rate, which adds eight products at a time and
// keeps of each what lies above 2^-14 or so of the group's largest (measured: 1.5e-5 of the result's norm for normal
// values, 5e-5 for codes drawn alike). The first is taken where the result is f32, and wherever memory and not the
// matrix cores are the bound; the second where many rows go to f16 or bf16, whose own rounding, 1.4e-4 and
// 1.1e-3 of the norm, is far larger.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <string>
#include <type_traits>

#include "abi_internal.h"
#include "elem.h"
#include "fp8.h"
#include "product_ops.h"
#include "wave_ops.h"

namespace tabby {
namespace {

typedef int32_t i32x8 __attribute__((ext_vector_type(8)));

// A tile's codes of a lane: both halves.
struct TileCodes { u32x4 half[2]; };

__device__ __forceinline__ TileCodes read_tile(const uint8_t *at) {
  return {{*reinterpret_cast<const u32x4 *>(at), *reinterpret_cast<const u32x4 *>(at + kF8TileBytes / 2)}};
}

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// A tile as the f16 instructions take it, or as it is.
struct HalfOperand {
  f16x8 part[4];
  __device__ __forceinline__ HalfOperand() {}
  __device__ __forceinline__ explicit HalfOperand(const TileCodes &t) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t word = t.half[i / 4][i % 4];
      const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word, 1.0f, false);
      const f16x2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word, 1.0f, true);
      part[i / 2][4 * (i % 2)] = a[0];
      part[i / 2][4 * (i % 2) + 1] = a[1];
      part[i / 2][4 * (i % 2) + 2] = b[0];
      part[i / 2][4 * (i % 2) + 3] = b[1];
    }
  }
};
struct CodeOperand {
  i32x8 codes;
  __device__ __forceinline__ CodeOperand() {}
  __device__ __forceinline__ explicit CodeOperand(const TileCodes &t) {
#pragma unroll
    for (int i = 0; i < 8; ++i) codes[i] = (int)t.half[i / 4][i % 4];
  }
};

// The 16 x 16 product of one tile of each side.
__device__ __forceinline__ f32x4 tile_product(const HalfOperand &w, const HalfOperand &x) {
  f32x4 t = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i) t = __builtin_amdgcn_mfma_f32_16x16x32_f16(w.part[i], x.part[i], t, 0, 0, 0);
  return t;
}
__device__ __forceinline__ f32x4 tile_product(const CodeOperand &w, const CodeOperand &x) {
  constexpr int kE4m3 = 0;
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w.codes, x.codes, f32x4{0, 0, 0, 0}, kE4m3, kE4m3, 0, 0, 0, 0);
}

__device__ __forceinline__ void add_scaled(f32x4 &acc, f32x4 t, float s) {
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i] = __builtin_fmaf(t[i], s, acc[i]);
}

struct Fp8Product {
  Fp8Matrix w, x;  // square blocks; blocks of one row
  ProductOut y;
};

// A workgroup of WM x WN waves has a tile of WM PM x WN PN panels of Y (64 x 64), PM x PN to a wave, and takes a
// panel of k (128) at a time. The panels of a stage lie in LDS as they do in memory, W's before X's, then X's scales,
// brought there without passing through registers, a stage ahead. A wave holds the tiles of X and goes through those
// of W; a tile's results are added while the next one's products run.
template <int PM, int PN, int WM, int WN>
struct TileShape {
  static constexpr int kWaves = WM * WN;
  static constexpr int kPanels = WM * PM + WN * PN;
  static constexpr int kCodes = kPanels * kF8PanelBytes;  // of a stage
  static constexpr int kStage = kCodes + WN * PN * kF8PanelScales;
  static constexpr int kStages = 2;
  static constexpr int kTiles = 4 * kPanels / kWaves;  // tiles that a wave brings to a stage
  static_assert(4 * kPanels % kWaves == 0, "every wave brings as much");
  static_assert(PM <= 2, "a wave's panels of W lie in one square block");
  static constexpr int kLoads = 2 * kTiles + 1;
};

__device__ __forceinline__ void bring_tile(const uint8_t *from, uint8_t *to) {
  static_assert(kF8TileBytes == 2048, "the literal below");
  __builtin_amdgcn_global_load_lds((GlobalVoid *)from, (LdsVoid *)to, 16, 0, 0);
  __builtin_amdgcn_global_load_lds((GlobalVoid *)from, (LdsVoid *)to, 16, 1024, 0);
}
__device__ __forceinline__ void bring_scales(const uint8_t *from, uint8_t *to) {
  __builtin_amdgcn_global_load_lds((GlobalVoid *)from, (LdsVoid *)to, 4, 0, 0);
}

template <int DT, int PM, int PN, int WM, int WN>
__global__ __launch_bounds__(WM *WN * 64, 2) void fp8_tile_kernel(Fp8Product p, int tiles_w, int tiles_x) {
  using S = TileShape<PM, PN, WM, WN>;
  using Operand = typename std::conditional<DT == TABBY_F32, HalfOperand, CodeOperand>::type;
  __shared__ __align__(1024) uint8_t lds[S::kStages][S::kStage];
  const int lane = (int)threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int wm = wave % WM, wn = wave / WM;
  const int kp = p.w.col_panels();
  const TilePlace place = tile_place((int)blockIdx.x, tiles_w, tiles_x);

  // Panels past the last are the last again; what they give is not stored.
  const int w_panels = (int)f8_parts(p.w.rows, kF8PanelRows), x_panels = (int)f8_parts(p.x.rows, kF8PanelRows);
  auto panel_at = [&](int panel) {
    return panel < WM * PM ? (int64_t)min(place.w * WM * PM + panel, w_panels - 1) * kp
                           : (int64_t)min(place.x * WN * PN + panel - WM * PM, x_panels - 1) * kp;
  };
  const uint8_t *codes[S::kTiles];
#pragma unroll
  for (int h = 0; h < S::kTiles; ++h) {
    const int tile = wave * S::kTiles + h, panel = tile >> 2;
    codes[h] = (panel < WM * PM ? p.w.codes : p.x.codes) + panel_at(panel) * kF8PanelBytes + (tile & 3) * kF8TileBytes + lane * 16;
  }
  const int scales_of = wave % (WN * PN);  // twice or more where there are more waves
  const uint8_t *x_scales = (const uint8_t *)p.x.scales + panel_at(WM * PM + scales_of) * kF8PanelScales + lane * 4;
  int brought = 0;
  auto bring = [&](uint8_t *stage) {
    // Past the last panel of k it is the last one again, which nothing reads: every stage has as many loads.
    const int step = ++brought < kp ? 1 : 0;
#pragma unroll
    for (int h = 0; h < S::kTiles; ++h) {
      bring_tile(codes[h], stage + (wave * S::kTiles + h) * kF8TileBytes);
      codes[h] += step * kF8PanelBytes;
    }
    bring_scales(x_scales, stage + S::kCodes + scales_of * kF8PanelScales);
    x_scales += step * kF8PanelScales;
  };
  // The wave's panels of W lie in one square block.
  const float *w_scales = p.w.scales + (int64_t)(min((place.w * WM + wm) * PM, w_panels - 1) >> 1) * kp;

  constexpr int kW = PM * 4, kX = PN * 4;  // tiles of a wave
  f32x4 acc[kW][kX] = {};
  const int w_from = wm * PM * kF8PanelBytes + lane * 16, x_from = (WM * PM + wn * PN) * kF8PanelBytes + lane * 16;
  const int sx_from = S::kCodes + wn * PN * kF8PanelScales + (lane & 15) * 4;
  bring(lds[0]);
  int now = 0;
  for (int k = 0; k < kp; ++k) {
    wait_and_meet<0>();
    const uint8_t *stage = lds[now];
    now ^= 1;
    bring(lds[now]);
    const float sw = w_scales[k];
    Operand x[kX];
    TileCodes w[2];
    float s[kX];
    w[0] = read_tile(stage + w_from);
#pragma unroll
    for (int c = 0; c < kX; ++c) {
      x[c] = Operand(read_tile(stage + x_from + c * kF8TileBytes));
      s[c] = *reinterpret_cast<const float *>(stage + sx_from + c * 64) * sw;
    }
    f32x4 t[2][kX];
#pragma unroll
    for (int r = 0; r < kW; ++r) {
      if (r + 1 < kW) w[(r + 1) & 1] = read_tile(stage + w_from + (r + 1) * kF8TileBytes);
      const Operand of_w(w[r & 1]);
#pragma unroll
      for (int c = 0; c < kX; ++c) t[r & 1][c] = tile_product(of_w, x[c]);
      if (r > 0) {
#pragma unroll
        for (int c = 0; c < kX; ++c) add_scaled(acc[r - 1][c], t[(r - 1) & 1][c], s[c]);
      }
    }
#pragma unroll
    for (int c = 0; c < kX; ++c) add_scaled(acc[kW - 1][c], t[(kW - 1) & 1][c], s[c]);
  }
  wait_and_meet<0>();
#pragma unroll
  for (int i = 0; i < PM; ++i) {
#pragma unroll
    for (int j = 0; j < kX; ++j) {
      const int row = (place.x * WN + wn) * PN * kF8PanelRows + j * kF8TileRows + (lane & 15);
      const int col = ((place.w * WM + wm) * PM + i) * kF8PanelRows;
      store_panel<DT>(p.y, row, col, acc[i * 4][j], acc[i * 4 + 1][j], acc[i * 4 + 2][j], acc[i * 4 + 3][j]);
    }
  }
}

// Few rows: W is streamed from memory straight into registers, a wave to a panel of 64 columns of Y and
// NT tiles of 16 rows; where there are few panels, `slices` waves of the workgroup take a part of k each and add up
// through LDS.
struct FewShape {
  int waves, slices;  // of a workgroup; powers of two
};
constexpr int kSlicesMax = 8;
constexpr int kSumsMax = 16;  // slices * NT
// The upper half of the slices' sums lie in LDS, 4 KB to a wave's tile of rows.
__host__ __device__ constexpr int sums_bytes(int waves, int tiles) { return waves / 2 * tiles * 4096; }

template <int DT, int NT>
__global__ __launch_bounds__(kSlicesMax * 64) void fp8_few_kernel(Fp8Product p, FewShape shape) {
  __shared__ __align__(16) uint8_t lds[std::max(sums_bytes(4, NT), sums_bytes(std::min(kSlicesMax, kSumsMax / NT), NT))];
  const int lane = (int)threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int slice = wave & (shape.slices - 1);
  const int panel = (int)blockIdx.x * (shape.waves / shape.slices) + wave / shape.slices;
  const int kp = p.w.col_panels();
  const int tile = (int)blockIdx.y * NT;
  f32x4 acc[4][NT] = {};
  struct Step {
    TileCodes w[4], x[NT];
    float sx[NT], sw;
  };
  // A wave past the last panel has nothing to do but to meet the others.
  const bool works = panel * kF8PanelRows < p.w.rows;
  const uint8_t *wc = p.w.codes + (int64_t)panel * kp * kF8PanelBytes + lane * 16;
  const float *ws = p.w.scales + (int64_t)(panel >> 1) * kp;
  // NT tiles from `tile` on lie in one panel.
  const int64_t x_panel = (int64_t)(tile >> 2) * kp;
  const uint8_t *xc = p.x.codes + x_panel * kF8PanelBytes + (tile & 3) * kF8TileBytes + lane * 16;
  const float *xs = p.x.scales + x_panel * kF8PanelRows + (tile & 3) * kF8TileRows + (lane & 15);
  int k = (int)((int64_t)kp * slice / shape.slices);
  const int end = works ? (int)((int64_t)kp * (slice + 1) / shape.slices) : k;
  auto load = [&](int at, Step &s) {
#pragma unroll
    for (int t = 0; t < 4; ++t) s.w[t] = read_tile(wc + (int64_t)at * kF8PanelBytes + t * kF8TileBytes);
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      s.x[u] = read_tile(xc + (int64_t)at * kF8PanelBytes + u * kF8TileBytes);
      s.sx[u] = xs[(int64_t)at * kF8PanelRows + u * kF8TileRows];
    }
    s.sw = ws[at];
  };
  auto multiply = [&](const Step &s) {
    HalfOperand x[NT];
    float both[NT];
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      x[u] = HalfOperand(s.x[u]);
      both[u] = s.sx[u] * s.sw;
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const HalfOperand w(s.w[t]);
#pragma unroll
      for (int u = 0; u < NT; ++u) add_scaled(acc[t][u], tile_product(w, x[u]), both[u]);
    }
  };
  Step now, next;
  if (k < end) load(k, now);
  for (; k + 1 < end; ++k) {
    load(k + 1, next);
    multiply(now);
    now = next;
  }
  if (k < end) multiply(now);
  // The slices in halves: the upper half's sums go through LDS to the lower half's waves.
  f32x4 *const sums = reinterpret_cast<f32x4 *>(lds) + lane;
  for (int half = shape.slices / 2; half > 0; half /= 2) {
    const int at = (wave / shape.slices * half + (slice & (half - 1))) * NT * 4;
    if (slice >= half && slice < 2 * half) {
#pragma unroll
      for (int i = 0; i < 4 * NT; ++i) sums[(at + i) * 64] = acc[i / NT][i % NT];
    }
    __syncthreads();
    if (slice < half) {
#pragma unroll
      for (int i = 0; i < 4 * NT; ++i) acc[i / NT][i % NT] += sums[(at + i) * 64];
    }
    __syncthreads();
  }
  if (!works || slice != 0) return;
#pragma unroll
  for (int u = 0; u < NT; ++u)
    store_panel<DT>(p.y, (tile + u) * kF8TileRows + (lane & 15), panel * kF8PanelRows, acc[0][u], acc[1][u], acc[2][u], acc[3][u]);
}

constexpr int kCus = 256;               // an MI355X's compute units
constexpr int64_t kTilesMax = 1 << 22;  // of a launch: 2^32 threads are too many

// Whether W is streamed into registers: up to 64 rows, which one wave takes, and where tiles of 128 x 128
// would leave half the units idle.
bool few_rows(int n, int rows) {
  return rows <= kF8PanelRows || f8_parts(n, 128) * f8_parts(rows, 128) <= kCus / 2;
}

template <int DT, int PM, int PN, int WM, int WN>
int launch_tiles(const Fp8Product &p, hipStream_t s) {
  const int64_t tiles_w = f8_parts(p.w.rows, kF8PanelRows * PM * WM), tiles_x = f8_parts(p.x.rows, kF8PanelRows * PN * WN);
  if (tiles_w * tiles_x > kTilesMax) return record_failure(TABBY_EINVAL, "the product is too large for one launch");
  hipLaunchKernelGGL((fp8_tile_kernel<DT, PM, PN, WM, WN>), dim3((unsigned)(tiles_w * tiles_x)), dim3(WM * WN * 64), 0, s, p,
                     (int)tiles_w, (int)tiles_x);
  TABBY_HIP_CHECK(hipGetLastError());
  return TABBY_OK;
}

// Whether tiles of 256 x 256 are the better choice, else 128 x 128: a last round of them that few units take part in
// costs as much as a full one.
bool large_tiles(int n, int rows) {
  const int64_t large = f8_parts(n, 256) * f8_parts(rows, 256), small = f8_parts(n, 128) * f8_parts(rows, 128);
  return 7 * f8_parts(large, kCus) <= 2 * f8_parts(small, kCus);
}

template <int DT, int NT>
int launch_few(const Fp8Product &p, hipStream_t s) {
  const int64_t panels = f8_parts(p.w.rows, kF8PanelRows), groups = f8_parts(p.x.rows, kF8TileRows * NT);
  // Enough waves to fill the chip, eight to a unit, while every one has a panel of k.
  int slices = 1;
  while (slices < kSlicesMax && slices * 2 <= p.w.col_panels() && slices * 2 * NT <= kSumsMax && panels * groups * slices < 8 * kCus) slices *= 2;
  const FewShape shape{std::max(slices, 4), slices};
  const int64_t blocks = f8_parts(panels, shape.waves / shape.slices);
  hipLaunchKernelGGL((fp8_few_kernel<DT, NT>), dim3((unsigned)blocks, (unsigned)groups), dim3(64 * shape.waves), 0, s, p, shape);
  TABBY_HIP_CHECK(hipGetLastError());
  return TABBY_OK;
}

template <int DT>
int launch_product(const Fp8Product &p, hipStream_t s) {
  if (!few_rows(p.w.rows, p.x.rows)) return large_tiles(p.w.rows, p.x.rows) ? launch_tiles<DT, 2, 1, 2, 4>(p, s) : launch_tiles<DT, 1, 1, 2, 2>(p, s);
  switch (f8_parts(p.x.rows, kF8TileRows)) {
    case 1: return launch_few<DT, 1>(p, s);
    case 2: return launch_few<DT, 2>(p, s);
    default: return launch_few<DT, 4>(p, s);
  }
}

int product(const Fp8Product &p, int32_t out_dtype, hipStream_t s) {
  switch (out_dtype) {
    case TABBY_F32: return launch_product<TABBY_F32>(p, s);
    case TABBY_F16: return launch_product<TABBY_F16>(p, s);
    default: return launch_product<TABBY_BF16>(p, s);
  }
}

// The rows apart from the weights and the bias.
int check_apart(const RowSpan &rows, const Fp8Product &p) {
  const int rc = check_fp8_apart(rows, p.w.codes, p.w.scales, p.w.rows, p.w.cols, kF8Block);
  if (rc) return rc;
  if (p.y.bias && rows_meet(rows, p.y.bias, (int64_t)p.w.rows * (int64_t)sizeof(float)))
    return record_failure(TABBY_EINVAL, "what a call writes must not overlap its bias");
  return TABBY_OK;
}

int check_bias(const float *bias) {
  if ((uintptr_t)bias % 4 != 0) return record_failure(TABBY_EINVAL, "bias must be aligned to its elements");
  return TABBY_OK;
}

}  // namespace
}  // namespace tabby

using namespace tabby;

extern "C" int tabby_fp8_matmul_device(const void *x_codes_dev, const void *x_scales_dev, int32_t rows,
                                       const void *w_codes_dev, const void *w_scales_dev, const float *bias_dev,
                                       int32_t n, int32_t k, void *out_dev, int32_t out_dtype, int64_t out_stride,
                                       void *stream) {
  int rc = check_fp8_operand(x_codes_dev, x_scales_dev);
  if (!rc) rc = check_fp8_operand(w_codes_dev, w_scales_dev);
  if (!rc) rc = check_fp8_shape(rows, k, 1);
  if (!rc) rc = check_fp8_shape(n, k, kF8Block);
  if (!rc) rc = check_output(out_dev, out_dtype, rows, n, out_stride);
  if (!rc) rc = check_bias(bias_dev);
  if (rc) return rc;
  const Fp8Product p{{(const uint8_t *)w_codes_dev, (const float *)w_scales_dev, n, k},
                     {(const uint8_t *)x_codes_dev, (const float *)x_scales_dev, rows, k},
                     {rows, n, bias_dev, out_dev, out_stride}};
  const RowSpan out = row_span(out_dev, rows, n, out_stride, dtype_size(out_dtype));
  rc = check_apart(out, p);
  if (!rc) rc = check_fp8_apart(out, x_codes_dev, x_scales_dev, rows, k, 1);
  if (rc) return rc;
  return product(p, out_dtype, (hipStream_t)stream);
}

extern "C" int tabby_fp8_linear_device(const void *x_dev, int32_t x_dtype, int64_t x_stride, int32_t rows,
                                       const void *w_codes_dev, const void *w_scales_dev, const float *bias_dev,
                                       int32_t n, int32_t k, void *out_dev, int32_t out_dtype, int64_t out_stride,
                                       void *workspace_dev, int64_t workspace_bytes, void *stream) {
  if (!x_dev || !workspace_dev) return record_failure(TABBY_EINVAL, "null pointer");
  int rc = check_fp8_operand(w_codes_dev, w_scales_dev);
  if (!rc) rc = check_fp8_shape(rows, k, 1);
  if (!rc) rc = check_fp8_shape(n, k, kF8Block);
  if (!rc) rc = check_output(out_dev, out_dtype, rows, n, out_stride);
  if (!rc) rc = check_bias(bias_dev);
  if (rc) return rc;
  if (!known_dtype(x_dtype)) return record_failure(TABBY_EINVAL, "dtype must be TABBY_F32, TABBY_F16 or TABBY_BF16");
  if (rows > 1 && x_stride < k) return record_failure(TABBY_EINVAL, "x_stride must be at least k");
  if ((uintptr_t)x_dev % dtype_size(x_dtype) != 0) return record_failure(TABBY_EINVAL, "x must be aligned to its elements");
  int64_t code_bytes, scale_bytes;
  fp8_sizes(rows, k, 1, &code_bytes, &scale_bytes);
  const int64_t need = code_bytes + scale_bytes;
  if ((uintptr_t)workspace_dev % 16 != 0 || workspace_bytes < need)
    return record_failure(TABBY_EINVAL, "workspace must be 16-byte aligned and hold the quantised x (tabby_fp8_bytes)");
  uint8_t *codes = (uint8_t *)workspace_dev;
  float *scales = (float *)(codes + code_bytes);
  const Fp8Product p{{(const uint8_t *)w_codes_dev, (const float *)w_scales_dev, n, k},
                     {codes, scales, rows, k}, {rows, n, bias_dev, out_dev, out_stride}};
  const RowSpan x = row_span(x_dev, rows, k, x_stride, dtype_size(x_dtype));
  const RowSpan out = row_span(out_dev, rows, n, out_stride, dtype_size(out_dtype));
  rc = check_apart(out, p);
  if (!rc) rc = check_apart(row_span(workspace_dev, 1, need, 0, 1), p);
  if (rc) return rc;
  if (rows_meet(out, workspace_dev, need) || rows_meet(x, workspace_dev, need))
    return record_failure(TABBY_EINVAL, "workspace must not overlap x or out");
  rc = fp8_quantize(x_dev, x_dtype, rows, k, x_stride, 1, codes, scales, (hipStream_t)stream);
  if (rc) return rc;
  return product(p, out_dtype, (hipStream_t)stream);
}
