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

// Exchanges a's upper half of the wave with b's lower half, and a's odd quarters with b's even ones.
__device__ __forceinline__ void swap_halves(uint32_t &a, uint32_t &b) {
  const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
  a = r[0];
  b = r[1];
}
__device__ __forceinline__ void swap_quarters(uint32_t &a, uint32_t &b) {
  const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
  a = r[0];
  b = r[1];
}

// A lane's 4 x 4 columns of one row of Y: tile t has columns col + 16 t + 4 q on, q the lane's quarter of
// the wave. Inside the matrix the quarters exchange them, so that each stores 16 columns in a row: four
// lanes fill whole lines, where 8 bytes here and there would be merged in the cache.
template <int DT>
__device__ __forceinline__ void store_panel(const Mx4Product &p, int row, int col, f32x4 t0, f32x4 t1, f32x4 t2, f32x4 t3) {
  using E = Elem<DT>;
  using Bits = typename E::Bits;
  const int q = (int)(threadIdx.x & 63) >> 4;
  constexpr int kAlign = 16 / (int)sizeof(Bits);
  if (col + kMxPanelRows > p.w.rows || (uintptr_t)p.out % 16 != 0 || p.out_stride % kAlign != 0) {
    store4<DT>(p, row, col + 4 * q, t0);
    store4<DT>(p, row, col + 16 + 4 * q, t1);
    store4<DT>(p, row, col + 32 + 4 * q, t2);
    store4<DT>(p, row, col + 48 + 4 * q, t3);
    return;
  }
  f32x4 v[4] = {t0, t1, t2, t3};
  if (p.bias) {
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[t][i] += p.bias[col + 16 * t + 4 * q + i];
    }
  }
  constexpr int kWords = (int)sizeof(Bits);  // 32-bit words of four columns
  uint32_t u[4][kWords];
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    if constexpr (kWords == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) u[t][i] = E::narrow(v[t][i]);
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) u[t][i] = (uint32_t)E::narrow(v[t][2 * i]) | ((uint32_t)E::narrow(v[t][2 * i + 1]) << 16);
    }
  }
#pragma unroll
  for (int i = 0; i < kWords; ++i) {
    swap_halves(u[0][i], u[2][i]);
    swap_halves(u[1][i], u[3][i]);
    swap_quarters(u[0][i], u[1][i]);
    swap_quarters(u[2][i], u[3][i]);
  }
  if (row >= p.x.rows) return;
  Bits *dst = (Bits *)p.out + (int64_t)row * p.out_stride + col + 16 * q;
  if constexpr (kWords == 4) {
#pragma unroll
    for (int t = 0; t < 4; ++t) *reinterpret_cast<u32x4 *>(dst + 4 * t) = u32x4{u[t][0], u[t][1], u[t][2], u[t][3]};
  } else {
    *reinterpret_cast<u32x4 *>(dst) = u32x4{u[0][0], u[0][1], u[1][0], u[1][1]};
    *reinterpret_cast<u32x4 *>(dst + 8) = u32x4{u[2][0], u[2][1], u[3][0], u[3][1]};
  }
}

// Where a workgroup's tile lies. Workgroups go to the eight dies in turn, so each die is given a run of
// tiles that lie together: bands of eight tiles of X, along W, whose panels its cache then holds.
struct TilePlace { int w, x; };
__device__ __forceinline__ TilePlace tile_place(int id, int tiles_w, int tiles_x) {
  constexpr int kDies = 8, kBand = 8;
  const int total = tiles_w * tiles_x;
  const int die = id % kDies, each = total / kDies, more = total % kDies;
  const int at = die * each + min(die, more) + id / kDies;
  const int band = at / (kBand * tiles_w);
  const int in_band = at - band * kBand * tiles_w;
  const int wide = min(kBand, tiles_x - band * kBand);
  return {in_band / wide, band * kBand + in_band % wide};
}

// Waits until at most N of this wave's loads from memory are on their way and its reads of LDS are done,
// then for the workgroup's other waves. The memory clobbers keep the compiler from moving reads over it.
template <int N>
__device__ __forceinline__ void wait_and_meet() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// A constant that a lambda's body can use in constant expressions.
template <int V>
struct Const { static constexpr int value = V; };
template <int N, int I = 0, typename F>
__device__ __forceinline__ void unrolled(F f) {
  if constexpr (I < N) {
    f(Const<I>{});
    unrolled<N, I + 1>(f);
  }
}

typedef __attribute__((address_space(3))) void LdsVoid;
typedef const __attribute__((address_space(1))) void GlobalVoid;

// Large products, bound by the matrix cores and the LDS that feeds them: 4096 x 16384, k = 8192 in 243 us,
// 4.5 PFLOP/s. A workgroup of WM x WN waves has a tile of WM PM x WN PN panels of Y (64 x 64), PM x PN
// to a wave, and takes a panel of k (128) at a time. The panels of a stage lie in LDS as they do in
// memory, W's before X's, brought there without passing through registers, three stages in turn: one
// is in the waves' registers, one is being read into them, one or two are on their way. Eight waves of
// 128 x 64 read 96 KB of LDS to a stage's 512 multiplications, three quarters of its rate; four of 128 x 128
// would read 64 but need every register for the sums, which the compiler then copies about.
template <int PM, int PN, int WM, int WN>
struct TileShape {
  static constexpr int kWaves = WM * WN;
  static constexpr int kPanels = WM * PM + WN * PN;
  static constexpr int kCodes = kPanels * kMxPanelBytes;  // of a stage
  static constexpr int kStage = kCodes + kPanels * kMxPanelScales;
  static constexpr int kStages = 3;
  static constexpr int kHalves = 2 * kPanels / kWaves;  // half panels that a wave brings to a stage
  static_assert(2 * kPanels % kWaves == 0, "every wave brings as much");
  static constexpr int kScales = (kPanels + kWaves - 1) / kWaves;  // panels' scales, likewise
  static constexpr int kLoads = 2 * kHalves + kScales;
};

// Two tiles, from memory to LDS in lane order (the instruction's literal offset moves both addresses), and
// a panel's scales.
__device__ __forceinline__ void bring_half_panel(const uint8_t *from, uint8_t *to) {
  static_assert(kMxTileBytes == 1024, "the literal below");
  __builtin_amdgcn_global_load_lds((GlobalVoid *)from, (LdsVoid *)to, 16, 0, 0);
  __builtin_amdgcn_global_load_lds((GlobalVoid *)from, (LdsVoid *)to, 16, 1024, 0);
}
__device__ __forceinline__ void bring_scales(const uint8_t *from, uint8_t *to) {
  __builtin_amdgcn_global_load_lds((GlobalVoid *)from, (LdsVoid *)to, 4, 0, 0);
}

template <int DT, int PM, int PN, int WM, int WN>
__global__ __launch_bounds__(WM *WN * 64, 2) void mx4_tile_kernel(Mx4Product p, int tiles_w, int tiles_x) {
  using S = TileShape<PM, PN, WM, WN>;
  __shared__ __align__(1024) uint8_t lds[S::kStages][S::kStage];
  const int lane = (int)threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int wm = wave % WM, wn = wave / WM;
  const int kp = p.w.col_panels();
  const TilePlace place = tile_place((int)blockIdx.x, tiles_w, tiles_x);

  // Panels past the last are the last again; what they give is not stored.
  const int w_panels = (int)mx_panels(p.w.rows, kMxPanelRows), x_panels = (int)mx_panels(p.x.rows, kMxPanelRows);
  auto panel_at = [&](int panel) {
    return panel < WM * PM ? (int64_t)min(place.w * WM * PM + panel, w_panels - 1) * kp
                           : (int64_t)min(place.x * WN * PN + panel - WM * PM, x_panels - 1) * kp;
  };
  const uint8_t *codes[S::kHalves], *scales[S::kScales];
#pragma unroll
  for (int h = 0; h < S::kHalves; ++h) {
    const int half = wave * S::kHalves + h, panel = half >> 1;
    codes[h] = (panel < WM * PM ? p.w.codes : p.x.codes) + panel_at(panel) * kMxPanelBytes + (half & 1) * 2 * kMxTileBytes + lane * 16;
  }
#pragma unroll
  for (int h = 0; h < S::kScales; ++h) {
    const int panel = (wave + h * S::kWaves) % S::kPanels;  // twice where the waves do not come out even
    scales[h] = (panel < WM * PM ? p.w.scales : p.x.scales) + panel_at(panel) * kMxPanelScales + lane * 4;
  }
  int brought = 0;
  auto bring = [&](uint8_t *stage) {
    // Past the last panel of k it is the last one again, which nothing reads: every stage has as many loads.
    const int step = ++brought < kp ? 1 : 0;
#pragma unroll
    for (int h = 0; h < S::kHalves; ++h) {
      bring_half_panel(codes[h], stage + (wave * S::kHalves + h) * 2 * kMxTileBytes);
      codes[h] += step * kMxPanelBytes;
    }
#pragma unroll
    for (int h = 0; h < S::kScales; ++h) {
      bring_scales(scales[h], stage + S::kCodes + (wave + h * S::kWaves) % S::kPanels * kMxPanelScales);
      scales[h] += step * kMxPanelScales;
    }
  };

  constexpr int kW = PM * 4, kX = PN * 4;  // tiles of a wave
  f32x4 acc[kW][kX] = {};
  u32x4 w[kW], x[2][kX];
  uint32_t sw[2][PM], sx[2][PN];
  const int w_from = wm * PM * kMxPanelBytes + lane * 16, x_from = (WM * PM + wn * PN) * kMxPanelBytes + lane * 16;
  const int sw_from = S::kCodes + wm * PM * kMxPanelScales + lane * 4;
  const int sx_from = S::kCodes + (WM * PM + wn * PN) * kMxPanelScales + lane * 4;
  auto read16 = [&](const uint8_t *at) { return *reinterpret_cast<const u32x4 *>(at); };
  auto read_scales = [&](const uint8_t *stage, uint32_t(&to_w)[PM], uint32_t(&to_x)[PN]) {
#pragma unroll
    for (int i = 0; i < PM; ++i) to_w[i] = *reinterpret_cast<const uint32_t *>(stage + sw_from + i * kMxPanelScales);
#pragma unroll
    for (int j = 0; j < PN; ++j) to_x[j] = *reinterpret_cast<const uint32_t *>(stage + sx_from + j * kMxPanelScales);
  };
  bring(lds[0]);
  bring(lds[1]);
  bring(lds[2]);
  wait_and_meet<2 * S::kLoads>();
#pragma unroll
  for (int t = 0; t < kW; ++t) w[t] = read16(lds[0] + w_from + t * kMxTileBytes);
#pragma unroll
  for (int t = 0; t < kX; ++t) x[0][t] = read16(lds[0] + x_from + t * kMxTileBytes);
  read_scales(lds[0], sw[0], sx[0]);
  int now = 0;  // the stage whose values are in registers
  auto step = [&](auto parity) {
    constexpr int P = decltype(parity)::value;
    wait_and_meet<S::kLoads>();
    bring(lds[now]);
    now = now == S::kStages - 1 ? 0 : now + 1;
    const uint8_t *next = lds[now];
    read_scales(next, sw[1 - P], sx[1 - P]);
    // One of W's tiles at a time: after its products its registers take its next one, and beside them
    // some of the next tiles of X are read.
    unrolled<kW>([&](auto r) {
      constexpr int R = decltype(r)::value;
      unrolled<kX>([&](auto c) {
        constexpr int C = decltype(c)::value;
        acc[R][C] = mx4_mfma<R % 4, C % 4>(w[R], x[P][C], acc[R][C], sw[P][R / 4], sx[P][C / 4]);
      });
      unrolled<kX>([&](auto c) {
        constexpr int C = decltype(c)::value;
        if constexpr (C * kW / kX == R) x[1 - P][C] = read16(next + x_from + C * kMxTileBytes);
      });
      w[R] = read16(next + w_from + R * kMxTileBytes);
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  int k = 0;
  for (; k + 1 < kp; k += 2) {
    step(Const<0>{});
    step(Const<1>{});
  }
  if (k < kp) step(Const<0>{});
  wait_and_meet<0>();
#pragma unroll
  for (int i = 0; i < PM; ++i) {
#pragma unroll
    for (int j = 0; j < kX; ++j) {
      const int row = (place.x * WN + wn) * PN * kMxPanelRows + j * kMxTileRows + (lane & 15);
      const int col = ((place.w * WM + wm) * PM + i) * kMxPanelRows;
      store_panel<DT>(p, row, col, acc[i * 4][j], acc[i * 4 + 1][j], acc[i * 4 + 2][j], acc[i * 4 + 3][j]);
    }
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

constexpr int64_t kTilesMax = 1 << 22;  // of a launch: 2^32 threads are too many

template <int DT, int PM, int PN, int WM, int WN>
int launch_tiles(const Mx4Product &p, hipStream_t s) {
  const int64_t tiles_w = mx_panels(p.w.rows, kMxPanelRows * PM * WM), tiles_x = mx_panels(p.x.rows, kMxPanelRows * PN * WN);
  if (tiles_w * tiles_x > kTilesMax) return record_failure(TABBY_EINVAL, "the product is too large for one launch");
  hipLaunchKernelGGL((mx4_tile_kernel<DT, PM, PN, WM, WN>), dim3((unsigned)(tiles_w * tiles_x)), dim3(WM * WN * 64), 0, s, p,
                     (int)tiles_w, (int)tiles_x);
  TABBY_HIP_CHECK(hipGetLastError());
  return TABBY_OK;
}

constexpr int kTileRowsMin = 64;  // rows of X from which a tile pays
constexpr int kCus = 256;         // an MI355X's compute units

// Whether tiles of 256 x 256 are the better choice, else 128 x 128. A unit holds one of the large tiles,
// and they do the same work in 3.5/4 of the time (4096 x 16384, k = 8192: 243 us and 270), but a last
// round of them that few units take part in costs as much as a full one: 318 x 44368, k = 6704: 86 us
// and 66; 2048 x 4096, k = 4096: 29 and 22.
bool large_tiles(int n, int rows) {
  const int64_t large = mx_panels(n, 256) * mx_panels(rows, 256), small = mx_panels(n, 128) * mx_panels(rows, 128);
  return 7 * mx_panels(large, kCus) <= 2 * mx_panels(small, kCus);
}

template <int DT>
int launch_product(const Mx4Product &p, hipStream_t s) {
  if (p.x.rows >= kTileRowsMin) return large_tiles(p.w.rows, p.x.rows) ? launch_tiles<DT, 2, 1, 2, 4>(p, s) : launch_tiles<DT, 1, 1, 2, 2>(p, s);
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
