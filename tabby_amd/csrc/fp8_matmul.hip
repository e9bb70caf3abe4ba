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
// keeps of each what lies above 2^-13 of the group's largest, or better (measured: 1.5e-5 of the result's norm for normal
// values, 5e-5 for codes drawn alike; where large products cancel it is what is left). The first is taken unless the caller
// asks for the second (TABBY_FP8_FAST_SUMS), which more than 64 rows to f16 or bf16 then take: fewer are bound by
// memory, and f32 would show the difference.

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

// Both scales' product is formed first, in f32: t, 0 or from 2^-18 to 2^25, is then one multiplication and addition away from
// the sum. That product may be no ordinary number (blocks whose scales lie near f32's ends), although s_x s_w t is one: a wave that has met
// such a block goes over its part again, in 64 bits, which hold s_x s_w exactly.
struct ScaleRange {
  float least = 1.0f, most = 1.0f;  // of the products' magnitudes; NaN is as good as any
  template <int N>
  __device__ __forceinline__ void see(const float (&s)[N], float sw) {
    float low = __builtin_fabsf(s[0]), high = low;
#pragma unroll
    for (int i = 1; i < N; ++i) {
      low = __builtin_fminf(low, __builtin_fabsf(s[i]));
      high = __builtin_fmaxf(high, __builtin_fabsf(s[i]));
    }
    least = __builtin_fminf(least, sw == 0.0f ? 1.0f : low);  // (a weights' block that is empty; X's are not)
    most = __builtin_fmaxf(most, high);
  }
  __device__ __forceinline__ bool odd() const { return __ballot(least < 0x1p-100f || most > 0x1p100f) != 0; }
};
__device__ __forceinline__ void add_scaled_wide(f32x4 &acc, f32x4 t, float sx, float sw) {
  const double s = (double)sx * (double)sw;
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i] = (float)__builtin_fma((double)t[i], s, (double)acc[i]);
}

// A square block's scale, the same for the whole wave: by the scalar unit, whose loads no wait for the vector ones holds up.
__device__ __forceinline__ float block_scale_at(const float *scales, int64_t at) {
  typedef const __attribute__((address_space(4))) float Constant;
  return ((Constant *)(uintptr_t)scales)[at];
}

struct Fp8Product {
  Fp8Matrix w, x;  // square blocks; blocks of one row
  ProductOut y;
};

// A workgroup of WM x WN waves has a tile of WM PM x WN PN panels of Y (64 x 64), PM x PN to a wave, and takes a
// panel of k (128) at a time. The panels of a stage lie in LDS as they do in memory, W's before X's, then X's scales,
// brought there without passing through registers, a stage ahead. A wave holds the tiles of X and goes through those
// of W; a tile's results are added while the next one's products run. 4,096 rows, W of 16,384 x 4,096 to bf16: 460 to 473 us, one card or
// another, 1.2 PFLOP/s, of which the f16 instructions' rate allows some 450 (the library's bf16 product runs at 1.23); to f32 499 to
// 511. As codes, in tiles of 256 x 256: 252 us, 2.2 PFLOP/s, and the chip's power bounds it (orders of a step that take 674,000, 600,000 and 544,000 cycles,
// 262,000 of them the matrix cores', take the same time, at 2.2 to 1.87 GHz; without the scaled additions 13 % less), so the
// order is the simplest. Where there are few tiles, KG groups of such waves take every KG-th panel of k, each with stages of
// its own, and add up through LDS.
template <int PM, int PN, int WM, int WN, int KG>
struct TileShape {
  static constexpr int kWaves = WM * WN;
  static constexpr int kPanels = WM * PM + WN * PN;
  static constexpr int kCodes = kPanels * kF8PanelBytes;  // of a stage
  static constexpr int kStage = kCodes + WN * PN * kF8PanelScales;
  static constexpr int kStages = 2;
  static constexpr int kTiles = 4 * kPanels / kWaves;  // tiles that a wave brings to a stage
  static_assert(4 * kPanels % kWaves == 0, "every wave brings as much");
  static_assert(PM <= 2, "a wave's panels of W lie in one square block");
  static constexpr int kLds = KG * kStages * kStage;
  static_assert(KG == 1 || (KG == 2 && kWaves * PM * PN * 16 * 1024 <= kLds), "a group's sums find room");
};

__device__ __forceinline__ void bring_tile(const uint8_t *from, uint8_t *to) {
  static_assert(kF8TileBytes == 2048, "the literal below");
  __builtin_amdgcn_global_load_lds((GlobalVoid *)from, (LdsVoid *)to, 16, 0, 0);
  __builtin_amdgcn_global_load_lds((GlobalVoid *)from, (LdsVoid *)to, 16, 1024, 0);
}
__device__ __forceinline__ void bring_scales(const uint8_t *from, uint8_t *to) {
  __builtin_amdgcn_global_load_lds((GlobalVoid *)from, (LdsVoid *)to, 4, 0, 0);
}

template <int DT, typename Operand, int PM, int PN, int WM, int WN, int KG>
__global__ __launch_bounds__(KG *WM *WN * 64, 2) void fp8_tile_kernel(Fp8Product p, int tiles_w, int tiles_x) {
  using S = TileShape<PM, PN, WM, WN, KG>;
  __shared__ __align__(1024) uint8_t all_lds[S::kLds];
  const int lane = (int)threadIdx.x & 63;
  const int all_waves = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int group = all_waves / S::kWaves, wave = all_waves % S::kWaves;
  const int wm = wave % WM, wn = wave / WM;
  const int kp = p.w.col_panels();
  uint8_t(*const lds)[S::kStage] = reinterpret_cast<uint8_t(*)[S::kStage]>(all_lds + group * S::kStages * S::kStage);
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
  int at = 0;  // the panel of k that comes next
  auto advance = [&](int to) {
    // Past the last panel of k it is the last one again, which nothing uses: every stage has as many loads.
    const int step = min(to, kp - 1) - at;
    at += step;
#pragma unroll
    for (int h = 0; h < S::kTiles; ++h) codes[h] += step * kF8PanelBytes;
    x_scales += step * kF8PanelScales;
  };
  advance(group);
  auto bring = [&](uint8_t *stage) {
#pragma unroll
    for (int h = 0; h < S::kTiles; ++h) bring_tile(codes[h], stage + (wave * S::kTiles + h) * kF8TileBytes);
    bring_scales(x_scales, stage + S::kCodes + scales_of * kF8PanelScales);
  };
  // The wave's panels of W lie in one square block.
  const float *w_scales = p.w.scales + (int64_t)(min((place.w * WM + wm) * PM, w_panels - 1) >> 1) * kp;

  constexpr int kW = PM * 4, kX = PN * 4;  // tiles of a wave
  f32x4 acc[kW][kX] = {};
  const int w_from = wm * PM * kF8PanelBytes + lane * 16, x_from = (WM * PM + wn * PN) * kF8PanelBytes + lane * 16;
  const int sx_from = S::kCodes + wn * PN * kF8PanelScales + (lane & 15) * 4;
  bring(lds[0]);
  int now = 0;
  float sw = block_scale_at(w_scales, at);
  ScaleRange range;
  for (int first = 0; first < kp; first += KG) {
    const bool works = first + group < kp;  // the last group may have a panel less
    wait_and_meet<0>();
    const uint8_t *stage = lds[now];
    now ^= 1;
    advance(first + group + KG);
    bring(lds[now]);
    const float sw_next = block_scale_at(w_scales, at);
    if (KG > 1 && !works) continue;
    Operand x[kX];
    TileCodes w[3];
    float s[kX];
    w[0] = read_tile(stage + w_from);
#pragma unroll
    for (int c = 0; c < kX; ++c) x[c] = Operand(read_tile(stage + x_from + c * kF8TileBytes));
    w[1] = read_tile(stage + w_from + kF8TileBytes);
#pragma unroll
    for (int c = 0; c < kX; ++c) s[c] = *reinterpret_cast<const float *>(stage + sx_from + c * 64) * sw;
    f32x4 t[2][kX];
#pragma unroll
    for (int r = 0; r < kW; ++r) {
      // Two tiles ahead of the products.
      if (r + 2 < kW) w[(r + 2) % 3] = read_tile(stage + w_from + (r + 2) * kF8TileBytes);
      __builtin_amdgcn_sched_barrier(0);
      const Operand of_w(w[r % 3]);
#pragma unroll
      for (int c = 0; c < kX; ++c) {
        // A product is on its way while an earlier one's results are added: in this order, or they would be waited for.
        t[r & 1][c] = tile_product(of_w, x[c]);
        __builtin_amdgcn_sched_barrier(0);
        if (r > 0) add_scaled(acc[r - 1][c], t[(r - 1) & 1][c], s[c]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
#pragma unroll
    for (int c = 0; c < kX; ++c) add_scaled(acc[kW - 1][c], t[(kW - 1) & 1][c], s[c]);
    range.see(s, sw);
    sw = sw_next;
  }
  if (range.odd()) {
#pragma unroll
    for (int i = 0; i < kW * kX; ++i) {
      const int r = i / kX, c = i % kX;
      const int64_t w_panel = panel_at(wm * PM + r / 4), x_panel = panel_at(WM * PM + wn * PN + c / 4);
      const uint8_t *w_from_memory = p.w.codes + w_panel * kF8PanelBytes + r % 4 * kF8TileBytes + lane * 16;
      const uint8_t *x_from_memory = p.x.codes + x_panel * kF8PanelBytes + c % 4 * kF8TileBytes + lane * 16;
      const float *sx = p.x.scales + x_panel * kF8PanelRows + c % 4 * kF8TileRows + (lane & 15);
      f32x4 sum = {0, 0, 0, 0};
#pragma unroll 1
      for (int64_t k = group; k < kp; k += KG)
        add_scaled_wide(sum, tile_product(Operand(read_tile(w_from_memory + k * kF8PanelBytes)), Operand(read_tile(x_from_memory + k * kF8PanelBytes))),
                        sx[k * kF8PanelRows], block_scale_at(w_scales, k));
      acc[r][c] = sum;
    }
  }
  wait_and_meet<0>();
  if constexpr (KG > 1) {
    f32x4 *const sums = reinterpret_cast<f32x4 *>(all_lds) + wave * kW * kX * 64 + lane;
    if (group == 1) {
#pragma unroll
      for (int i = 0; i < kW * kX; ++i) sums[i * 64] = acc[i / kX][i % kX];
    }
    __syncthreads();
    if (group == 1) return;
#pragma unroll
    for (int i = 0; i < kW * kX; ++i) acc[i / kX][i % kX] += sums[i * 64];
  }
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
// through LDS. The registers of a tile of W take the next panel's as soon as the tile is read, so a panel is on its way
// all the time (two for one tile of rows, which leaves the registers). Workgroups of four waves where the slices allow:
// one token, W of 151,936 x 896: 22 us, 6.2 TB/s, and 27 us a call; with workgroups of eight the call took 30 us.
struct FewShape {
  int waves, slices;  // of a workgroup; powers of two
};
constexpr int kSlicesMax = 8;
constexpr int kSumsMax = 16;  // slices * NT
constexpr int kFewWaves = 8;
constexpr int kFewWavesMin = 4;
// The upper half of the slices' sums lie in LDS, 4 KB to a wave's tile of rows.
__host__ __device__ constexpr int sums_bytes(int waves, int tiles) { return waves / 2 * tiles * 4096; }
constexpr int kStepBytes = kF8TileBytes + 64;  // codes and scales of 16 rows, 128 columns

// The tiles of X as they are held.
template <int NT, typename OP>
struct HeldTiles {
  using Args = Fp8Matrix;
  using Operand = OP;
  static constexpr int kTiles = NT;
  static constexpr bool kFills = false;
  static constexpr int kAhead = NT == 1 ? 2 : 1;
  static constexpr int kLds = sums_bytes(kFewWaves, NT);
  struct Raw {
    TileCodes x[NT];
    float scale[NT];
  };
  const uint8_t *codes;
  const float *scales;
  __device__ __forceinline__ HeldTiles(const Fp8Matrix &m, const uint8_t *, int tile, int lane) {
    // NT tiles from `tile` on lie in one panel.
    const int64_t panel = (int64_t)(tile >> 2) * m.col_panels();
    codes = m.codes + panel * kF8PanelBytes + (tile & 3) * kF8TileBytes + lane * 16;
    scales = m.scales + panel * kF8PanelRows + (tile & 3) * kF8TileRows + (lane & 15);
  }
  static __device__ __forceinline__ void fill(const Fp8Matrix &, uint8_t *, int) {}
  __device__ __forceinline__ void load(int k, Raw &r) const {
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      r.x[u] = read_tile(codes + (int64_t)k * kF8PanelBytes + u * kF8TileBytes);
      r.scale[u] = scales[(int64_t)k * kF8PanelRows + u * kF8TileRows];
    }
  }
  __device__ __forceinline__ Operand tile(const Raw &r, int, int u, float &scale) const {
    scale = r.scale[u];
    return Operand(r.x[u]);
  }
};

// Up to 16 rows of x's own values, kFillPanels blocks at most: every workgroup quantises all of them into LDS while its
// first panels of W are on their way. Rows past the last hold anything.
constexpr int kFillPanels = 32;

struct FloatRows {
  const void *x;
  int64_t stride;
  int rows, cols;
};

template <int XDT>
struct FloatTiles {
  using E = Elem<XDT>;
  using Args = FloatRows;
  using Operand = HalfOperand;
  static constexpr int kTiles = 1;
  static constexpr bool kFills = true;
  static constexpr int kAhead = 2;
  static constexpr int kBlockLanes = kF8Block / E::kVec;  // they lie together: the workgroup's threads are a multiple
  static constexpr int kLoads = kFillPanels * kBlockLanes / (kFewWavesMin * 64);  // of a thread, 16 bytes each
  static constexpr int kLds = kFillPanels * kStepBytes;
  static_assert(kLds >= sums_bytes(kFewWaves, 1), "the slices' sums find room");
  struct Raw {};
  const uint8_t *codes;
  bool held;  // the lane's row is one of x
  __device__ __forceinline__ FloatTiles(const FloatRows &a, const uint8_t *lds, int, int lane) : codes(lds + lane * 16), held((lane & 15) < a.rows) {}
  static __device__ __forceinline__ void fill(const FloatRows &a, uint8_t *lds, int kp) {
    const int row_lanes = kp * kBlockLanes, all = a.rows * row_lanes;
    const float per_row = 1.0f / (float)row_lanes;  // all <= 2^10: (i + 1/2) / row_lanes has bits to spare
    u32x4 raw[kLoads];
#pragma unroll
    for (int n = 0; n < kLoads; ++n) {
      const int i = n * (int)blockDim.x + (int)threadIdx.x, r = (int)(((float)i + 0.5f) * per_row);
      raw[n] = i < all ? load_values<XDT, false>((const typename E::Bits *)a.x + (int64_t)r * a.stride, (i - r * row_lanes) * E::kVec, a.cols) : u32x4{0, 0, 0, 0};
    }
#pragma unroll
    for (int n = 0; n < kLoads; ++n) {
      const int i = n * (int)blockDim.x + (int)threadIdx.x, r = (int)(((float)i + 0.5f) * per_row);
      const int at = i - r * row_lanes;
      uint32_t top = f8_largest<XDT>(raw[n]);
#pragma unroll
      for (int lanes = 1; lanes < kBlockLanes; lanes *= 2) top = max(top, xor_lane_by(top, lanes));
      float scale, inverse;
      f8_scale(top, scale, inverse);
      if (i >= all) break;
      uint8_t *to = lds + at / kBlockLanes * kStepBytes;
      f8_encode<XDT>(to + f8_code_byte(r, at % kBlockLanes * E::kVec), raw[n], inverse);
      if (at % kBlockLanes == 0) reinterpret_cast<float *>(to + kF8TileBytes)[r] = scale;
    }
  }
  __device__ __forceinline__ void load(int, Raw &) const {}
  __device__ __forceinline__ HalfOperand tile(const Raw &, int k, int, float &scale) const {
    const uint8_t *at = codes + k * kStepBytes;
    scale = *reinterpret_cast<const float *>(at - (int)(threadIdx.x & 63) * 16 + kF8TileBytes + (threadIdx.x & 15) * 4);
    if (!held) scale = 1.0f;  // (nothing has been written there)
    return HalfOperand(read_tile(at));
  }
};

template <int DT, typename Rows>
__global__ __launch_bounds__(kFewWaves * 64, 2) void fp8_few_kernel(Fp8Product p, typename Rows::Args xs, FewShape shape) {
  constexpr int NT = Rows::kTiles;
  __shared__ __align__(16) uint8_t lds[Rows::kLds];
  const int lane = (int)threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int slice = wave & (shape.slices - 1);
  const int panel = (int)blockIdx.x * (shape.waves / shape.slices) + wave / shape.slices;
  const int kp = p.w.col_panels();
  const int tile = (int)blockIdx.y * NT;
  // A wave past the last panel has nothing to do but to meet the others.
  const bool works = panel * kF8PanelRows < p.w.rows;
  const Rows rows(xs, lds, tile, lane);
  const uint8_t *wc = p.w.codes + (int64_t)panel * kp * kF8PanelBytes + lane * 16;
  const float *ws = p.w.scales + (int64_t)(panel >> 1) * kp;
  int k = (int)((int64_t)kp * slice / shape.slices);
  const int end = works ? (int)((int64_t)kp * (slice + 1) / shape.slices) : k;
  // The panels of W that come next, two or one; a tile's registers take the one after as soon as it is read.
  constexpr int kAhead = Rows::kAhead;
  struct Step {
    TileCodes w[4];
    float scale;
  } steps[kAhead];
  auto bring = [&](int at, Step &s, int t) { s.w[t] = read_tile(wc + (int64_t)at * kF8PanelBytes + t * kF8TileBytes); };
  typename Rows::Raw raw;
  f32x4 acc[4][NT] = {};
  const int begin = k;
  ScaleRange range;
  auto multiply = [&](int at, Step &s, auto more) {
    constexpr bool kMore = decltype(more)::value != 0;
    typename Rows::Operand x[NT];
    float both[NT];
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      x[u] = rows.tile(raw, at, u, both[u]);
      both[u] *= s.scale;
    }
    range.see(both, s.scale);
    rows.load(min(at + 1, end - 1), raw);
    if constexpr (kMore) s.scale = block_scale_at(ws, at + kAhead);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const typename Rows::Operand w(s.w[t]);
      if constexpr (kMore) bring(at + kAhead, s, t);
#pragma unroll
      for (int u = 0; u < NT; ++u) add_scaled(acc[t][u], tile_product(w, x[u]), both[u]);
    }
  };
  if (k < end) {
    rows.load(k, raw);
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      const int at = min(k + a, end - 1);
      steps[a].scale = block_scale_at(ws, at);
#pragma unroll
      for (int t = 0; t < 4; ++t) bring(at, steps[a], t);
    }
  }
  if constexpr (Rows::kFills) {
    Rows::fill(xs, lds, kp);
    __syncthreads();
  }
  constexpr Const<1> kWith;
  constexpr Const<0> kWithout;
  if constexpr (kAhead == 1) {
    for (; k + 1 < end; ++k) multiply(k, steps[0], kWith);
    if (k < end) multiply(k, steps[0], kWithout);
  } else {
    for (; k + 3 < end; k += 2) {
      multiply(k, steps[0], kWith);
      multiply(k + 1, steps[1], kWith);
    }
    if (k + 2 < end) {
      multiply(k, steps[0], kWith);
      multiply(k + 1, steps[1], kWithout);
      multiply(k + 2, steps[0], kWithout);
    } else {
      if (k < end) multiply(k, steps[0], kWithout);
      if (k + 1 < end) multiply(k + 1, steps[1], kWithout);
    }
  }
  if (range.odd()) {
#pragma unroll
    for (int i = 0; i < 4 * NT; ++i) acc[i / NT][i % NT] = f32x4{0, 0, 0, 0};
#pragma unroll 1
    for (k = begin; k < end; ++k) {
      rows.load(k, raw);
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        float sx;
        const typename Rows::Operand x = rows.tile(raw, k, u, sx);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const typename Rows::Operand w(read_tile(wc + (int64_t)k * kF8PanelBytes + t * kF8TileBytes));
          add_scaled_wide(acc[t][u], tile_product(w, x), sx, block_scale_at(ws, k));
          __builtin_amdgcn_sched_barrier(0);  // one at a time, in few registers
        }
      }
    }
  }
  // The slices in halves: the upper half's sums go through LDS to the lower half's waves.
  if constexpr (Rows::kFills) {
    if (shape.slices > 1) __syncthreads();
  }
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

// What the caller asks for: the result's type, and whether its sums may be the codes' own.
struct OutType {
  int32_t dtype;
  bool fast;
  explicit OutType(int32_t asked) : dtype(asked & ~TABBY_FP8_FAST_SUMS), fast((asked & TABBY_FP8_FAST_SUMS) != 0) {}
};

constexpr int kCus = 256;               // an MI355X's compute units
constexpr int64_t kTilesMax = 1 << 22;  // of a launch: 2^32 threads are too many

// Tiles of 128 x 128.
int64_t small_tiles(int n, int rows) { return f8_parts(n, 128) * f8_parts(rows, 128); }

// Whether W is streamed into registers: up to 64 rows, which one wave takes, and where tiles of 128 x 128 would leave half
// of the units idle (W of 4,864 x 4,096 to bf16, the product alone. 300 rows: 19 us, in tiles 33; as codes 15, in tiles 20. 512 rows: 30 us, in
// tiles 33; as codes 26, in tiles 21).
bool few_rows(int n, int rows) { return rows <= kF8PanelRows || small_tiles(n, rows) < kCus / 2; }

template <int DT, typename Operand, int PM, int PN, int WM, int WN, int KG>
int launch_tiles(const Fp8Product &p, hipStream_t s) {
  const int64_t tiles_w = f8_parts(p.w.rows, kF8PanelRows * PM * WM), tiles_x = f8_parts(p.x.rows, kF8PanelRows * PN * WN);
  if (tiles_w * tiles_x > kTilesMax) return record_failure(TABBY_EINVAL, "the product is too large for one launch");
  hipLaunchKernelGGL((fp8_tile_kernel<DT, Operand, PM, PN, WM, WN, KG>), dim3((unsigned)(tiles_w * tiles_x)), dim3(KG * WM * WN * 64), 0, s, p,
                     (int)tiles_w, (int)tiles_x);
  TABBY_HIP_CHECK(hipGetLastError());
  return TABBY_OK;
}

// Whether tiles of 256 x 256 are the better choice, else 128 x 128: a last round of them that few units take part in
// costs as much as a full one.
bool large_tiles(int n, int rows) {
  const int64_t large = f8_parts(n, 256) * f8_parts(rows, 256);
  return 7 * f8_parts(large, kCus) <= 2 * f8_parts(small_tiles(n, rows), kCus);
}

template <int DT, typename Rows>
int launch_few(const Fp8Product &p, const typename Rows::Args &xs, hipStream_t s) {
  constexpr int NT = Rows::kTiles;
  const int64_t panels = f8_parts(p.w.rows, kF8PanelRows), groups = f8_parts(p.x.rows, kF8TileRows * NT);
  // As many waves as the chip holds at once, eight to a unit, while every one has a panel of k.
  int slices = 1;
  while (slices < kSlicesMax && slices * 2 <= p.w.col_panels() && slices * 2 * NT <= kSumsMax && panels * groups * slices * 2 <= kFewWaves * kCus) slices *= 2;
  const FewShape shape{std::max(slices, kFewWavesMin), slices};
  const int64_t blocks = f8_parts(panels, shape.waves / shape.slices);
  hipLaunchKernelGGL((fp8_few_kernel<DT, Rows>), dim3((unsigned)blocks, (unsigned)groups), dim3(64 * shape.waves), 0, s, p, xs, shape);
  TABBY_HIP_CHECK(hipGetLastError());
  return TABBY_OK;
}

// X as it is held; `Most` is what more than 64 rows are multiplied as.
template <int DT, typename Most>
int launch_product(const Fp8Product &p, hipStream_t s) {
  if (!few_rows(p.w.rows, p.x.rows)) {
    // (As f16, X's tiles take twice the registers: the large ones do not fit.)
    if constexpr (std::is_same<Most, CodeOperand>::value) {
      if (large_tiles(p.w.rows, p.x.rows)) return launch_tiles<DT, Most, 2, 1, 2, 4, 1>(p, s);
    }
    // (512 rows, W of 4,864 x 4,096 to bf16: 33 us with two groups of waves, 41 us with one; as codes 21 and 25.)
    return small_tiles(p.w.rows, p.x.rows) <= kCus ? launch_tiles<DT, Most, 1, 1, 2, 2, 2>(p, s) : launch_tiles<DT, Most, 1, 1, 2, 2, 1>(p, s);
  }
  switch (f8_parts(p.x.rows, kF8TileRows)) {
    case 1: return launch_few<DT, HeldTiles<1, HalfOperand>>(p, p.x, s);
    case 2: return launch_few<DT, HeldTiles<2, HalfOperand>>(p, p.x, s);
    case 3: return launch_few<DT, HeldTiles<3, HalfOperand>>(p, p.x, s);
    case 4: return launch_few<DT, HeldTiles<4, HalfOperand>>(p, p.x, s);
    default: return launch_few<DT, HeldTiles<4, Most>>(p, p.x, s);
  }
}

int product(const Fp8Product &p, const OutType &out, hipStream_t s) {
  switch (out.dtype) {
    case TABBY_F32: return launch_product<TABBY_F32, HalfOperand>(p, s);
    case TABBY_F16: return out.fast ? launch_product<TABBY_F16, CodeOperand>(p, s) : launch_product<TABBY_F16, HalfOperand>(p, s);
    default: return out.fast ? launch_product<TABBY_BF16, CodeOperand>(p, s) : launch_product<TABBY_BF16, HalfOperand>(p, s);
  }
}

// X quantised in the product's own launch.
bool fills(int rows, int kp) { return rows <= kF8TileRows && kp <= kFillPanels / rows; }

template <int DT>
int launch_linear(const Fp8Product &p, const FloatRows &x, int x_dtype, hipStream_t s) {
  switch (x_dtype) {
    case TABBY_F32: return launch_few<DT, FloatTiles<TABBY_F32>>(p, x, s);
    case TABBY_F16: return launch_few<DT, FloatTiles<TABBY_F16>>(p, x, s);
    default: return launch_few<DT, FloatTiles<TABBY_BF16>>(p, x, s);
  }
}

int linear(const Fp8Product &p, const FloatRows &x, int x_dtype, int32_t out_dtype, hipStream_t s) {
  switch (out_dtype) {
    case TABBY_F32: return launch_linear<TABBY_F32>(p, x, x_dtype, s);
    case TABBY_F16: return launch_linear<TABBY_F16>(p, x, x_dtype, s);
    default: return launch_linear<TABBY_BF16>(p, x, x_dtype, s);
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

int check_result(const void *out_dev, const OutType &out, int32_t rows, int32_t n, int64_t stride) {
  const int rc = check_output(out_dev, out.dtype, rows, n, stride);
  if (!rc && out.fast && out.dtype == TABBY_F32) return record_failure(TABBY_EINVAL, "TABBY_FP8_FAST_SUMS is for f16 and bf16 results");
  return rc;
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
  const OutType type(out_dtype);
  if (!rc) rc = check_result(out_dev, type, rows, n, out_stride);
  if (!rc) rc = check_bias(bias_dev);
  if (rc) return rc;
  const Fp8Product p{{(const uint8_t *)w_codes_dev, (const float *)w_scales_dev, n, k},
                     {(const uint8_t *)x_codes_dev, (const float *)x_scales_dev, rows, k},
                     {rows, n, bias_dev, out_dev, out_stride}};
  const RowSpan out = row_span(out_dev, rows, n, out_stride, dtype_size(type.dtype));
  rc = check_apart(out, p);
  if (!rc) rc = check_fp8_apart(out, x_codes_dev, x_scales_dev, rows, k, 1);
  if (rc) return rc;
  return product(p, type, (hipStream_t)stream);
}

extern "C" int tabby_fp8_linear_device(const void *x_dev, int32_t x_dtype, int64_t x_stride, int32_t rows,
                                       const void *w_codes_dev, const void *w_scales_dev, const float *bias_dev,
                                       int32_t n, int32_t k, void *out_dev, int32_t out_dtype, int64_t out_stride,
                                       void *workspace_dev, int64_t workspace_bytes, void *stream) {
  if (!x_dev || !workspace_dev) return record_failure(TABBY_EINVAL, "null pointer");
  int rc = check_fp8_operand(w_codes_dev, w_scales_dev);
  if (!rc) rc = check_fp8_shape(rows, k, 1);
  if (!rc) rc = check_fp8_shape(n, k, kF8Block);
  const OutType type(out_dtype);
  if (!rc) rc = check_result(out_dev, type, rows, n, out_stride);
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
  const RowSpan out = row_span(out_dev, rows, n, out_stride, dtype_size(type.dtype));
  rc = check_apart(out, p);
  if (!rc) rc = check_apart(row_span(workspace_dev, 1, need, 0, 1), p);
  if (rc) return rc;
  if (rows_meet(out, workspace_dev, need) || rows_meet(x, workspace_dev, need))
    return record_failure(TABBY_EINVAL, "workspace must not overlap x or out");
  // A result that lies on x (a layer whose input and output share a buffer) is written after a launch that has read
  // all of x; in the product's own launch some workgroups would read what others have written.
  const bool apart = !rows_meet({out_dev, 1, out.bytes(), 0}, x_dev, x.bytes());
  if (apart && fills(rows, p.w.col_panels()))
    return linear(p, FloatRows{x_dev, x_stride, rows, k}, x_dtype, type.dtype, (hipStream_t)stream);
  rc = fp8_quantize(x_dev, x_dtype, rows, k, x_stride, 1, codes, scales, (hipStream_t)stream);
  if (rc) return rc;
  return product(p, type, (hipStream_t)stream);
}
