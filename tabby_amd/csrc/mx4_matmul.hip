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
#include "wave_ops.h"

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
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (col + i < n) dst[i] = E::narrow(v[i]);
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
// lanes fill whole lines, where 8 bytes here and there would be merged in the cache. Rows of odd strides are
// stored as widely: the hardware takes any address (589 x 46311 f16, k = 1336: 53 us, element by element 72).
template <int DT>
__device__ __forceinline__ void store_panel(const Mx4Product &p, int row, int col, f32x4 t0, f32x4 t1, f32x4 t2, f32x4 t3) {
  using E = Elem<DT>;
  using Bits = typename E::Bits;
  const int q = (int)(threadIdx.x & 63) >> 4;
  if (col + kMxPanelRows > p.w.rows) {
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
    for (int t = 0; t < 4; ++t) *reinterpret_cast<u32x4_any *>(dst + 4 * t) = u32x4{u[t][0], u[t][1], u[t][2], u[t][3]};
  } else {
    *reinterpret_cast<u32x4_any *>(dst) = u32x4{u[0][0], u[0][1], u[1][0], u[1][1]};
    *reinterpret_cast<u32x4_any *>(dst + 8) = u32x4{u[2][0], u[2][1], u[3][0], u[3][1]};
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

// Large products: 4096 x 16384, k = 8192 in 227 to 243 us, one card or another, 4.5 to 4.8 PFLOP/s (random operands
// that stay in registers run at 7.3). Bound by the schedule and the clock. The matrix cores are busy in 59 % of
// 446,000 cycles; the rest is each step's wait for LDS and for the slowest wave, and a tenth the stores of Y. Zeros
// take as many cycles (435,000) at 2.47 GHz, 176 us; random operands draw more power and the card runs them at 1.86.
// A workgroup of WM x WN waves has a tile of WM PM x WN PN panels
// of Y (64 x 64), PM x PN to a wave, and takes a panel of k (128) at a time. The panels of a stage lie in
// LDS as they do in memory, W's before X's, brought there without passing through registers, three stages in
// turn: one is in the waves' registers, one is being read into them, one or two are on their way. Eight waves
// of 128 x 64 leave registers for the next operands; four of 128 x 128 would read a third less of LDS but need
// every register for the sums, which the compiler then copies about (368 us).
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

// Few rows: W is streamed from memory straight into registers, a wave to a panel of 64 columns of Y and
// NT tiles of 16 rows. Bound by HBM where W is large (1 x 151936, k = 896: 13 us, 5.6 TB/s); where it is
// small, by how long a wave takes for its share of k, so `slices` waves of the workgroup take a part of
// k each and add up through LDS.
struct FewShape {
  int waves, slices;  // of a workgroup; powers of two
};
constexpr int kSlicesMax = 8;
constexpr int kSumsMax = 16;                   // slices * NT
// The upper half of the slices' sums lie in LDS, 4 KB to a wave's tile of rows.
__host__ __device__ constexpr int sums_bytes(int waves, int tiles) { return waves / 2 * tiles * 4096; }
constexpr int kStepBytes = kMxTileBytes + 64;  // codes and scales of 16 rows, 128 columns
constexpr int kFloatSteps = 60;                // of them in LDS, of X quantised in the workgroup
constexpr int kFloatPanels = 192;              // a row's panels of k, over all rows: about a microsecond's work

// The tiles of X as they are held.
template <int NT>
struct HeldTiles {
  using Args = Mx4Matrix;
  static constexpr int kTiles = NT;
  static constexpr bool kFills = false;
  static constexpr int kWavesMax = kSlicesMax;
  // Four waves, or as many as there are slices.
  static constexpr int kLds = std::max(sums_bytes(4, NT), sums_bytes(std::min(kSlicesMax, kSumsMax / NT), NT));
  struct Raw { u32x4 codes[NT]; uint32_t scales; };
  const uint8_t *codes, *scales;
  uint32_t shift;
  __device__ __forceinline__ HeldTiles(const Mx4Matrix &m, const uint8_t *, int tile, int lane) {
    // NT tiles from `tile` on lie in one panel.
    const int64_t panel = (int64_t)(tile >> 2) * m.col_panels();
    codes = m.codes + panel * kMxPanelBytes + (tile & 3) * kMxTileBytes + lane * 16;
    scales = m.scales + panel * kMxPanelScales + lane * 4;
    shift = 8 * (tile & 3);
  }
  static __device__ __forceinline__ void fill(const Mx4Matrix &, uint8_t *, int) {}
  __device__ __forceinline__ void load(int k, Raw &r) const {
#pragma unroll
    for (int t = 0; t < NT; ++t) r.codes[t] = *reinterpret_cast<const u32x4 *>(codes + (int64_t)k * kMxPanelBytes + t * kMxTileBytes);
    r.scales = *reinterpret_cast<const uint32_t *>(scales + (int64_t)k * kMxPanelScales);
  }
  __device__ __forceinline__ uint32_t tiles(const Raw &r, int, u32x4 (&c)[NT]) const {
#pragma unroll
    for (int t = 0; t < NT; ++t) c[t] = r.codes[t];
    return r.scales >> shift;
  }
};

// A few rows of x's own values: every workgroup quantises all of them into LDS, 16 bytes to a thread at a
// time, which costs it less than a launch before this one does. Rows past the last hold anything.
struct FloatRows {
  const void *x;
  int64_t stride;
  int rows, cols;
};

template <int XDT, int NT>
struct FloatTiles {
  using Args = FloatRows;
  static constexpr int kTiles = NT;
  static constexpr bool kFills = true;
  static constexpr int kWavesMax = NT <= 2 ? 16 : 8;
  static constexpr int kLds = std::max(kFloatSteps * kStepBytes, sums_bytes(kWavesMax, NT));
  struct Raw {};
  const uint8_t *codes;
  __device__ __forceinline__ FloatTiles(const FloatRows &, const uint8_t *lds, int, int) : codes(lds) {}
  static __device__ __forceinline__ void fill(const FloatRows &a, uint8_t *lds, int kp) {
    using E = Elem<XDT>;
    constexpr int kBatch = 4, kBlockLanes = kMxBlock / E::kVec;
    const int row_lanes = kp * (kMxPanelCols / E::kVec), all = a.rows * row_lanes;
    const float per_row = 1.0f / (float)row_lanes;  // all < 2^13: (i + 1/2) / row_lanes has bits to spare
    auto row_of = [&](int i) { return (int)(((float)i + 0.5f) * per_row); };
    for (int first = (int)threadIdx.x; first < all; first += kBatch * (int)blockDim.x) {
      u32x4 raw[kBatch];
#pragma unroll
      for (int n = 0; n < kBatch; ++n) {
        const int i = first + n * (int)blockDim.x, r = row_of(i), col = (i - r * row_lanes) * E::kVec;
        raw[n] = i < all ? load_values<XDT, false>((const typename E::Bits *)a.x + (int64_t)r * a.stride, col, a.cols) : u32x4{0, 0, 0, 0};
      }
#pragma unroll
      for (int n = 0; n < kBatch; ++n) {
        const int i = first + n * (int)blockDim.x, r = row_of(i), at = i - r * row_lanes, b = at / kBlockLanes;
        if (i >= all) break;
        uint32_t word;
        const uint32_t s = encode_lane<XDT>(raw[n], word);
        uint8_t *to = lds + ((b >> 2) * NT + (r >> 4)) * kStepBytes;
        const int lane = (r & 15) + 16 * (b & 3);
        store_codes<E::kVec>(to + lane * 16 + at % kBlockLanes * (E::kVec / 2), word);
        if (at % kBlockLanes == 0) to[kMxTileBytes + lane] = (uint8_t)(b * kMxBlock < a.cols ? s : kMxScaleOne);
      }
    }
  }
  __device__ __forceinline__ void load(int, Raw &) const {}
  __device__ __forceinline__ uint32_t tiles(const Raw &, int k, u32x4 (&c)[NT]) const {
    const int lane = (int)threadIdx.x & 63;
    uint32_t scales = 0;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const uint8_t *at = codes + (k * NT + t) * kStepBytes;
      c[t] = *reinterpret_cast<const u32x4 *>(at + lane * 16);
      scales |= (uint32_t)at[kMxTileBytes + lane] << (8 * t);
    }
    return scales;
  }
};

template <int DT, typename Rows>
__global__ __launch_bounds__(Rows::kWavesMax * 64) void mx4_few_kernel(Mx4Product p, typename Rows::Args xs, FewShape shape) {
  constexpr int NT = Rows::kTiles;
  __shared__ __align__(16) uint8_t lds[Rows::kLds];
  const int lane = (int)threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int slice = wave & (shape.slices - 1);
  const int panel = (int)blockIdx.x * (shape.waves / shape.slices) + wave / shape.slices;
  const int kp = p.w.col_panels();
  const int tile = (int)blockIdx.y * NT;
  f32x4 acc[4][NT] = {};
  struct Step {
    u32x4 w[4];
    uint32_t sw;
    typename Rows::Raw x;
  };
  // A wave past the last panel has nothing to do but to meet the others.
  const bool works = panel * kMxPanelRows < p.w.rows;
  const Rows rows(xs, lds, tile, lane);
  const uint8_t *wc = p.w.codes + (int64_t)panel * kp * kMxPanelBytes + lane * 16;
  const uint8_t *ws = p.w.scales + (int64_t)panel * kp * kMxPanelScales + lane * 4;
  int k = (int)((int64_t)kp * slice / shape.slices);
  const int end = works ? (int)((int64_t)kp * (slice + 1) / shape.slices) : k;
  auto load = [&](int at, Step &s) {
#pragma unroll
    for (int t = 0; t < 4; ++t) s.w[t] = *reinterpret_cast<const u32x4 *>(wc + (int64_t)at * kMxPanelBytes + t * kMxTileBytes);
    s.sw = *reinterpret_cast<const uint32_t *>(ws + (int64_t)at * kMxPanelScales);
    rows.load(at, s.x);
  };
  auto multiply = [&](int at, const Step &s) {
    u32x4 x[NT];
    const uint32_t sx = rows.tiles(s.x, at, x);
    unrolled<4>([&](auto t) {
      unrolled<NT>([&](auto u) {
        constexpr int T = decltype(t)::value, U = decltype(u)::value;
        acc[T][U] = mx4_mfma<T, U>(s.w[T], x[U], acc[T][U], s.sw, sx);
      });
    });
  };
  // Three steps in registers: 128 x 4864, k = 4096 in 8.2 us, with two in 9.7. (The compiled copies between them wait
  // for the next step before the one after it is asked for: one is on its way during a step's products.)
  Step now, next, after;
  if (k < end) load(k, now);
  if (k + 1 < end) load(k + 1, next);
  if constexpr (Rows::kFills) {
    Rows::fill(xs, lds, kp);
    __syncthreads();
  }
  if (k < end) {
    for (; k + 2 < end; ++k) {
      load(k + 2, after);
      multiply(k, now);
      now = next;
      next = after;
    }
    multiply(k, now);
    if (k + 1 < end) multiply(k + 1, next);
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
    store_panel<DT>(p, (tile + u) * kMxTileRows + (lane & 15), panel * kMxPanelRows, acc[0][u], acc[1][u], acc[2][u], acc[3][u]);
}

constexpr int kCus = 256;             // an MI355X's compute units
constexpr int64_t kTilesMax = 1 << 22;  // of a launch: 2^32 threads are too many

// Whether W is streamed into registers: up to 64 rows, which one wave takes, and where tiles of 128 x 128
// would leave half the units idle (128 x 4864, k = 4096: 10.9 us in tiles, 8.2 so; 100 x 50257, k = 800, with
// 393 tiles: 14.4 and 18.4).
bool few_rows(int n, int rows) {
  return rows <= kMxPanelRows || mx_panels(n, 128) * mx_panels(rows, 128) <= kCus / 2;
}

template <int DT, int PM, int PN, int WM, int WN>
int launch_tiles(const Mx4Product &p, hipStream_t s) {
  const int64_t tiles_w = mx_panels(p.w.rows, kMxPanelRows * PM * WM), tiles_x = mx_panels(p.x.rows, kMxPanelRows * PN * WN);
  if (tiles_w * tiles_x > kTilesMax) return record_failure(TABBY_EINVAL, "the product is too large for one launch");
  hipLaunchKernelGGL((mx4_tile_kernel<DT, PM, PN, WM, WN>), dim3((unsigned)(tiles_w * tiles_x)), dim3(WM * WN * 64), 0, s, p,
                     (int)tiles_w, (int)tiles_x);
  TABBY_HIP_CHECK(hipGetLastError());
  return TABBY_OK;
}

// Whether tiles of 256 x 256 are the better choice, else 128 x 128. A unit holds one of the large tiles,
// and they do the same work in 3.5/4 of the time (4096 x 16384, k = 8192: 243 us and 270), but a last
// round of them that few units take part in costs as much as a full one: 318 x 44368, k = 6704: 86 us
// and 66; 2048 x 4096, k = 4096: 29 and 22.
bool large_tiles(int n, int rows) {
  const int64_t large = mx_panels(n, 256) * mx_panels(rows, 256), small = mx_panels(n, 128) * mx_panels(rows, 128);
  return 7 * mx_panels(large, kCus) <= 2 * mx_panels(small, kCus);
}

// The slices of k: enough waves to fill the chip, eight to a unit, while every one has a panel of k. A
// workgroup that quantises X does so for eight waves, or sixteen where slices make that many workgroups
// for most units (24 x 50257, k = 800 from f32: 12.3 us in eight, 10.1 in sixteen; 16 x 200000, k = 1024, a panel
// of W to a wave: 21.0 and 24.5).
template <typename Rows>
FewShape few_shape(int64_t panels, int kp) {
  int slices = 1;
  while (slices < kSlicesMax && slices * 2 <= kp && slices * 2 * Rows::kTiles <= kSumsMax && panels * slices < 8 * kCus) slices *= 2;
  if (!Rows::kFills) return {std::max(slices, 4), slices};
  const bool wide = Rows::kWavesMax == 16 && slices > 1 && panels * slices >= 16 * (kCus * 3 / 4);
  return {wide ? 16 : 8, slices};
}

template <int DT, typename Rows>
int launch_few(const Mx4Product &p, const typename Rows::Args &xs, hipStream_t s) {
  constexpr int NT = Rows::kTiles;
  const int64_t panels = mx_panels(p.w.rows, kMxPanelRows), groups = mx_panels(p.x.rows, kMxTileRows * NT);
  const FewShape shape = few_shape<Rows>(panels * groups, p.w.col_panels());
  const int64_t blocks = mx_panels(panels, shape.waves / shape.slices);
  hipLaunchKernelGGL((mx4_few_kernel<DT, Rows>), dim3((unsigned)blocks, (unsigned)groups), dim3(64 * shape.waves), 0, s, p, xs, shape);
  TABBY_HIP_CHECK(hipGetLastError());
  return TABBY_OK;
}

// X as it is held.
template <int DT>
int launch_product(const Mx4Product &p, hipStream_t s) {
  if (!few_rows(p.w.rows, p.x.rows)) return large_tiles(p.w.rows, p.x.rows) ? launch_tiles<DT, 2, 1, 2, 4>(p, s) : launch_tiles<DT, 1, 1, 2, 2>(p, s);
  const Mx4Matrix &xs = p.x;
  switch (mx_panels(p.x.rows, kMxTileRows)) {
    case 1: return launch_few<DT, HeldTiles<1>>(p, xs, s);
    case 2: return launch_few<DT, HeldTiles<2>>(p, xs, s);
    case 3: return launch_few<DT, HeldTiles<3>>(p, xs, s);
    default: return launch_few<DT, HeldTiles<4>>(p, xs, s);
  }
}

int product(const Mx4Product &p, int32_t out_dtype, hipStream_t s) {
  switch (out_dtype) {
    case TABBY_F32: return launch_product<TABBY_F32>(p, s);
    case TABBY_F16: return launch_product<TABBY_F16>(p, s);
    default: return launch_product<TABBY_BF16>(p, s);
  }
}

// X quantised in the product's own launch.
bool fills(int rows, int kp) {
  return rows <= kMxPanelRows && mx_panels(rows, kMxTileRows) * kp <= kFloatSteps && rows * kp <= kFloatPanels;
}

template <int DT, int XDT>
int launch_linear(const Mx4Product &p, const FloatRows &x, hipStream_t s) {
  switch (mx_panels(x.rows, kMxTileRows)) {
    case 1: return launch_few<DT, FloatTiles<XDT, 1>>(p, x, s);
    case 2: return launch_few<DT, FloatTiles<XDT, 2>>(p, x, s);
    case 3: return launch_few<DT, FloatTiles<XDT, 3>>(p, x, s);
    default: return launch_few<DT, FloatTiles<XDT, 4>>(p, x, s);
  }
}

template <int DT>
int launch_linear(const Mx4Product &p, const FloatRows &x, int x_dtype, hipStream_t s) {
  switch (x_dtype) {
    case TABBY_F32: return launch_linear<DT, TABBY_F32>(p, x, s);
    case TABBY_F16: return launch_linear<DT, TABBY_F16>(p, x, s);
    default: return launch_linear<DT, TABBY_BF16>(p, x, s);
  }
}

int linear(const Mx4Product &p, const FloatRows &x, int x_dtype, int32_t out_dtype, hipStream_t s) {
  switch (out_dtype) {
    case TABBY_F32: return launch_linear<TABBY_F32>(p, x, x_dtype, s);
    case TABBY_F16: return launch_linear<TABBY_F16>(p, x, x_dtype, s);
    default: return launch_linear<TABBY_BF16>(p, x, x_dtype, s);
  }
}

int check_output(const void *out, int32_t dtype, int32_t rows, int32_t n, int64_t stride) {
  if (!out) return record_failure(TABBY_EINVAL, "null pointer");
  if (!known_dtype(dtype)) return record_failure(TABBY_EINVAL, "dtype must be TABBY_F32, TABBY_F16 or TABBY_BF16");
  if (rows > 1 && stride < n) return record_failure(TABBY_EINVAL, "out_stride must be at least n");
  if ((uintptr_t)out % dtype_size(dtype) != 0) return record_failure(TABBY_EINVAL, "out must be aligned to its elements");
  return TABBY_OK;
}

// The rows apart from the weights and the bias.
int check_apart(const RowSpan &rows, const Mx4Product &p) {
  const int rc = check_mx4_apart(rows, p.w.codes, p.w.scales, p.w.rows, p.w.cols);
  if (rc) return rc;
  if (p.bias && rows_meet(rows, p.bias, (int64_t)p.w.rows * (int64_t)sizeof(float)))
    return record_failure(TABBY_EINVAL, "what a call writes must not overlap its bias");
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
  const RowSpan out = row_span(out_dev, rows, n, out_stride, dtype_size(out_dtype));
  rc = check_apart(out, p);
  if (!rc) rc = check_mx4_apart(out, x_codes_dev, x_scales_dev, rows, k);
  if (rc) return rc;
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
  const Mx4Product p{{(const uint8_t *)w_codes_dev, (const uint8_t *)w_scales_dev, n, k},
                     {codes, scales, rows, k}, bias_dev, out_dev, out_stride};
  const RowSpan x = row_span(x_dev, rows, k, x_stride, dtype_size(x_dtype));
  const RowSpan out = row_span(out_dev, rows, n, out_stride, dtype_size(out_dtype));
  rc = check_apart(out, p);
  if (!rc) rc = check_apart(row_span(workspace_dev, 1, code_bytes + scale_bytes, 0, 1), p);
  if (rc) return rc;
  if (rows_meet(out, workspace_dev, code_bytes + scale_bytes) || rows_meet(x, workspace_dev, code_bytes + scale_bytes))
    return record_failure(TABBY_EINVAL, "workspace must not overlap x or out");
  // A result that lies on x (a layer whose input and output share a buffer) is written after a launch that has read
  // all of x; in the product's own launch some workgroups would read what others have written.
  const bool apart = !rows_meet({out_dev, 1, out.bytes(), 0}, x_dev, x.bytes());
  if (apart && fills(rows, p.w.col_panels())) {
    return linear(p, FloatRows{x_dev, x_stride, rows, k}, x_dtype, out_dtype, (hipStream_t)stream);
  }
  rc = mx4_quantize(x_dev, x_dtype, rows, k, x_stride, codes, scales, (hipStream_t)stream);
  if (rc) return rc;
  return product(p, out_dtype, (hipStream_t)stream);
}
