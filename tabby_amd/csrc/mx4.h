// Microscaled 4-bit floating point (MXFP4): a row's columns in blocks of 32 values, each value a
// 4-bit e2m1 code (0, 1/2, 1, 3/2, 2, 3, 4, 6 and a sign), each block one power of two held as a
// biased 8-bit exponent (byte b stands for 2^(b - 127); 255: the block is NaN).
//
// Layout in HBM. Rows are padded to 64 and columns to 128, and each 64 x 128 panel is contiguous,
// panels in row-major order:
//   codes   4,096 bytes a panel: four 1 KB tiles of 16 rows; in a tile, 16 bytes (one block of one
//           row, two codes to a byte, the lower column in the low half) at 16 * lane, where
//           lane = row % 16 + 16 * (block within the panel);
//   scales  256 bytes a panel: byte 4 * lane + tile.
// That is the order in which a wave's 64 lanes hold the operand of a 16 x 16 x 128 scaled matrix
// instruction: one 16-byte load a lane brings a tile, 1 KB contiguous to the wave, and one 4-byte
// load brings the scales of four tiles, picked by the instruction's byte selectors. Copied to LDS
// as it lies, a tile is read back without bank conflicts. Columns past the end hold code 0 and
// exponent 127; rows past the end hold anything (they reach no result that is stored).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "elem.h"
#include "wave_ops.h"

namespace tabby {

constexpr int kMxBlock = 32;           // values to a scale
constexpr int kMxTileRows = 16;        // rows of one operand tile
constexpr int kMxPanelRows = 64;       // rows of a panel
constexpr int kMxPanelCols = 128;      // columns of a panel
constexpr int kMxTileBytes = 1024;     // codes of a tile
constexpr int kMxPanelBytes = 4096;    // codes of a panel
constexpr int kMxPanelScales = 256;    // scales of a panel
constexpr uint32_t kMxScaleOne = 127;  // 2^0
constexpr uint32_t kMxScaleNan = 255;

__host__ __device__ __forceinline__ int64_t mx_panels(int64_t size, int64_t to) { return (size + to - 1) / to; }

struct Mx4Matrix {
  const uint8_t *codes;
  const uint8_t *scales;
  int rows, cols;
  __host__ __device__ int col_panels() const { return (cols + kMxPanelCols - 1) / kMxPanelCols; }
};

// A block's exponent is E = floor(log2(max|x|)) - 2, the power of two that puts the largest value into [4, 8),
// held to [-127, 127] (a block of zeros: -127). A value's code is x / 2^E rounded to the nearest of the eight
// magnitudes, ties to the even code, and what lies above 6 becomes 6. A block with a NaN or an infinity is
// NaN as a whole, its codes 0. The rounding is the hardware's scaled conversion; the division by a power
// of two is exact, so there is one rounding to a value.

// The block's biased exponent from the largest magnitude's bits (f32).
__device__ __forceinline__ uint32_t block_scale(uint32_t amax_bits) {
  if (amax_bits >= 0x7f800000u) return kMxScaleNan;
  const int e = (int)(amax_bits >> 23) - 2;  // a subnormal's field is 0: below the range all the same
  return (uint32_t)max(e, 0);
}

// The codes of N = 4 or 8 values, two to a byte.
template <int N>
__device__ __forceinline__ uint32_t encode_values(const float *v, float scale) {
  uint32_t word = 0;
  word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[0], v[1], scale, 0);
  word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[2], v[3], scale, 1);
  if constexpr (N == 8) {
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[4], v[5], scale, 2);
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[6], v[7], scale, 3);
  }
  return word;
}

template <int N>
__device__ __forceinline__ void decode_values(uint32_t word, uint32_t s, float *v) {
  const float scale = __uint_as_float(s << 23);
  const auto a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, scale, 0);
  const auto b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, scale, 1);
  v[0] = a[0];
  v[1] = a[1];
  v[2] = b[0];
  v[3] = b[1];
  if constexpr (N == 8) {
    const auto c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, scale, 2);
    const auto d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, scale, 3);
    v[4] = c[0];
    v[5] = c[1];
    v[6] = d[0];
    v[7] = d[1];
  }
  if (s == kMxScaleNan) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = __uint_as_float(0x7fc00000u);
  }
}

// The codes of a lane's 16 bytes, whose block lies in neighbouring lanes, and the block's biased exponent.
template <int DT>
__device__ __forceinline__ uint32_t encode_lane(u32x4 raw, uint32_t &codes) {
  using E = Elem<DT>;
  float v[E::kVec];
  E::widen16(raw, v);
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < E::kVec; ++j) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
#pragma unroll
  for (int lanes = 1; lanes < kMxBlock / E::kVec; lanes *= 2) top = max(top, xor_lane_by(top, lanes));
  const uint32_t s = block_scale(top);
  codes = s != kMxScaleNan ? encode_values<E::kVec>(v, __uint_as_float(s << 23)) : 0u;
  return s;
}

// N codes, two to a byte.
template <int N>
__device__ __forceinline__ void store_codes(uint8_t *to, uint32_t word) {
  if constexpr (N == 4) *reinterpret_cast<uint16_t *>(to) = (uint16_t)word;
  else *reinterpret_cast<uint32_t *>(to) = word;
}

}  // namespace tabby
