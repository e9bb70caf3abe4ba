// 8-bit floating point (e4m3: four exponent bits, three of the significand, no infinities, 448 the largest) with a
// float32 scale to each block: 128 columns of `block_rows` rows, 128 for weights and 1 for activations.
//
// Layout in HBM. Rows are padded to 64 and columns to 128, and each 64 x 128 panel is contiguous,
// panels in row-major order:
//   codes   8,192 bytes a panel: four 2 KB tiles of 16 rows, each two halves of 1 KB; in half h, 16 bytes at
//           16 * lane hold row lane % 16, columns 32 * (lane / 16) + 16 * h on;
//   scales  of square blocks: one to a block, blocks in row-major order; of blocks of one row: 64 a panel, one to a
//           row, panels in row-major order.
// That is an operand of the 16 x 16 x 128 matrix instruction, a lane's 32 codes of one row, as two 16-byte loads a lane, 1 KB
// contiguous to the wave each; copied to LDS as it lies, it is read back without bank conflicts. (Which 32 of a
// row's columns a lane holds does not matter as long as both operands agree.) Columns past the end hold code
// 0; rows past the end hold anything (they reach no result that is stored).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "elem.h"
#include "wave_ops.h"

namespace tabby {

constexpr int kF8Block = 128;        // columns to a scale, and rows of a square block
constexpr int kF8TileRows = 16;      // rows of one operand tile
constexpr int kF8PanelRows = 64;     // rows of a panel
constexpr int kF8PanelCols = 128;    // columns of a panel
constexpr int kF8TileBytes = 2048;   // codes of a tile
constexpr int kF8PanelBytes = 8192;  // codes of a panel
constexpr int kF8PanelScales = 256;  // bytes of a panel's scales, a row to each

__host__ __device__ __forceinline__ int64_t f8_parts(int64_t size, int64_t to) { return (size + to - 1) / to; }

struct Fp8Matrix {
  const uint8_t *codes;
  const float *scales;
  int rows, cols;
  __host__ __device__ int col_panels() const { return (cols + kF8PanelCols - 1) / kF8PanelCols; }
};

// A block's scale is the smallest power of two 2^E with max|x| <= 448 * 2^E, E at least -126 (a block of
// zeros: 1). A value's code is x / 2^E rounded to the nearest e4m3 value, ties to the even code; the division is
// exact but for values whose code is 0, so there is one rounding to a value. (A scale of max|x| / 448 would use up to a bit
// more of the range at the bottom, and round twice.) A block with a NaN or an infinity is NaN as a whole: its scale
// is NaN, its codes 0.

// The block's scale and what its values are multiplied by, from the largest magnitude's bits (f32).
__device__ __forceinline__ void f8_scale(uint32_t amax_bits, float &scale, float &inverse) {
  // 448 = 1.75 * 2^8: one power more where the significand is above 1.75.
  const int e = (int)(amax_bits >> 23) + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0) - 8;  // biased
  const int held = max(e, 1);
  scale = __uint_as_float((uint32_t)held << 23);
  inverse = __uint_as_float((uint32_t)(254 - held) << 23);
  if (amax_bits == 0) scale = inverse = 1.0f;
  if (amax_bits >= 0x7f800000u) {
    scale = __uint_as_float(0x7fc00000u);
    inverse = 0.0f;
  }
}

// The codes of four values that lie within the range.
__device__ __forceinline__ uint32_t f8_encode4(float a, float b, float c, float d) {
  int word = 0;
  word = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, word, false);
  word = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, word, true);
  return (uint32_t)word;
}

__device__ __forceinline__ void f8_decode4(uint32_t word, float *v) {
  const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)word, false);
  const auto b = __builtin_amdgcn_cvt_pk_f32_fp8((int)word, true);
  v[0] = a[0];
  v[1] = a[1];
  v[2] = b[0];
  v[3] = b[1];
}

// The largest magnitude of 16 bytes, as f32 bits; what is no number is larger than any.
template <int DT>
__device__ __forceinline__ uint32_t f8_largest(u32x4 raw) {
  using E = Elem<DT>;
  float v[E::kVec];
  E::widen16(raw, v);
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < E::kVec; ++j) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
  return top;
}

// The codes of 16 bytes, to LDS.
template <int DT>
__device__ __forceinline__ void f8_encode(uint8_t *to, u32x4 raw, float inverse) {
  using E = Elem<DT>;
  float v[E::kVec];
  E::widen16(raw, v);
  uint32_t word[E::kVec / 4];
#pragma unroll
  for (int i = 0; i < E::kVec / 4; ++i) {
    word[i] = f8_encode4(v[4 * i] * inverse, v[4 * i + 1] * inverse, v[4 * i + 2] * inverse, v[4 * i + 3] * inverse);
    if (inverse == 0.0f) word[i] = 0;  // a block that is NaN as a whole
  }
  if constexpr (E::kVec == 4) *reinterpret_cast<uint32_t *>(to) = word[0];
  else *reinterpret_cast<uint64_t *>(to) = word[0] | ((uint64_t)word[1] << 32);
}

// Where the code of row r, column c of a panel lies in it.
__device__ __forceinline__ int f8_code_byte(int r, int c) {
  return (r >> 4) * kF8TileBytes + ((c >> 4) & 1) * (kF8TileBytes / 2) + ((r & 15) + 16 * (c >> 5)) * 16 + (c & 15);
}

}  // namespace tabby
