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

}  // namespace tabby
