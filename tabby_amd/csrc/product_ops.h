// What the products of packed matrices have in common: Y [rows, n] stored from a wave's tiles of a 16-row matrix
// instruction, where a workgroup's tile lies, and the waits and loads of a pipeline of stages in LDS.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "abi_internal.h"
#include "elem.h"
#include "wave_ops.h"

namespace tabby {

constexpr int kProductCols = 64;  // columns of Y that a wave stores together: four tiles of 16

struct ProductOut {
  int rows, n;
  const float *bias;  // [n] or null
  void *out;
  int64_t stride;
};

// Four consecutive columns of one row of Y.
template <int DT>
__device__ __forceinline__ void store4(const ProductOut &p, int row, int col, f32x4 v) {
  using E = Elem<DT>;
  using Bits = typename E::Bits;
  const int n = p.n;
  if (row >= p.rows || col >= n) return;
  if (p.bias) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] += col + i < n ? p.bias[col + i] : 0.0f;
  }
  Bits *dst = (Bits *)p.out + (int64_t)row * p.stride + col;
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
__device__ __forceinline__ void store_panel(const ProductOut &p, int row, int col, f32x4 t0, f32x4 t1, f32x4 t2, f32x4 t3) {
  using E = Elem<DT>;
  using Bits = typename E::Bits;
  const int q = (int)(threadIdx.x & 63) >> 4;
  if (col + kProductCols > p.n) {
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
  if (row >= p.rows) return;
  Bits *dst = (Bits *)p.out + (int64_t)row * p.stride + col + 16 * q;
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

inline int check_output(const void *out, int32_t dtype, int32_t rows, int32_t n, int64_t stride) {
  if (!out) return record_failure(TABBY_EINVAL, "null pointer");
  if (!known_dtype(dtype)) return record_failure(TABBY_EINVAL, "dtype must be TABBY_F32, TABBY_F16 or TABBY_BF16");
  if (rows > 1 && stride < n) return record_failure(TABBY_EINVAL, "out_stride must be at least n");
  if ((uintptr_t)out % dtype_size(dtype) != 0) return record_failure(TABBY_EINVAL, "out must be aligned to its elements");
  return TABBY_OK;
}

}  // namespace tabby
