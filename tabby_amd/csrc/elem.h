// The element types of the operators that take f32, f16 or bf16 alike, by tabby_dtype value: 16
// bytes widened to f32, one element read or written, rounding to nearest even on the way down.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "loads.h"
#include "tabby_sampler.h"

namespace tabby {

typedef u32x4 u32x4_any __attribute__((aligned(1)));  // rows of odd strides: the hardware takes any address

template <int DT>
struct Elem;

template <>
struct Elem<TABBY_F32> {
  using Bits = uint32_t;
  static constexpr int kVec = 4;  // elements in 16 bytes
  __device__ static float widen(uint32_t b) { return __uint_as_float(b); }
  __device__ static uint32_t narrow(float v) { return __float_as_uint(v); }
  __device__ static void widen16(u32x4 u, float (&v)[4]) { Widen<float, 4>::from(u, v); }
};

template <>
struct Elem<TABBY_F16> {
  using Bits = uint16_t;
  static constexpr int kVec = 8;
  __device__ static float widen(uint32_t b) { return half_bits_to_float(b); }
  __device__ static uint16_t narrow(float v) { return __builtin_bit_cast(uint16_t, (_Float16)v); }
  __device__ static void widen16(u32x4 u, float (&v)[8]) { Widen<uint16_t, 8>::from(u, v); }
};

template <>
struct Elem<TABBY_BF16> {
  using Bits = uint16_t;
  static constexpr int kVec = 8;
  __device__ static float widen(uint32_t b) { return __uint_as_float(b << 16); }
  __device__ static uint16_t narrow(float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }
  __device__ static void widen16(u32x4 u, float (&v)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
};

inline size_t dtype_size(int dtype) { return dtype == TABBY_F32 ? 4 : 2; }

inline bool known_dtype(int dtype) { return dtype == TABBY_F32 || dtype == TABBY_F16 || dtype == TABBY_BF16; }

}  // namespace tabby
