// Rows of BF16 or FP32 values as the kernels around a layer's experts read and write them.
#pragma once

#include "cfmoe_device.h"

namespace cfmoe {

// Values of a row type that one lane takes at a time: 16 bytes of them, or one where
// sizes or addresses do not allow whole vectors.
template <bool kFp32, bool kVector>
struct Lane {
  static constexpr int kValues = kVector ? (kFp32 ? 4 : 8) : 1;
};

// kValues values of a row at element `at`.
template <bool kFp32, bool kVector>
__device__ __forceinline__ void load_values(const void *row, int64_t at, float *v) {
  if constexpr (kFp32 && kVector) {
    const f32x4 a = *reinterpret_cast<const f32x4 *>(static_cast<const float *>(row) + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = a[i];
  } else if constexpr (kFp32) {
    v[0] = static_cast<const float *>(row)[at];
  } else if constexpr (kVector) {
    const u32x4 a = *reinterpret_cast<const u32x4 *>(static_cast<const uint16_t *>(row) + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(a[i] << 16);
      v[2 * i + 1] = __uint_as_float(a[i] & 0xffff0000u);
    }
  } else {
    v[0] = bf16_value(static_cast<const uint16_t *>(row)[at]);
  }
}

// Each value is rounded here, once, to the row's type.
template <bool kFp32, bool kVector>
__device__ __forceinline__ void store_values(void *row, int64_t at, const float *v) {
  if constexpr (kFp32 && kVector) {
    *reinterpret_cast<f32x4 *>(static_cast<float *>(row) + at) = f32x4{v[0], v[1], v[2], v[3]};
  } else if constexpr (kFp32) {
    static_cast<float *>(row)[at] = v[0];
  } else if constexpr (kVector) {
    *reinterpret_cast<u32x4 *>(static_cast<uint16_t *>(row) + at) =
        u32x4{bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3]), bf16_pair(v[4], v[5]), bf16_pair(v[6], v[7])};
  } else {
    static_cast<uint16_t *>(row)[at] = bf16_bits(v[0]);
  }
}

// Sum over the wave, in every lane, always in the same order.
__device__ __forceinline__ float wave_total(float v) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m);
  return v;
}

inline bool misaligned16(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 != 0; }

}  // namespace cfmoe
