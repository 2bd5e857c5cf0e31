// Device helpers shared by the router, whole-layer and 4-bit kernels.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "cfmoe_reader.h"

namespace cfmoe {

int fail(int code, const char *message);
int check_launch(const char *stage);

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ float bf16_value(uint32_t half) { return __uint_as_float(half << 16); }

// Two FP32 values to BF16, to nearest even, NaN kept quiet; `low` in the low half.
__device__ __forceinline__ uint32_t bf16_pair(float low, float high) {
  bf16x2 v;
  v.x = static_cast<__bf16>(low);
  v.y = static_cast<__bf16>(high);
  return __builtin_bit_cast(uint32_t, v);
}

__device__ __forceinline__ uint16_t bf16_bits(float v) {
  return __builtin_bit_cast(uint16_t, static_cast<__bf16>(v));
}

// D += A B of one 16 x 16 tile over 32 products. Lane l holds A[l % 16][8 (l /
// 16) ..] and B[8 (l / 16) ..][l % 16]; D[4 (l / 16) + r][l % 16] is its d[r].
__device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 d) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                 __builtin_bit_cast(bf16x8, b), d, 0, 0, 0);
}

// Eight E2M1 codes (even elements in the low nibbles) times 2^(byte - 127), in
// BF16. The conversion reads only the scale's exponent bits, so that byte << 23
// stands for every E8M0 byte: 0 is 2^-127 and 255 makes the values NaN.
__device__ __forceinline__ u32x4 fp4_values(uint32_t codes, float scale) {
  u32x4 v;
  v.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0));
  v.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1));
  v.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2));
  v.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3));
  return v;
}

}  // namespace cfmoe
