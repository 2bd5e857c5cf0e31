// MI355X (gfx950) microscaled 4-bit floating point: quantisation and values.
//
// A block of 32 values v shares one E8M0 scale X = 2^(byte - 127) and holds each
// value as a 4-bit E2M1 number:
//   byte = clamp(floor(log2 max|v|) - 2 + 127, 2, 254)  (2 = the largest exponent of E2M1)
//   code = sign, and |v| / X to the nearest of 0, .5, 1, 1.5, 2, 3, 4, 6, ties to
//          the even mantissa, 6 for what is larger
// Bytes start at 2 so that every nonzero value X e2m1 is a normal BF16 number. A
// block that holds a NaN or an infinity gets byte 255 (NaN) and zero codes: it
// reads back as NaN, not as finite values that were never there. Element 2 i of a
// row sits in the low nibble of byte i, element 2 i + 1 in the high one.

#include "cfmoe_device.h"

namespace cfmoe {
namespace {

constexpr int kThreads = 256;
constexpr int kLaneValues = 8;   // values of one lane; four lanes hold a block
constexpr int kInfinity = 0x7f800000;

template <int kControl>
__device__ __forceinline__ int quad_max(int v) {
  return max(v, __builtin_amdgcn_mov_dpp(v, kControl, 0xf, 0xf, true));
}

// Lane = eight values of a block, a quad of lanes = the block; largest |v| by
// integer compare of the bits (a NaN's are above infinity's). One pass at the rate of
// memory: 403 M values 170 to 189 us from BF16 (1.02 GB, 5.4 to 6.0 TB/s), 323 from FP32
// (1.83 GB, 5.7 TB/s). A small call is its launch: 2.8 us for 2.1 M values.
template <bool kFp32>
__global__ __launch_bounds__(kThreads) void quantise_fp4_kernel(const void *weights, uint32_t *codes,
                                                                uint8_t *scales, int64_t lanes) {
  const int64_t step = static_cast<int64_t>(gridDim.x) * kThreads;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < lanes; i += step) {
    float v[kLaneValues];
    if (kFp32) {
      const f32x4 *row = reinterpret_cast<const f32x4 *>(weights) + 2 * i;
      const f32x4 a = row[0], b = row[1];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = a[j], v[4 + j] = b[j];
    } else {
      const u32x4 a = reinterpret_cast<const u32x4 *>(weights)[i];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[2 * j] = bf16_value(a[j] & 0xffffu);
        v[2 * j + 1] = __uint_as_float(a[j] & 0xffff0000u);
      }
    }
    int largest = 0;
#pragma unroll
    for (int j = 0; j < kLaneValues; ++j) largest = max(largest, __float_as_int(v[j]) & 0x7fffffff);
    largest = quad_max<0x4e>(quad_max<0xb1>(largest));
    const bool finite = largest < kInfinity;
    const int byte = finite ? max((largest >> 23) - 2, 2) : 255;
    const float scale = __int_as_float(byte << 23);
    uint32_t word = 0;
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[0], v[1], scale, 0);
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[2], v[3], scale, 1);
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[4], v[5], scale, 2);
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[6], v[7], scale, 3);
    codes[i] = finite ? word : 0u;
    if (threadIdx.x % 4 == 0) scales[i / 4] = static_cast<uint8_t>(byte);
  }
}

// 403 M values 174 to 183 us (1.02 GB, 5.6 to 5.9 TB/s).
__global__ __launch_bounds__(kThreads) void dequantise_fp4_kernel(const uint32_t *codes,
                                                                  const uint8_t *scales, u32x4 *values,
                                                                  int64_t lanes) {
  const int64_t step = static_cast<int64_t>(gridDim.x) * kThreads;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < lanes; i += step)
    values[i] = fp4_values(codes[i], __int_as_float(static_cast<int>(scales[i / 4]) << 23));
}

unsigned grid_of(int64_t lanes) {
  const int64_t groups = (lanes + kThreads - 1) / kThreads;
  return static_cast<unsigned>(groups < (1 << 20) ? groups : (1 << 20));
}

bool misaligned(const void *p, unsigned bytes) { return reinterpret_cast<uintptr_t>(p) % bytes != 0; }

}  // namespace
}  // namespace cfmoe

extern "C" {

using namespace cfmoe;

CFMOE_API int cfmoe_quantise_fp4(int64_t blocks, uint32_t flags, const void *weights, void *codes,
                                 uint8_t *scales, cfmoe_stream stream) {
  if (blocks < 0 || blocks > (INT64_C(1) << 40)) return fail(CFMOE_EINVAL, "quantise_fp4 needs 0 to 2^40 blocks");
  if (blocks == 0) return 0;
  if (!weights || !codes || !scales) return fail(CFMOE_EINVAL, "NULL argument");
  if (misaligned(weights, 16) || misaligned(codes, 4))
    return fail(CFMOE_EINVAL, "quantise_fp4 needs 16-byte aligned weights and 4-byte aligned codes");
  const int64_t lanes = 4 * blocks;
  auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(grid_of(lanes)), dim3(kThreads), 0, stream, weights,
                       static_cast<uint32_t *>(codes), scales, lanes);
  };
  launch(flags & CFMOE_FP32 ? quantise_fp4_kernel<true> : quantise_fp4_kernel<false>);
  return check_launch("quantise_fp4");
}

CFMOE_API int cfmoe_dequantise_fp4(int64_t blocks, const void *codes, const uint8_t *scales, void *values,
                                   cfmoe_stream stream) {
  if (blocks < 0 || blocks > (INT64_C(1) << 40)) return fail(CFMOE_EINVAL, "dequantise_fp4 needs 0 to 2^40 blocks");
  if (blocks == 0) return 0;
  if (!codes || !scales || !values) return fail(CFMOE_EINVAL, "NULL argument");
  if (misaligned(values, 16) || misaligned(codes, 4))
    return fail(CFMOE_EINVAL, "dequantise_fp4 needs 16-byte aligned values and 4-byte aligned codes");
  const int64_t lanes = 4 * blocks;
  hipLaunchKernelGGL(dequantise_fp4_kernel, dim3(grid_of(lanes)), dim3(kThreads), 0, stream,
                     static_cast<const uint32_t *>(codes), scales, static_cast<u32x4 *>(values), lanes);
  return check_launch("dequantise_fp4");
}

}  // extern "C"
