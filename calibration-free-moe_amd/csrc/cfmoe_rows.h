// Rows of BF16 or FP32 values as the kernels around a layer's experts read and write them.
#pragma once

#include <type_traits>

#include "cfmoe_device.h"

namespace cfmoe {

template <bool kOnce, typename T>
__device__ __forceinline__ T load_from(const T *p) {
  return kOnce ? __builtin_nontemporal_load(p) : *p;
}

template <bool kOnce, typename T>
__device__ __forceinline__ void store_to(T *p, T v) {
  if (kOnce) __builtin_nontemporal_store(v, p);
  else *p = v;
}

// What one lane takes of a row at a time: 16 bytes, or one value where sizes or addresses
// do not allow whole vectors. kOnce is for what no later load finds in a cache.
template <bool kFp32, bool kVector>
struct Lane {
  using Value = std::conditional_t<kFp32, float, uint16_t>;
  using Raw = std::conditional_t<kVector, u32x4, Value>;
  static constexpr int kValues = kVector ? (kFp32 ? 4 : 8) : 1;

  template <bool kOnce = false>
  static __device__ __forceinline__ Raw load(const void *row, int64_t at) {
    return load_from<kOnce>(reinterpret_cast<const Raw *>(static_cast<const Value *>(row) + at));
  }

  static __device__ __forceinline__ void values(Raw raw, float *v) {
    if constexpr (kFp32 && kVector) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(raw[i]);
    } else if constexpr (kVector) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(raw[i] << 16);
        v[2 * i + 1] = __uint_as_float(raw[i] & 0xffff0000u);
      }
    } else if constexpr (kFp32) {
      v[0] = raw;
    } else {
      v[0] = bf16_value(raw);
    }
  }
};

// The values of a row from element `at`.
template <bool kFp32, bool kVector, bool kOnce = false>
__device__ __forceinline__ void load_values(const void *row, int64_t at, float *v) {
  Lane<kFp32, kVector>::values(Lane<kFp32, kVector>::template load<kOnce>(row, at), v);
}

// Each value is rounded here, once, to the row's type.
template <bool kFp32, bool kVector, bool kOnce = false>
__device__ __forceinline__ void store_values(void *row, int64_t at, const float *v) {
  if constexpr (kFp32 && kVector) {
    store_to<kOnce>(reinterpret_cast<f32x4 *>(static_cast<float *>(row) + at), f32x4{v[0], v[1], v[2], v[3]});
  } else if constexpr (kFp32) {
    store_to<kOnce>(static_cast<float *>(row) + at, v[0]);
  } else if constexpr (kVector) {
    store_to<kOnce>(reinterpret_cast<u32x4 *>(static_cast<uint16_t *>(row) + at),
                    u32x4{bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3]), bf16_pair(v[4], v[5]), bf16_pair(v[6], v[7])});
  } else {
    store_to<kOnce>(static_cast<uint16_t *>(row) + at, bf16_bits(v[0]));
  }
}

template <int kControl, int kRows = 0xf>
__device__ __forceinline__ float lane_moved(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), kControl, kRows, 0xf, false));
}

// Sum over the wave, the same in every lane, always in the same order: pairs, quads, halves
// and rows of 16 lanes by lane moves, then the rows one after the other.
__device__ __forceinline__ float wave_total(float v) {
  v += lane_moved<0xb1>(v);
  v += lane_moved<0x4e>(v);
  v += lane_moved<0x141>(v);
  v += lane_moved<0x140>(v);
  v += lane_moved<0x142, 0xa>(v);  // last lane of the row before, into rows 1 and 3
  v += lane_moved<0x143, 0xc>(v);  // last lane of row 1, into rows 2 and 3
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

inline bool misaligned16(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 != 0; }

}  // namespace cfmoe
