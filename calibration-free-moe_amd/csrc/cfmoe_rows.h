// Rows of BF16 or FP32 values as the kernels around a layer's experts read and write them.
#pragma once

#include <type_traits>

#include "cfmoe_device.h"

namespace cfmoe {

// 16 bytes at any address of 4-byte or 2-byte values.
typedef uint32_t vector_of_4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t vector_of_2 __attribute__((ext_vector_type(4), aligned(2)));

// What one lane takes of a row at a time: 16 bytes, or one value of rows that are shorter.
// Memory takes 16 bytes from any value's address, so that rows need no alignment of their
// own. A row's last lane takes its last 16 bytes: where the row is no whole number of them,
// it has values that the lane before has too, which stores them alike and is the one that
// counts them in a sum. kOnce is for what no later load finds in a cache.
enum Rows { kSingle, kWhole, kRagged };

template <bool kFp32, Rows kRows>
struct Lane {
  using Value = std::conditional_t<kFp32, float, uint16_t>;
  using Raw = std::conditional_t<kRows != kSingle, u32x4, Value>;
  static constexpr int kValues = kRows != kSingle ? (kFp32 ? 4 : 8) : 1;

  // First element of the lane whose values would begin at `column` (the row's last ones past
  // its end), and how many of the values from there are another lane's.
  static __device__ __forceinline__ int first(int column, int size) { return min(column, size - kValues); }
  static __device__ __forceinline__ int others(int column, int size) { return column - first(column, size); }

  template <bool kOnce = false>
  static __device__ __forceinline__ Raw load(const void *row, int64_t at) {
    const Value *from = static_cast<const Value *>(row) + at;
    // (the types by name: as a template's argument they would lose their alignment)
    if constexpr (kRows == kSingle) {
      return *from;
    } else if constexpr (kFp32) {
      const vector_of_4 *p = reinterpret_cast<const vector_of_4 *>(from);
      return kOnce ? __builtin_nontemporal_load(p) : *p;
    } else {
      const vector_of_2 *p = reinterpret_cast<const vector_of_2 *>(from);
      return kOnce ? __builtin_nontemporal_load(p) : *p;
    }
  }

  static __device__ __forceinline__ void values(Raw raw, float *v) {
    if constexpr (kFp32 && kRows != kSingle) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(raw[i]);
    } else if constexpr (kRows != kSingle) {
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

  // Each value is rounded here, once, to the row's type.
  static __device__ __forceinline__ void store(void *row, int64_t at, const float *v) {
    Raw raw;
    if constexpr (kFp32 && kRows != kSingle) {
#pragma unroll
      for (int i = 0; i < 4; ++i) raw[i] = __float_as_uint(v[i]);
    } else if constexpr (kRows != kSingle) {
#pragma unroll
      for (int i = 0; i < 4; ++i) raw[i] = bf16_pair(v[2 * i], v[2 * i + 1]);
    } else if constexpr (kFp32) {
      raw = v[0];
    } else {
      raw = bf16_bits(v[0]);
    }
    Value *to = static_cast<Value *>(row) + at;
    if constexpr (kRows == kSingle) *to = raw;
    else if constexpr (kFp32) *reinterpret_cast<vector_of_4 *>(to) = raw;
    else *reinterpret_cast<vector_of_2 *>(to) = raw;
  }
};

inline Rows rows_of(int size, bool fp32) {
  const int values = fp32 ? 4 : 8;
  return size < values ? kSingle : size % values ? kRagged : kWhole;
}

template <int kControl, int kLanes = 0xf>
__device__ __forceinline__ float lane_moved(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), kControl, kLanes, 0xf, false));
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

// What lanes of a wave wrote to LDS before is what its lanes read after: their accesses are
// done in order, and the compiler keeps them so. No instruction of its own.
__device__ __forceinline__ void wave_in_step() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

inline bool misaligned16(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 != 0; }

}  // namespace cfmoe
