// MI355X (gfx950): low-rank adapters of many requests beside a shared projection.
//
//   out[t] = base[t] + s_a D_a (C_a x[t])        a = slots[t]
//
// with C_a [R, H] and D_a [O, R] of the adapter that token t's request has, s_a its scale;
// a token whose slot names none keeps its row of `base`, bit for bit.
//
// Tokens of one adapter share its weights: they form tiles, and a tile's products are
// matrix instructions, C_a x over the hidden dimension (adapter_inner_kernel, waves share
// it and add up in LDS) and D_a v over the rank (adapter_out_kernel). A decode step's tiles
// hold a token or two, which leaves most columns of an instruction empty: what bounds it
// is the weights' reading, once for each tile.
//
// v = s_a C_a x is FP32 in memory between the two. As operand of the second product it is
// the sum of two BF16 numbers (2^-16 off: the first cut off, so that the second has its
// sign and an infinite weight meets no zero where v is not one), and out is rounded once.

#include "cfmoe_rows.h"

namespace cfmoe {
namespace {

constexpr int kMaxAdapters = 4096;
constexpr int kMaxRank = 256;
constexpr int kMaxSize = 65536;
constexpr int kInnerTokens = 16;  // of a tile of the first product
constexpr int kInnerWaves = 16;
constexpr int kOutWaves = 4;
constexpr int kOutColumns = 64;   // outputs of one wave
constexpr int kFewTokens = 1024;  // up to which a workgroup finds its tile by itself

struct AdapterArgs {
  const uint16_t *base, *x, *encoder, *decoder;
  const void *slots;
  const float *scales;
  uint16_t *out;
  float *inner;            // [T, R]
  const int32_t *offsets;  // [N + 1] and
  const int32_t *pairs;    // [T]: tokens by adapter (many tokens only)
  int64_t base_stride, x_stride, out_stride;
  int tokens, hidden, outputs, rank, adapters;
  bool slots64;
};

// The adapter of a token; `adapters` where its slot names none.
__device__ __forceinline__ int slot_of(const AdapterArgs &a, int t) {
  const int64_t s = a.slots64 ? static_cast<const int64_t *>(a.slots)[t] : static_cast<const int32_t *>(a.slots)[t];
  return s >= 0 && s < a.adapters ? static_cast<int>(s) : a.adapters;
}

// Tokens of one adapter, up to kTile: tile `index` of the call. False for a workgroup that
// has none. Few tokens (kSorted false): tile t is led by token t, if a whole number of
// tiles' tokens of its adapter come before it; the workgroup reads all slots. Many: the
// tokens are sorted, and the tile is found from the adapters' offsets. All threads of the
// workgroup call it; it ends with a barrier.
template <bool kSorted, int kTile, int kWaves>
__device__ __forceinline__ bool find_tile(const AdapterArgs &a, int index, int *members, int &adapter, int &count) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if constexpr (kSorted) {
    int before = 0;  // tiles of earlier adapters
    for (int first = 0; first <= a.adapters; first += 64) {
      const int n = first + lane;
      int from = 0, to = 0;
      if (n <= a.adapters) {
        from = a.offsets[n];
        to = n < a.adapters ? a.offsets[n + 1] : a.tokens;
      }
      const int tiles = (to - from + kTile - 1) / kTile;
      int scan = tiles;
#pragma unroll
      for (int m = 1; m < 64; m <<= 1) {
        const int below = __shfl_up(scan, m);
        if (lane >= m) scan += below;
      }
      const uint64_t past = __ballot(before + scan > index);
      if (past) {
        const int owner = __builtin_ctzll(past);
        const int start = __shfl(from, owner) + (index - before - __shfl(scan - tiles, owner)) * kTile;
        adapter = __builtin_amdgcn_readfirstlane(first + owner);
        count = __builtin_amdgcn_readfirstlane(min(kTile, __shfl(to, owner) - start));
        for (int i = threadIdx.x; i < count; i += 64 * kWaves) members[i] = a.pairs[start + i];
        __syncthreads();
        return true;
      }
      before += __shfl(scan, 63);
    }
    return false;
  } else {
    __shared__ uint64_t masks[kFewTokens / 64];
    adapter = __builtin_amdgcn_readfirstlane(slot_of(a, index));
    for (int first = wave * 64; first < a.tokens; first += 64 * kWaves) {
      const int t = first + lane;
      const uint64_t same = __ballot(t < a.tokens && slot_of(a, t) == adapter);
      if (lane == 0) masks[first / 64] = same;
    }
    __syncthreads();
    int before = 0;
    for (int w = 0; w < index / 64; ++w) before += __builtin_popcountll(masks[w]);
    before += __builtin_popcountll(masks[index / 64] & ((UINT64_C(1) << (index % 64)) - 1));
    if (before % kTile) return false;
    // each token from `index` on takes its place
    int total = before;
    for (int w = index / 64; w < (a.tokens + 63) / 64; ++w) total += __builtin_popcountll(w == index / 64 ? masks[w] >> (index % 64) : masks[w]);
    count = min(kTile, total - before);
    int place = 0;
    for (int w = 0; w < (a.tokens + 63) / 64; ++w) {
      if (w % kWaves == wave && (masks[w] >> lane) & 1) {
        const int rank = place + __builtin_popcountll(masks[w] & ((UINT64_C(1) << lane) - 1)) - before;
        if (rank >= 0 && rank < kTile) members[rank] = 64 * w + lane;
      }
      place += __builtin_popcountll(masks[w]);
    }
    __syncthreads();
    return true;
  }
}

__device__ __forceinline__ u32x4 load16(const uint16_t *p) { return *reinterpret_cast<const u32x4 *>(p); }

// inner[t, r] = s sum_h C[r, h] x[t, h] for a tile of 16 tokens and kTiles tiles of 16
// ranks. The waves take the hidden dimension in turns of 64; a lane's operands are 16
// values that follow one another (the order of products in a sum is free, and both
// operands have the same), so that four lanes read 128 bytes of a row.
template <bool kSorted, int kTiles>
__global__ __launch_bounds__(64 * kInnerWaves) void adapter_inner_kernel(AdapterArgs a) {
  __shared__ int members[kInnerTokens];
  __shared__ float sums[kInnerWaves][kTiles][256];
  int adapter, count;
  if (!find_tile<kSorted, kInnerTokens, kInnerWaves>(a, blockIdx.x, members, adapter, count)) return;
  if (adapter >= a.adapters) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m = lane & 15, q = lane >> 4;
  const int r0 = blockIdx.y * 16 * kTiles;
  const uint16_t *x = a.x + members[min(m, count - 1)] * a.x_stride;
  const uint16_t *c[kTiles];
#pragma unroll
  for (int i = 0; i < kTiles; ++i)
    c[i] = a.encoder + (static_cast<int64_t>(adapter) * a.rank + min(r0 + 16 * i + m, a.rank - 1)) * a.hidden;
  f32x4 d[kTiles] = {};
  for (int h = 64 * wave + 16 * q; h - 16 * q < a.hidden; h += 64 * kInnerWaves) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const bool in = h + 8 * s < a.hidden;
      const u32x4 zero = {0, 0, 0, 0};
      const u32x4 xv = in ? load16(x + h + 8 * s) : zero;
#pragma unroll
      for (int i = 0; i < kTiles; ++i) d[i] = mma(in ? load16(c[i] + h + 8 * s) : zero, xv, d[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < kTiles; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) sums[wave][i][m * 16 + 4 * q + r] = d[i][r];
  __syncthreads();
  const float scale = a.scales ? a.scales[adapter] : 1.0f;
  for (int i = threadIdx.x; i < 256 * kTiles; i += 64 * kInnerWaves) {
    const int tile = i / 256, token = i % 256 / 16, r = r0 + 16 * tile + i % 16;
    if (token >= count || r >= a.rank) continue;
    float total = 0.0f;
#pragma unroll
    for (int w = 0; w < kInnerWaves; ++w) total += sums[w][tile][i % 256];
    a.inner[static_cast<int64_t>(members[token]) * a.rank + r] = scale * total;
  }
}

// Two BF16 numbers whose sum is v to 2^-16, the first cut off: high and low halves of eight.
__device__ __forceinline__ void split(const float *v, u32x4 &high, u32x4 &low) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t a = __float_as_uint(v[2 * i]) & 0xffff0000u, b = __float_as_uint(v[2 * i + 1]) & 0xffff0000u;
    high[i] = a >> 16 | b;
    low[i] = bf16_pair(v[2 * i] - __uint_as_float(a), v[2 * i + 1] - __uint_as_float(b));
  }
}

// out = base + D v for a tile of tokens, a wave 64 outputs of them. Row 4 q + r of the i-th
// matrix tile is output 16 q + 4 i + r, so that a lane ends with 16 outputs that follow one
// another, and four lanes with 128 bytes of a row.
template <bool kSorted, int kGroups>
__global__ __launch_bounds__(64 * kOutWaves) void adapter_out_kernel(AdapterArgs a) {
  __shared__ int members[16 * kGroups];
  int adapter, count;
  if (!find_tile<kSorted, 16 * kGroups, kOutWaves>(a, blockIdx.x, members, adapter, count)) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m = lane & 15, q = lane >> 4;
  const int o0 = (blockIdx.y * kOutWaves + wave) * kOutColumns;
  if (o0 >= a.outputs) return;
  const bool bare = adapter >= a.adapters;
  if (bare && a.out == a.base) return;
  const uint16_t *d[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    d[i] = a.decoder + (static_cast<int64_t>(bare ? 0 : adapter) * a.outputs + min(o0 + m / 4 * 16 + 4 * i + m % 4, a.outputs - 1)) * a.rank;
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    if (16 * g >= count) break;
    const int64_t t = members[min(16 * g + m, count - 1)];
    f32x4 sum[4] = {};
    if (!bare) {
      for (int k = 8 * q; k - 8 * q < a.rank; k += 32) {
        const bool in = k < a.rank;
        u32x4 high = {0, 0, 0, 0}, low = {0, 0, 0, 0};
        if (in) {
          float v[8];
          load_values<true, true>(a.inner, t * a.rank + k, v);
          load_values<true, true>(a.inner, t * a.rank + k + 4, v + 4);
          split(v, high, low);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const u32x4 w = in ? load16(d[i] + k) : u32x4{0, 0, 0, 0};
          sum[i] = mma(w, low, mma(w, high, sum[i]));
        }
      }
    }
    if (16 * g + m >= count) continue;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int o = o0 + 16 * q + 8 * s;
      if (o >= a.outputs) continue;
      u32x4 row = load16(a.base + t * a.base_stride + o);
      if (!bare) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[2 * i] = __uint_as_float(row[i] << 16) + sum[2 * s + i / 2][2 * i % 4];
          v[2 * i + 1] = __uint_as_float(row[i] & 0xffff0000u) + sum[2 * s + i / 2][2 * i % 4 + 1];
        }
        row = u32x4{bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3]), bf16_pair(v[4], v[5]), bf16_pair(v[6], v[7])};
      }
      *reinterpret_cast<u32x4 *>(a.out + t * a.out_stride + o) = row;
    }
  }
}

int64_t rounded(int64_t bytes) { return (bytes + 15) / 16 * 16; }

bool sorts(int tokens) { return tokens > kFewTokens; }

}  // namespace
}  // namespace cfmoe

extern "C" {

using namespace cfmoe;

CFMOE_API int64_t cfmoe_apply_adapters_scratch_bytes(int32_t rank, int32_t adapters, int32_t tokens) {
  if (rank < 8 || rank > kMaxRank || rank % 8) return -fail(CFMOE_EINVAL, "apply_adapters needs a rank that is a multiple of 8, at most 256");
  if (adapters < 1 || adapters > kMaxAdapters) return -fail(CFMOE_EINVAL, "apply_adapters needs 1 to 4096 adapters");
  if (tokens < 0 || tokens > (1 << 24)) return -fail(CFMOE_EINVAL, "apply_adapters needs 0 to 2^24 tokens");
  int64_t bytes = static_cast<int64_t>(tokens) * rank * 4;
  if (sorts(tokens))
    bytes += rounded(4 * (adapters + 1)) + 2 * rounded(4 * static_cast<int64_t>(tokens)) +
             cfmoe_sort_by_expert_scratch_bytes(tokens, 1, adapters);
  return bytes;
}

CFMOE_API int cfmoe_apply_adapters(int32_t hidden_size, int32_t outputs, int32_t rank, int32_t adapters, uint32_t flags,
                                   const void *base, int64_t base_stride, const void *hidden, int64_t hidden_stride,
                                   const void *encoder, const void *decoder, const void *slots, const float *scales,
                                   void *out, int64_t out_stride, void *scratch, int32_t tokens, cfmoe_stream stream) {
  const int64_t bytes = cfmoe_apply_adapters_scratch_bytes(rank, adapters, tokens);
  if (bytes < 0) return static_cast<int>(-bytes);
  if (hidden_size < 8 || hidden_size > kMaxSize || hidden_size % 8 || outputs < 8 || outputs > kMaxSize || outputs % 8)
    return fail(CFMOE_EINVAL, "apply_adapters needs hidden and output sizes that are multiples of 8, at most 65536");
  if (base_stride % 8 || hidden_stride % 8 || out_stride % 8 || base_stride < 0 || hidden_stride < 0 || out_stride < outputs)
    return fail(CFMOE_EINVAL, "apply_adapters needs row strides that are multiples of 8");
  if (tokens == 0) return 0;
  if (!base || !hidden || !encoder || !decoder || !slots || !out || !scratch) return fail(CFMOE_EINVAL, "NULL argument");
  if (misaligned16(base) || misaligned16(hidden) || misaligned16(encoder) || misaligned16(decoder) || misaligned16(out) ||
      misaligned16(scratch))
    return fail(CFMOE_EINVAL, "apply_adapters needs 16-byte aligned rows, weights and scratch");
  AdapterArgs a = {};
  a.base = static_cast<const uint16_t *>(base);
  a.x = static_cast<const uint16_t *>(hidden);
  a.encoder = static_cast<const uint16_t *>(encoder);
  a.decoder = static_cast<const uint16_t *>(decoder);
  a.slots = slots;
  a.scales = scales;
  a.out = static_cast<uint16_t *>(out);
  a.inner = static_cast<float *>(scratch);
  a.base_stride = base_stride;
  a.x_stride = hidden_stride;
  a.out_stride = out_stride;
  a.tokens = tokens;
  a.hidden = hidden_size;
  a.outputs = outputs;
  a.rank = rank;
  a.adapters = adapters;
  a.slots64 = flags & CFMOE_IDS_INT64;
  const unsigned columns = (outputs + kOutWaves * kOutColumns - 1) / (kOutWaves * kOutColumns);
  const unsigned ranks = (rank + 15) / 16;
  if (!sorts(tokens)) {
    hipLaunchKernelGGL((adapter_inner_kernel<false, 1>), dim3(tokens, ranks), dim3(64 * kInnerWaves), 0, stream, a);
    if (int rc = check_launch("adapter_inner")) return rc;
    hipLaunchKernelGGL((adapter_out_kernel<false, 1>), dim3(tokens, columns), dim3(64 * kOutWaves), 0, stream, a);
    return check_launch("adapter_out");
  }
  char *at = static_cast<char *>(scratch) + static_cast<int64_t>(tokens) * rank * 4;
  auto take = [&](int64_t size) {
    void *p = at;
    at += rounded(size);
    return static_cast<int32_t *>(p);
  };
  int32_t *offsets = take(4 * (adapters + 1)), *pairs = take(4 * static_cast<int64_t>(tokens));
  int32_t *places = take(4 * static_cast<int64_t>(tokens));
  if (int rc = cfmoe_sort_by_expert(adapters, 1, flags & CFMOE_IDS_INT64, slots, nullptr, offsets, places, pairs, at, tokens, stream))
    return rc;
  a.offsets = offsets;
  a.pairs = pairs;
  // tiles there can be at most: one more for each adapter, and for the tokens without one
  auto tiles = [&](int tile) {
    return static_cast<unsigned>((tokens + tile - 1) / tile + (adapters + 1 < tokens ? adapters + 1 : tokens));
  };
  if (ranks > 1)
    hipLaunchKernelGGL((adapter_inner_kernel<true, 4>), dim3(tiles(kInnerTokens), (ranks + 3) / 4), dim3(64 * kInnerWaves), 0, stream, a);
  else
    hipLaunchKernelGGL((adapter_inner_kernel<true, 1>), dim3(tiles(kInnerTokens), 1), dim3(64 * kInnerWaves), 0, stream, a);
  if (int rc = check_launch("adapter_inner")) return rc;
  hipLaunchKernelGGL((adapter_out_kernel<true, 4>), dim3(tiles(64), columns), dim3(64 * kOutWaves), 0, stream, a);
  return check_launch("adapter_out");
}

}  // extern "C"
