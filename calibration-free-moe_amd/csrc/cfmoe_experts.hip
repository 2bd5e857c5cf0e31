// MI355X (gfx950) whole MoE layer for a batch of few tokens.
//
//   out[t] = sum_k w[t, k] D_e (phi(G_e x_t) * (U_e x_t)),  e = ids[t, k]
//
// A (token, slot) pair is one row of its expert's products. The layer's time is
// that of reading every touched expert's weights once, so each workgroup owns a
// piece of one expert's weights and computes it for all of that expert's pairs:
// it gathers them from the ids itself (pairs of one expert, ascending), 16 to a
// matrix instruction's columns. Three launches:
//
//   experts_up_kernel    act[p, c] = bf16(w phi(g) u), g and u in FP32
//   experts_down_kernel  partial[s, p, h] = FP32 sum over split s of the channels
//   experts_join_kernel  out[t, h] = bf16(sum over t's slots and splits, in order)
//
// A pair whose id lies outside [0, E) or whose token is padded belongs to no
// expert: nothing computes it, and the join leaves it out.
//
// Rounding act to BF16 makes it the matrix operand of the second product; the
// router weight goes in before, so that a pair is rounded once.

#include <algorithm>

#include "cfmoe_device.h"

namespace cfmoe {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kMaxPairs = 8192;
constexpr int kColumns = 16;      // pairs of a matrix instruction
constexpr int kUpChannels = 8;    // channels of 16 rows: gate and up row in turn
constexpr int kDownRows = 128;    // outputs of a BF16 down workgroup
constexpr int kFp4DownRows = 64;  // of an FP4 one, 16 a wave

struct ExpertArgs {
  const uint16_t *x;
  const void *ids, *weights;
  const uint8_t *padding;
  const uint8_t *gate_up, *gate_up_scales, *down, *down_scales;
  uint16_t *act;   // [pairs, act_stride]
  float *partial;  // [splits, pairs, hidden]
  uint16_t *out;
  int tokens, top_k, pairs, experts, hidden, width, act_stride, tiles, splits;
  bool ids64, weights16, gelu, by_pair;
};

__device__ __forceinline__ int pair_expert(const ExpertArgs &a, int pair) {
  if (a.padding && a.padding[pair / a.top_k]) return -1;
  int64_t id;
  if (a.ids64) id = static_cast<const int64_t *>(a.ids)[pair];
  else id = static_cast<const int32_t *>(a.ids)[pair];
  return id >= 0 && id < a.experts ? static_cast<int>(id) : -1;
}

__device__ __forceinline__ float pair_weight(const ExpertArgs &a, int pair) {
  return a.weights16 ? bf16_value(static_cast<const uint16_t *>(a.weights)[pair])
                     : static_cast<const float *>(a.weights)[pair];
}

// The pairs of item z's expert into `list`, ascending; returns their number (the
// same in every thread). With by_pair the items are the pairs, and an expert's
// first pair takes all of them: the others' items get none.
__device__ __forceinline__ int gather_pairs(const ExpertArgs &a, int z, int &expert, uint16_t *list,
                                            int *counts) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  expert = a.by_pair ? pair_expert(a, z) : z;
  if (expert < 0) return 0;
  const int share = (a.pairs + kThreads - 1) / kThreads * 64;  // pairs a wave looks at
  const int begin = min(wave * share, a.pairs), end = min(begin + share, a.pairs);
  int mine = 0;
  for (int p = begin + lane; p - lane < end; p += 64)
    mine += __builtin_popcountll(__ballot(p < end && pair_expert(a, p) == expert));
  if (lane == 0) counts[wave] = mine;
  __syncthreads();
  int at = 0, total = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    at += w < wave ? counts[w] : 0;
    total += counts[w];
  }
  for (int p = begin + lane; p - lane < end; p += 64) {
    const uint64_t found = __ballot(p < end && pair_expert(a, p) == expert);
    if (found >> lane & 1) list[at + __builtin_popcountll(found & ((1ull << lane) - 1))] = p;
    at += __builtin_popcountll(found);
  }
  __syncthreads();
  return a.by_pair && list[0] != z ? 0 : total;
}

__device__ __forceinline__ float activated(float gate, float up, bool gelu) {
  const float inner = gelu ? 1.5957691216057308f * (gate + 0.044715f * gate * gate * gate) : gate;
  return gate / (1.0f + __expf(-inner)) * up;
}

// The wave sums of a tile, added in order, become activations: lane l of tile
// (m, n) holds rows 4 (l / 16) .. + 3 of pair l % 16, that is gate and up of two
// channels.
template <int kTiles, int kCols>
__device__ __forceinline__ void store_activations(const ExpertArgs &a, const f32x4 *sums, const uint16_t *list,
                                                  int count, int base, int channel0) {
  __syncthreads();
  for (int i = threadIdx.x; i < kTiles * kCols * 64; i += kThreads) {
    f32x4 v = sums[i];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) v += sums[w * kTiles * kCols * 64 + i];
    const int lane = i % 64, n = i / 64 % kCols, m = i / (64 * kCols);
    const int column = base + n * kColumns + lane % 16;
    const int channel = channel0 + m * kUpChannels + lane / 16 * 2;
    if (column < count && channel < a.width) {
      const int pair = list[column];
      const float w = pair_weight(a, pair);
      *reinterpret_cast<uint32_t *>(a.act + static_cast<int64_t>(pair) * a.act_stride + channel) =
          bf16_pair(w * activated(v[0], v[1], a.gelu), w * activated(v[2], v[3], a.gelu));
    }
  }
  __syncthreads();
}

// Rows of x for a pass of kCols column tiles; a column past the last pair is not
// live (its products are not stored).
template <int kCols>
struct Columns {
  const u32x4 *row[kCols];
  bool live[kCols];
  __device__ __forceinline__ Columns(const ExpertArgs &a, const uint16_t *list, int count, int base) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int n = 0; n < kCols; ++n) {
      const int column = base + n * kColumns + lane % 16;
      live[n] = column < count;
      const int token = live[n] ? list[column] / a.top_k : 0;
      row[n] = reinterpret_cast<const u32x4 *>(a.x + static_cast<int64_t>(token) * a.hidden);
    }
  }
  __device__ __forceinline__ u32x4 load(int n, int at) const {
    u32x4 v = {0, 0, 0, 0};
    if (live[n]) v = row[n][at];
    return v;
  }
};

template <bool kFp4, int kTiles, int kCols>
__device__ __forceinline__ void up_pass(const ExpertArgs &a, int expert, int channel0, const uint16_t *list,
                                        int count, int base, f32x4 *sums) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Columns<kCols> columns(a, list, count, base);
  f32x4 d[kTiles][kCols];
#pragma unroll
  for (int m = 0; m < kTiles; ++m)
#pragma unroll
    for (int n = 0; n < kCols; ++n) d[m][n] = f32x4{0, 0, 0, 0};
  int64_t row[kTiles];
#pragma unroll
  for (int m = 0; m < kTiles; ++m) {
    const int channel = min(channel0 + m * kUpChannels + lane % 16 / 2, a.width - 1);
    row[m] = static_cast<int64_t>(expert) * 2 * a.width + (lane & 1) * a.width + channel;
  }
  if (kFp4) {
    // a lane's 16 bytes are one block of 32: four products of eight, lane group g
    // taking block g of the 128 hidden values of a step
    for (int s = wave; s < a.hidden / 128; s += kWaves) {
      u32x4 codes[kTiles];
      float scale[kTiles];
#pragma unroll
      for (int m = 0; m < kTiles; ++m) {
        codes[m] = reinterpret_cast<const u32x4 *>(a.gate_up + row[m] * (a.hidden / 2))[4 * s + lane / 16];
        scale[m] = __int_as_float(
            static_cast<int>(a.gate_up_scales[row[m] * (a.hidden / 32) + 4 * s + lane / 16]) << 23);
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        u32x4 b[kCols];
#pragma unroll
        for (int n = 0; n < kCols; ++n) b[n] = columns.load(n, 16 * s + lane / 16 * 4 + q);
#pragma unroll
        for (int m = 0; m < kTiles; ++m) {
          const u32x4 w = fp4_values(codes[m][q], scale[m]);
#pragma unroll
          for (int n = 0; n < kCols; ++n) d[m][n] = mma(w, b[n], d[m][n]);
        }
      }
    }
  } else {
#pragma unroll 4
    for (int s = wave; s < a.hidden / 32; s += kWaves) {
      u32x4 w[kTiles], b[kCols];
#pragma unroll
      for (int m = 0; m < kTiles; ++m)
        w[m] = reinterpret_cast<const u32x4 *>(a.gate_up + row[m] * (2 * a.hidden))[4 * s + lane / 16];
#pragma unroll
      for (int n = 0; n < kCols; ++n) b[n] = columns.load(n, 4 * s + lane / 16);
#pragma unroll
      for (int m = 0; m < kTiles; ++m)
#pragma unroll
        for (int n = 0; n < kCols; ++n) d[m][n] = mma(w[m], b[n], d[m][n]);
    }
  }
#pragma unroll
  for (int m = 0; m < kTiles; ++m)
#pragma unroll
    for (int n = 0; n < kCols; ++n) sums[((wave * kTiles + m) * kCols + n) * 64 + lane] = d[m][n];
  store_activations<kTiles, kCols>(a, sums, list, count, base, channel0);
}

constexpr int kUpTiles = 2;
constexpr int kUpCols = 4;

template <bool kFp4>
__global__ __launch_bounds__(kThreads) void experts_up_kernel(ExpertArgs a) {
  __shared__ f32x4 sums[kWaves * kUpTiles * kUpCols * 64];
  __shared__ int counts[kWaves];
  extern __shared__ uint16_t list[];
  const int tile = blockIdx.x % a.tiles;
  int expert;
  const int count = gather_pairs(a, blockIdx.x / a.tiles, expert, list, counts);
  const int channel0 = tile * kUpTiles * kUpChannels;
  for (int base = 0; base < count;) {
    if (count - base > 2 * kColumns) {
      up_pass<kFp4, kUpTiles, 4>(a, expert, channel0, list, count, base, sums);
      base += 4 * kColumns;
    } else if (count - base > kColumns) {
      up_pass<kFp4, kUpTiles, 2>(a, expert, channel0, list, count, base, sums);
      base += 2 * kColumns;
    } else {
      up_pass<kFp4, kUpTiles, 1>(a, expert, channel0, list, count, base, sums);
      base += kColumns;
    }
  }
}

// Channel-major down rows hold an output per element, where the matrix operand
// wants eight channels of one output: a lane loads eight channels' rows at its
// eight outputs and turns the 8 x 8 square in registers. Output 8 (l % 16) + j of
// the tile is row l % 16 of product j.
__device__ __forceinline__ void turn(const u32x4 (&rows)[8], u32x4 (&turned)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t select = j & 1 ? 0x07060302u : 0x05040100u;
#pragma unroll
    for (int c = 0; c < 4; ++c)
      turned[j][c] = __builtin_amdgcn_perm(rows[2 * c + 1][j / 2], rows[2 * c][j / 2], select);
  }
}

// Workgroup = 128 outputs of one expert over one split of its channels, the waves
// every fourth 32 channels of it.
template <int kCols>
__device__ __forceinline__ void down_pass(const ExpertArgs &a, int expert, int row0, int split, const uint16_t *list,
                                          int count, int base, f32x4 *sums) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int steps = (a.width + 31) / 32;
  const int begin = steps * split / a.splits, end = steps * (split + 1) / a.splits;
  const uint16_t *act[kCols];
  bool live[kCols];
#pragma unroll
  for (int n = 0; n < kCols; ++n) {
    const int column = base + n * kColumns + lane % 16;
    live[n] = column < count;
    act[n] = a.act + static_cast<int64_t>(live[n] ? list[column] : 0) * a.act_stride;
  }
  f32x4 d[8][kCols];
#pragma unroll
  for (int j = 0; j < 8; ++j)
#pragma unroll
    for (int n = 0; n < kCols; ++n) d[j][n] = f32x4{0, 0, 0, 0};
  const uint16_t *down = reinterpret_cast<const uint16_t *>(a.down) +
                         static_cast<int64_t>(expert) * a.width * a.hidden + row0 + lane % 16 * 8;
  for (int s = begin + wave; s < end; s += kWaves) {
    const int channel = 32 * s + lane / 16 * 8;
    const bool inside = channel < a.width;  // (the width is a multiple of 16)
    u32x4 rows[8], turned[8], b[kCols];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      rows[i] = u32x4{0, 0, 0, 0};
      if (inside) rows[i] = *reinterpret_cast<const u32x4 *>(down + static_cast<int64_t>(channel + i) * a.hidden);
    }
#pragma unroll
    for (int n = 0; n < kCols; ++n) {
      b[n] = u32x4{0, 0, 0, 0};
      if (inside && live[n]) b[n] = *reinterpret_cast<const u32x4 *>(act[n] + channel);
    }
    turn(rows, turned);
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int n = 0; n < kCols; ++n) d[j][n] = mma(turned[j], b[n], d[j][n]);
  }
  // sums[wave][column tile][product j][lane]
#pragma unroll
  for (int n = 0; n < kCols; ++n)
#pragma unroll
    for (int j = 0; j < 8; ++j) sums[((wave * kCols + n) * 8 + j) * 64 + lane] = d[j][n];
  __syncthreads();
  for (int i = threadIdx.x; i < kCols * 8 * 64; i += kThreads) {
    f32x4 v = sums[i];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) v += sums[w * kCols * 8 * 64 + i];
    const int at = i % 64, j = i / 64 % 8, n = i / 512;
    const int column = base + n * kColumns + at % 16;
    if (column < count) {
      float *out = a.partial + (static_cast<int64_t>(split) * a.pairs + list[column]) * a.hidden + row0 + j;
#pragma unroll
      for (int r = 0; r < 4; ++r) out[8 * (at / 16 * 4 + r)] = v[r];
    }
  }
  __syncthreads();
}

__global__ __launch_bounds__(kThreads) void experts_down_kernel(ExpertArgs a) {
  __shared__ f32x4 sums[kWaves * 8 * 64];
  __shared__ int counts[kWaves];
  extern __shared__ uint16_t list[];
  const int tile = blockIdx.x % a.tiles, rest = blockIdx.x / a.tiles;
  int expert;
  const int count = gather_pairs(a, rest / a.splits, expert, list, counts);
  for (int base = 0; base < count;) {
    down_pass<1>(a, expert, tile * kDownRows, rest % a.splits, list, count, base, sums);
    base += kColumns;
  }
}

// Wave = 16 outputs of one expert, all its channels: a lane's 16 bytes are one
// block of its row, as in up_pass. A last step's groups past the width are zero.
template <int kCols>
__device__ __forceinline__ void fp4_down_pass(const ExpertArgs &a, int expert, int row0, const uint16_t *list,
                                              int count, int base) {
  const int lane = threadIdx.x & 63;
  const int blocks = a.width / 32;
  const int64_t row = static_cast<int64_t>(expert) * a.hidden + row0 + lane % 16;
  const u32x4 *codes = reinterpret_cast<const u32x4 *>(a.down + row * (a.width / 2));
  const uint8_t *scales = a.down_scales + row * blocks;
  const u32x4 *act[kCols];
  bool live[kCols];
  int pair[kCols];
  f32x4 d[kCols];
#pragma unroll
  for (int n = 0; n < kCols; ++n) {
    const int column = base + n * kColumns + lane % 16;
    live[n] = column < count;
    pair[n] = live[n] ? list[column] : 0;
    act[n] = reinterpret_cast<const u32x4 *>(a.act + static_cast<int64_t>(pair[n]) * a.act_stride);
    d[n] = f32x4{0, 0, 0, 0};
  }
  for (int block = lane / 16; block - lane / 16 < blocks; block += 4) {
    const bool inside = block < blocks;
    u32x4 word = {0, 0, 0, 0};
    float scale = 0.0f;
    if (inside) {
      word = codes[block];
      scale = __int_as_float(static_cast<int>(scales[block]) << 23);
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const u32x4 w = fp4_values(word[q], scale);
#pragma unroll
      for (int n = 0; n < kCols; ++n) {
        u32x4 b = {0, 0, 0, 0};
        if (inside && live[n]) b = act[n][4 * block + q];
        d[n] = mma(w, b, d[n]);
      }
    }
  }
#pragma unroll
  for (int n = 0; n < kCols; ++n)
    if (live[n])
      *reinterpret_cast<f32x4 *>(a.partial + static_cast<int64_t>(pair[n]) * a.hidden + row0 + lane / 16 * 4) = d[n];
}

__global__ __launch_bounds__(kThreads) void experts_fp4_down_kernel(ExpertArgs a) {
  __shared__ int counts[kWaves];
  extern __shared__ uint16_t list[];
  const int tile = blockIdx.x % a.tiles;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int expert;
  const int count = gather_pairs(a, blockIdx.x / a.tiles, expert, list, counts);
  const int row0 = tile * kFp4DownRows + wave * 16;
  for (int base = 0; base < count;) {
    if (count - base > 2 * kColumns) {
      fp4_down_pass<4>(a, expert, row0, list, count, base);
      base += 4 * kColumns;
    } else {
      fp4_down_pass<2>(a, expert, row0, list, count, base);
      base += 2 * kColumns;
    }
  }
}

// Thread = eight outputs of one token: its slots' partials in order, each split's
// in order within a slot.
__global__ __launch_bounds__(kThreads) void experts_join_kernel(ExpertArgs a) {
  const int groups = a.hidden / 8;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const int t = static_cast<int>(i / groups), h = static_cast<int>(i % groups) * 8;
  if (t >= a.tokens) return;
  f32x4 low = {0, 0, 0, 0}, high = {0, 0, 0, 0};
  for (int k = 0; k < a.top_k; ++k) {
    const int pair = t * a.top_k + k;
    if (pair_expert(a, pair) < 0) continue;
    for (int s = 0; s < a.splits; ++s) {
      const f32x4 *p = reinterpret_cast<const f32x4 *>(
          a.partial + (static_cast<int64_t>(s) * a.pairs + pair) * a.hidden + h);
      low += p[0];
      high += p[1];
    }
  }
  const u32x4 out = {bf16_pair(low[0], low[1]), bf16_pair(low[2], low[3]), bf16_pair(high[0], high[1]),
                     bf16_pair(high[2], high[3])};
  *reinterpret_cast<u32x4 *>(a.out + static_cast<int64_t>(t) * a.hidden + h) = out;
}

int validate(int hidden, int width, int experts, int top_k, uint32_t flags, int tokens) {
  if (hidden <= 0 || hidden % 128 || hidden > 16384)
    return fail(CFMOE_EINVAL, "routed_experts needs a hidden size that is a multiple of 128, at most 16384");
  const int grain = flags & CFMOE_FP4 ? 32 : 16;
  if (width <= 0 || width % grain || width > 16384)
    return fail(CFMOE_EINVAL, "routed_experts needs a width that is a multiple of 16 (of 32 with 4-bit weights), at most 16384");
  if (experts < 1 || experts > 4096) return fail(CFMOE_EINVAL, "routed_experts needs 1 to 4096 experts");
  if (top_k < 1 || top_k > 64) return fail(CFMOE_EINVAL, "routed_experts needs 1 to 64 experts per token");
  if (tokens < 0 || static_cast<int64_t>(tokens) * top_k > kMaxPairs)
    return fail(CFMOE_EINVAL, "routed_experts takes at most 8192 routed pairs per call");
  return 0;
}

// Down splits: workgroups that share an expert's channels, so that a batch of few
// pairs still covers the compute units.
int down_splits(int hidden, int width, int experts, int top_k, uint32_t flags, int tokens) {
  if (flags & CFMOE_FP4) return 1;
  const int items = std::min(tokens * top_k, experts) * (hidden / kDownRows);
  const int steps = (width + 31) / 32;
  int splits = 1;
  while (items * splits < 256 && splits * 2 * kWaves <= steps) splits *= 2;
  return splits;
}

int64_t act_bytes(int width, int pairs) {
  return static_cast<int64_t>(pairs) * width * 2;  // (a row is a multiple of 32 bytes)
}

}  // namespace
}  // namespace cfmoe

extern "C" {

using namespace cfmoe;

CFMOE_API int64_t cfmoe_routed_experts_scratch_bytes(int32_t hidden_size, int32_t width, int32_t experts,
                                                     int32_t top_k, uint32_t flags, int32_t tokens) {
  if (int rc = validate(hidden_size, width, experts, top_k, flags, tokens)) return -rc;
  const int pairs = tokens * top_k;
  const int splits = down_splits(hidden_size, width, experts, top_k, flags, tokens);
  return act_bytes(width, pairs) + static_cast<int64_t>(splits) * pairs * hidden_size * 4;
}

CFMOE_API int cfmoe_routed_experts(int32_t hidden_size, int32_t width, int32_t experts, int32_t top_k,
                                   uint32_t flags, const void *gate_up, const uint8_t *gate_up_scales,
                                   const void *down, const uint8_t *down_scales, const void *hidden,
                                   const void *ids, const void *weights, const uint8_t *padding, void *out,
                                   void *scratch, int32_t tokens, cfmoe_stream stream) {
  if (int rc = validate(hidden_size, width, experts, top_k, flags, tokens)) return rc;
  if (tokens == 0) return 0;
  const bool fp4 = flags & CFMOE_FP4;
  if (!gate_up || !down || !hidden || !ids || !weights || !out || !scratch ||
      (fp4 && (!gate_up_scales || !down_scales)))
    return fail(CFMOE_EINVAL, "NULL argument");
  uintptr_t addresses = 0;
  for (const void *p : {gate_up, down, hidden, static_cast<const void *>(out), static_cast<const void *>(scratch)})
    addresses |= reinterpret_cast<uintptr_t>(p);
  if (addresses % 16)
    return fail(CFMOE_EINVAL, "routed_experts needs 16-byte aligned weights, hidden rows, output and scratch");
  ExpertArgs a;
  a.x = static_cast<const uint16_t *>(hidden);
  a.ids = ids;
  a.weights = weights;
  a.padding = padding;
  a.gate_up = static_cast<const uint8_t *>(gate_up);
  a.gate_up_scales = gate_up_scales;
  a.down = static_cast<const uint8_t *>(down);
  a.down_scales = down_scales;
  a.out = static_cast<uint16_t *>(out);
  a.tokens = tokens;
  a.top_k = top_k;
  a.pairs = tokens * top_k;
  a.experts = experts;
  a.hidden = hidden_size;
  a.width = width;
  a.act_stride = width;
  a.splits = down_splits(hidden_size, width, experts, top_k, flags, tokens);
  a.act = static_cast<uint16_t *>(scratch);
  a.partial = reinterpret_cast<float *>(static_cast<uint8_t *>(scratch) + act_bytes(width, a.pairs));
  a.ids64 = flags & CFMOE_IDS_INT64;
  a.weights16 = flags & CFMOE_WEIGHTS_BF16;
  a.gelu = flags & CFMOE_GELU;
  a.by_pair = a.pairs <= experts;
  const int items = a.by_pair ? a.pairs : experts;
  const unsigned list = static_cast<unsigned>((a.pairs * 2 + 15) / 16 * 16);

  a.tiles = (width + kUpTiles * kUpChannels - 1) / (kUpTiles * kUpChannels);
  const dim3 up(static_cast<unsigned>(a.tiles) * items);
  if (fp4) hipLaunchKernelGGL(experts_up_kernel<true>, up, dim3(kThreads), list, stream, a);
  else hipLaunchKernelGGL(experts_up_kernel<false>, up, dim3(kThreads), list, stream, a);
  if (int rc = check_launch("experts_up")) return rc;

  a.tiles = hidden_size / (fp4 ? kFp4DownRows : kDownRows);
  const dim3 grid(static_cast<unsigned>(a.tiles) * items * a.splits);
  if (fp4) hipLaunchKernelGGL(experts_fp4_down_kernel, grid, dim3(kThreads), list, stream, a);
  else hipLaunchKernelGGL(experts_down_kernel, grid, dim3(kThreads), list, stream, a);
  if (int rc = check_launch("experts_down")) return rc;

  const int64_t threads = static_cast<int64_t>(tokens) * (hidden_size / 8);
  hipLaunchKernelGGL(experts_join_kernel, dim3(static_cast<unsigned>((threads + kThreads - 1) / kThreads)),
                     dim3(kThreads), 0, stream, a);
  return check_launch("experts_join");
}

}  // extern "C"
