// MI355X (gfx950): low-rank adapters of many requests beside a shared projection.
//
//   out[t] = base[t] + s_a D_a (C_a x[t])        a = slots[t]
//
// with C_a [R, H] and D_a [O, R] of the adapter that token t's request has, s_a its scale;
// a token whose slot names none keeps its row of `base`, bit for bit.
//
// Tokens of one adapter share its weights: they form tiles, and a tile's products are
// matrix instructions, C_a x over the hidden dimension and D_a v, v = s_a C_a x, over the rank. A
// decode step's tiles hold a token or two, which leaves most columns of an instruction
// empty: what bounds it is the weights' reading, once for each tile, and a compute unit
// takes about 75 GB/s from memory. So the hidden dimension and the ranks are spread over
// workgroups (adapter_inner_kernel), and the second launch (adapter_out_kernel) adds up
// their parts; of few ranks one workgroup reads all (adapter_one_kernel). Many tokens
// are sorted by adapter first.
//
// As operand of the second product v is the sum of three BF16 numbers, which hold all 24 bits
// of it, and out is rounded once. (Two hold 16: 4001 tokens of rank 64 then had 51000 of 16
// million outputs next to their exact value's rounding, where FP32 sums leave 7000.)

#include "cfmoe_rows.h"

namespace cfmoe {
namespace {

constexpr int kMaxAdapters = 4096;
constexpr int kMaxRank = 256;
constexpr int kMaxSize = 65536;
constexpr int kFewTokens = 256;    // up to which two launches find their tiles by themselves
constexpr int kTokens = 16;        // of a tile, few tokens
constexpr int kManyTokens = 32;    // of a tile, many tokens
constexpr int kWaves = 4;
constexpr int kOneWaves = 16;      // of the kernel of both products, and what it takes of
constexpr int kOneRank = 32;       // ranks,
constexpr int kOneValues = 131072; // values of C
constexpr int kOneGroups = 1024;   // and workgroups, so tokens too
constexpr int kUnit = 8;           // values of 16 bytes
constexpr int kColumns = 64;       // outputs of one wave
constexpr int kTurn = 64 * kWaves; // hidden values that the waves take at a time
constexpr int kFewSplits = 16;     // of the hidden dimension at most
constexpr int kManySplits = 2;
constexpr int kMostGroups = 2048;  // workgroups of the second launch, from which each takes more outputs

struct AdapterArgs {
  const uint16_t *base, *x, *encoder, *decoder;
  const void *slots;
  const float *scales;
  uint16_t *out;
  float *inner;            // [splits, T, R]: parts of C x, tokens in sorted order where they are sorted
  const int32_t *offsets;  // [N + 1] and
  const int32_t *pairs;    // [T]: tokens by adapter (many tokens only)
  int64_t base_stride, x_stride, out_stride;
  int tokens, hidden, outputs, rank, adapters;
  int splits, share;       // of the hidden dimension, and values of one
  bool slots64;
};

// The adapter of a token; `adapters` where its slot names none.
__device__ __forceinline__ int slot_of(const AdapterArgs &a, int t) {
  const int64_t s = a.slots64 ? static_cast<const int64_t *>(a.slots)[t] : static_cast<const int32_t *>(a.slots)[t];
  return s >= 0 && s < a.adapters ? static_cast<int>(s) : a.adapters;
}

// Tokens of one adapter, up to kTokens, of a call of few: tile t is led by token t, if a
// whole number of tiles' tokens of its adapter come before it; the workgroup reads all
// slots. False where no tile is. All threads of the workgroup call it.
template <int kWaves>
__device__ __forceinline__ bool find_tile(const AdapterArgs &a, int leader, int *members, int &adapter, int &count) {
  __shared__ uint64_t masks[kOneGroups / 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, words = (a.tokens + 63) / 64;
  adapter = __builtin_amdgcn_readfirstlane(slot_of(a, leader));
  for (int w = wave; w < words; w += kWaves) {
    const int t = 64 * w + lane;
    const uint64_t same = __ballot(t < a.tokens && slot_of(a, min(t, a.tokens - 1)) == adapter);
    if (lane == 0) masks[w] = same;
  }
  __syncthreads();
  int before = __builtin_popcountll(masks[leader / 64] & ((UINT64_C(1) << (leader % 64)) - 1));
  for (int w = 0; w < leader / 64; ++w) before += __builtin_popcountll(masks[w]);
  if (before % kTokens) return false;
  int passed = 0;
  for (int w = 0; w < words; ++w) {
    const uint64_t same = masks[w];
    const int rank = passed - before + __builtin_popcountll(same & ((UINT64_C(1) << lane) - 1));
    if (wave == 0 && (same >> lane & 1) && rank >= 0 && rank < kTokens) members[rank] = 64 * w + lane;
    passed += __builtin_popcountll(same);
  }
  count = __builtin_amdgcn_readfirstlane(min(kTokens, passed - before));
  __syncthreads();
  return true;
}

// The same of a call whose tokens are sorted by adapter: tile `index`, tiles counted
// through the adapters' offsets by each wave for itself.
template <int kTile>
__device__ __forceinline__ bool find_sorted_tile(const AdapterArgs &a, int index, int &adapter, int &start, int &count) {
  const int lane = threadIdx.x & 63;
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
      adapter = first + owner;
      start = __builtin_amdgcn_readlane(from, owner) +
              (index - before - __builtin_amdgcn_readlane(scan - tiles, owner)) * kTile;
      count = min(kTile, __builtin_amdgcn_readlane(to, owner) - start);
      return true;
    }
    before += __builtin_amdgcn_readlane(scan, 63);
  }
  return false;
}

__device__ __forceinline__ u32x4 load16(const uint16_t *p) { return *reinterpret_cast<const u32x4 *>(p); }

constexpr int kParts = 3;

// BF16 numbers whose sum is v. All but the last are cut off from the FP32 number below what
// is left, so that none is zero or of the other sign where v is not: an infinite weight times
// them is that infinity, and where v is infinite the last is. After the second cut at most 8
// bits are left or a power of two, so that the last number is exact. (So down to |v| =
// 2^-102; from there it is rounded up to BF16's last step, 2^-133, and below 2^-109 the
// second may be zero.)
__device__ __forceinline__ void split(f32x4 v, u32x2 (&part)[kParts]) {
#pragma unroll
  for (int k = 0; k + 1 < kParts; ++k) {
    uint32_t cut[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t bits = __float_as_uint(v[i]), size = bits & 0x7fffffffu;
      cut[i] = ((size - (size != 0)) | (bits & 0x80000000u)) & 0xffff0000u;
      v[i] -= __uint_as_float(cut[i]);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) part[k][i] = cut[2 * i] >> 16 | cut[2 * i + 1];
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
    part[kParts - 1][i] = (__float_as_uint(v[2 * i]) + 0xffffu) >> 16 | ((__float_as_uint(v[2 * i + 1]) + 0xffffu) & 0xffff0000u);
}

// sum + w v of 16 outputs and tokens, the parts of v from the smallest on.
__device__ __forceinline__ f32x4 parts_product(u32x4 w, const u32x4 (&v)[kParts], f32x4 sum) {
#pragma unroll
  for (int k = kParts - 1; k >= 0; --k) sum = mma(w, v[k], sum);
  return sum;
}

// Values of a row of v in LDS: whole steps of 32, and a unit for the banks.
__host__ __device__ __forceinline__ int parts_row(int rank) { return (rank + 31) / 32 * 32 + kUnit; }

// d[g][i] += C x of a wave's part of the hidden dimension: its turns of 64 values from `first`
// on, in steps of `step`, of kTiles tiles of 16 rows of C and kGroups of 16 tokens. The
// operands pass through the wave's own part of LDS: eight lanes read 128 bytes of a row from
// memory, where the matrix instruction's own layout has neighbouring lanes read from
// different rows, a quarter as fast (4001 tokens of 2048 values, rank 64: 14.5 us so, 10.5
// through LDS). Rows of LDS are an odd number of 16-byte units long, so that the 16 rows of
// an operand lie in different banks. row[j]: this lane's unit of every eighth row, C's, then
// the tokens' (past the end any, what they give is not stored).
constexpr int kStageRow = 64 + kUnit;

template <int kTiles, int kGroups>
__device__ __forceinline__ void staged_product(uint16_t (*stage)[kStageRow], const uint16_t *const *row, int first,
                                               int last, int step, f32x4 (*d)[kTiles]) {
  constexpr int kLoads = 2 * (kTiles + kGroups);
  const int lane = threadIdx.x & 63, m = lane & 15, q = lane >> 4;
  u32x4 raw[kLoads];
  auto fetch = [&](int h0) {
    if (h0 + 64 <= last) {
#pragma unroll
      for (int j = 0; j < kLoads; ++j) raw[j] = load16(row[j] + h0);
    } else if (h0 < last) {
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        raw[j] = u32x4{0, 0, 0, 0};
        if (h0 + kUnit * (lane % 8) < last) raw[j] = load16(row[j] + h0);
      }
    }
  };
  fetch(first);
  for (int h0 = first; h0 < last; h0 += step) {
#pragma unroll
    for (int j = 0; j < kLoads; ++j) *reinterpret_cast<u32x4 *>(&stage[8 * j + lane / 8][kUnit * (lane % 8)]) = raw[j];
    fetch(h0 + step);
    wave_in_step();
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      u32x4 xv[kGroups];
#pragma unroll
      for (int g = 0; g < kGroups; ++g) xv[g] = load16(&stage[16 * (kTiles + g) + m][32 * s + kUnit * q]);
#pragma unroll
      for (int i = 0; i < kTiles; ++i) {
        const u32x4 cv = load16(&stage[16 * i + m][32 * s + kUnit * q]);
#pragma unroll
        for (int g = 0; g < kGroups; ++g) d[g][i] = mma(cv, xv[g], d[g][i]);
      }
    }
    wave_in_step();
  }
}

// inner[split, token, r] = a split's part of sum_h C[r, h] x[token, h], of a tile of
// tokens and kTiles tiles of 16 ranks (s multiplies the whole sum, in the second launch: parts
// that it takes out of FP32 may cancel). The waves take the split's hidden values in turns of
// 64 and add up in LDS. What bounds it is the chain of offsets, tokens and rows in memory,
// four turns of them for a wave.
template <bool kSorted, int kTiles>
__global__ __launch_bounds__(64 * kWaves) void adapter_inner_kernel(AdapterArgs a) {
  constexpr int kTile = kSorted ? kManyTokens : kTokens, kGroups = kTile / 16;
  constexpr int kRows = 16 * kTiles + kTile, kLoads = kRows / 8, kRankLoads = 2 * kTiles;
  __shared__ __attribute__((aligned(16))) uint16_t stage[kWaves][kRows][kStageRow];
  __shared__ int members[kTokens];
  static_assert(sizeof(float) * kWaves * kGroups * kTiles * 256 <= sizeof(stage), "the sums take the stage's place");
  float(*sums)[kGroups][kTiles][256] = reinterpret_cast<float(*)[kGroups][kTiles][256]>(stage);
  int adapter, start = 0, count;
  if constexpr (kSorted) {
    if (!find_sorted_tile<kTile>(a, blockIdx.x, adapter, start, count)) return;
  } else {
    if (!find_tile<kWaves>(a, blockIdx.x, members, adapter, count)) return;
  }
  if (adapter >= a.adapters) return;
  const int lane = threadIdx.x & 63, m = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r0 = blockIdx.y * 16 * kTiles;
  const uint16_t *row[kLoads];
#pragma unroll
  for (int j = 0; j < kLoads; ++j) {
    const int r = min(r0 + 8 * j + lane / 8, a.rank - 1), t = min(8 * (j - kRankLoads) + lane / 8, count - 1);
    if (j < kRankLoads) row[j] = a.encoder + (static_cast<int64_t>(adapter) * a.rank + r) * a.hidden;
    else row[j] = a.x + static_cast<int64_t>(kSorted ? a.pairs[start + t] : members[t]) * a.x_stride;
    row[j] += kUnit * (lane % 8);
  }
  f32x4 d[kGroups][kTiles] = {};
  const int first = blockIdx.z * a.share, last = min(first + a.share, a.hidden);
  staged_product<kTiles, kGroups>(stage[wave], row, first + 64 * wave, last, kTurn, d);
  __syncthreads();
#pragma unroll
  for (int g = 0; g < kGroups; ++g)
#pragma unroll
    for (int i = 0; i < kTiles; ++i) *reinterpret_cast<f32x4 *>(&sums[wave][g][i][m * 16 + 4 * q]) = d[g][i];
  __syncthreads();
  const int n = threadIdx.x % 16;
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    const int t = 16 * g + threadIdx.x / 16;
    if (t >= count) return;
    float *to = a.inner + (static_cast<int64_t>(blockIdx.z) * a.tokens + (kSorted ? start + t : members[t])) * a.rank + r0 + n;
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
      if (r0 + 16 * i + n >= a.rank) break;
      float total = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) total += sums[w][g][i][threadIdx.x];
      to[16 * i] = total;
    }
  }
}

// Output of matrix row n of tile i, behind a wave's first: lane 16 q + m ends with outputs
// 8 q .. 8 q + 7 and 32 + 8 q .. of token m, so that four lanes take 64 bytes of a row.
__device__ __forceinline__ int output_of(int i, int n) { return i / 2 * 32 + n / 4 * 8 + i % 2 * 4 + n % 4; }

// Half s of a lane's outputs, rounded once.
__device__ __forceinline__ u32x4 added(u32x4 base, const f32x4 *sum, int s) {
  float v[kUnit];
  Lane<false, kWhole>::values(base, v);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    base[i] = bf16_pair(v[2 * i] + sum[2 * s + i / 2][2 * i % 4], v[2 * i + 1] + sum[2 * s + i / 2][2 * i % 4 + 1]);
  return base;
}

// out = base + D v for a tile of tokens, a wave 64 outputs of them at a time: rows of base
// and D on their way first, then v from its splits, as three BF16 numbers in LDS. kShort is for
// ranks up to 32, whose rows of D are read ahead with base. 4001 tokens of rank 64 to 4096
// outputs take 22 us, 14 of which the same call takes for tokens without an adapter (66 MB of
// base and out): the rest is a tile's chain of reads and its vector arithmetic. Rows of D
// and out through LDS, tiles of 16 or 64 tokens and D's rows read ahead at rank 64 took
// 21 to 26.
template <bool kSorted, bool kShort>
__global__ __launch_bounds__(64 * kWaves) void adapter_out_kernel(AdapterArgs a) {
  constexpr int kTile = kSorted ? kManyTokens : kTokens, kGroups = kTile / 16;
  extern __shared__ __attribute__((aligned(16))) uint16_t parts[];  // [kParts, kTile, parts_row(R)]
  __shared__ int members[kTokens];
  int adapter, start = 0, count;
  if constexpr (kSorted) {
    if (!find_sorted_tile<kTile>(a, blockIdx.x, adapter, start, count)) return;
  } else {
    if (!find_tile<kWaves>(a, blockIdx.x, members, adapter, count)) return;
  }
  const bool bare = adapter >= a.adapters;
  if (bare && a.out == a.base) return;
  const int lane = threadIdx.x & 63, m = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int step = gridDim.y * kWaves * kColumns, stride = parts_row(a.rank);
  int o0 = (blockIdx.y * kWaves + wave) * kColumns;
  // this lane's unit of its tokens' rows (a token past the end is the last again)
  const uint16_t *from[kGroups];
  uint16_t *to[kGroups];
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    const int at = min(16 * g + m, count - 1);
    const int64_t token = kSorted ? a.pairs[start + at] : members[at];
    from[g] = a.base + token * a.base_stride + kUnit * q;
    to[g] = a.out + token * a.out_stride + kUnit * q;
  }
  u32x4 base[kGroups][2], w[4];
  auto fetch_base = [&](int first) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      if (first + 32 * s + kUnit * q >= a.outputs) continue;
#pragma unroll
      for (int g = 0; g < kGroups; ++g) base[g][s] = load16(from[g] + first + 32 * s);
    }
  };
  const uint16_t *decoder = a.decoder + static_cast<int64_t>(bare ? 0 : adapter) * a.outputs * a.rank;
  unsigned unit[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) unit[i] = output_of(i, m) * a.rank + kUnit * q;
  // rows of D, zero past the last rank (rows past the last output are not stored)
  auto fetch_rows = [&](int first, int r0, u32x4 *rows) {
    const uint16_t *at = decoder + static_cast<int64_t>(first) * a.rank + r0;
    if (first + kColumns <= a.outputs && r0 + 32 <= a.rank) {
#pragma unroll
      for (int i = 0; i < 4; ++i) rows[i] = load16(at + unit[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        rows[i] = u32x4{0, 0, 0, 0};
        if (first + output_of(i, m) < a.outputs && r0 + kUnit * q < a.rank) rows[i] = load16(at + unit[i]);
      }
    }
  };
  auto fetch = [&](int first) {
    if (first >= a.outputs) return;
    fetch_base(first);
    if (kShort && !bare) fetch_rows(first, 0, w);
  };
  fetch(o0);
  if (!bare) {
    // (zeros behind the last rank: the matrix instructions take 32 at a time)
    const int fours = (stride - kUnit) / 4;
    const float scale = a.scales ? a.scales[adapter] : 1.0f;
    for (int i = threadIdx.x; i < count * fours; i += 64 * kWaves) {
      const int t = i / fours, r = i % fours * 4;
      const float *inner = a.inner + static_cast<int64_t>(kSorted ? start + t : members[t]) * a.rank + r;
      f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
      if (r < a.rank) {
        v = *reinterpret_cast<const f32x4 *>(inner);
#pragma unroll 4
        for (int s = 1; s < a.splits; ++s)
          v += *reinterpret_cast<const f32x4 *>(inner + static_cast<int64_t>(s) * a.tokens * a.rank);
        v *= scale;
      }
      u32x2 part[kParts];
      split(v, part);
#pragma unroll
      for (int k = 0; k < kParts; ++k) *reinterpret_cast<u32x2 *>(parts + (k * kTile + t) * stride + r) = part[k];
    }
    __syncthreads();
  }
  // (rows of `parts` past the last token hold what they held: their columns of the products
  // are not stored)
  const uint16_t *v = parts + m * stride + kUnit * q;
  for (; o0 < a.outputs; o0 += step) {
    f32x4 sum[kGroups][4] = {};
    auto multiply = [&](int r0, const u32x4 *rows) {
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        u32x4 part[kParts];
#pragma unroll
        for (int k = 0; k < kParts; ++k) part[k] = load16(v + (k * kTile + 16 * g) * stride + r0);
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[g][i] = parts_product(rows[i], part, sum[g][i]);
      }
    };
    if (!bare) {
      if constexpr (kShort) {
        multiply(0, w);
      } else {
        for (int r0 = 0; r0 < a.rank; r0 += 32) {
          u32x4 rows[4];
          fetch_rows(o0, r0, rows);
          multiply(r0, rows);
        }
      }
    }
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const u32x4 row = bare ? base[g][s] : added(base[g][s], sum[g], s);
        if (16 * g + m < count && o0 + 32 * s + kUnit * q < a.outputs)
          *reinterpret_cast<u32x4 *>(to[g] + o0 + 32 * s) = row;
      }
    }
    fetch(o0 + step);
  }
}

// Both products of few tokens and ranks in one launch: workgroup = a tile and 1024 of its
// outputs, v formed again for each (so out cannot be x, which others still read). The waves
// take the hidden dimension in turns of 64; rows of base and D are on their way meanwhile.
template <int kTiles>
__global__ __launch_bounds__(64 * kOneWaves) void adapter_one_kernel(AdapterArgs a) {
  constexpr int kRow = 32 + kUnit, kLoads = 2 * (kTiles + 1);
  __shared__ __attribute__((aligned(16))) uint16_t stage[kOneWaves][16 * (kTiles + 1)][kStageRow];
  __shared__ __attribute__((aligned(16))) uint16_t parts[kParts][kTokens][kRow];
  __shared__ int members[kTokens];
  static_assert(sizeof(float) * kOneWaves * kTiles * 256 <= sizeof(stage), "the sums take the stage's place");
  float(*sums)[kTiles][256] = reinterpret_cast<float(*)[kTiles][256]>(stage);
  int adapter, count;
  if (!find_tile<kOneWaves>(a, blockIdx.x, members, adapter, count)) return;
  const bool bare = adapter >= a.adapters;
  if (bare && a.out == a.base) return;
  const int lane = threadIdx.x & 63, m = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t token = members[min(m, count - 1)];
  const int o0 = (blockIdx.y * kOneWaves + wave) * kColumns;
  u32x4 base[2], w[4] = {};
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const int o = o0 + 32 * s + kUnit * q;
    if (o < a.outputs) base[s] = load16(a.base + token * a.base_stride + o);
  }
  f32x4 sum[4] = {};
  if (!bare) {
    // (outputs past the last are its again, and not stored)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t o = min(o0 + output_of(i, m), a.outputs - 1);
      if (kUnit * q < a.rank) w[i] = load16(a.decoder + (static_cast<int64_t>(adapter) * a.outputs + o) * a.rank + kUnit * q);
    }
    const uint16_t *row[kLoads];
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int r = min(8 * j + lane / 8, a.rank - 1), t = min(8 * (j - 2 * kTiles) + lane / 8, count - 1);
      if (j < 2 * kTiles) row[j] = a.encoder + (static_cast<int64_t>(adapter) * a.rank + r) * a.hidden;
      else row[j] = a.x + static_cast<int64_t>(members[t]) * a.x_stride;
      row[j] += kUnit * (lane % 8);
    }
    f32x4 d[1][kTiles] = {};
    staged_product<kTiles, 1>(stage[wave], row, 64 * wave, a.hidden, 64 * kOneWaves, d);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kTiles; ++i) *reinterpret_cast<f32x4 *>(&sums[wave][i][m * 16 + 4 * q]) = d[0][i];
    __syncthreads();
    if (threadIdx.x < 8 * kTokens) {
      // thread = four ranks of a token; zeros behind the last rank
      const int t = threadIdx.x / 8, r = threadIdx.x % 8 * 4;
      const float scale = a.scales ? a.scales[adapter] : 1.0f;
      f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
      if (r < a.rank) {
#pragma unroll
        for (int k = 0; k < kOneWaves; ++k) v += *reinterpret_cast<const f32x4 *>(&sums[k][r / 16][t * 16 + r % 16]);
        v *= scale;
      }
      u32x2 part[kParts];
      split(v, part);
#pragma unroll
      for (int k = 0; k < kParts; ++k) *reinterpret_cast<u32x2 *>(&parts[k][t][r]) = part[k];
    }
    __syncthreads();
    u32x4 part[kParts];
#pragma unroll
    for (int k = 0; k < kParts; ++k) part[k] = load16(&parts[k][m][kUnit * q]);
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[i] = parts_product(w[i], part, sum[i]);
  }
  if (m >= count) return;
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const int o = o0 + 32 * s + kUnit * q;
    if (o < a.outputs)
      *reinterpret_cast<u32x4 *>(a.out + token * a.out_stride + o) = bare ? base[s] : added(base[s], sum, s);
  }
}

int64_t rounded(int64_t bytes) { return (bytes + 15) / 16 * 16; }

// Workgroups of a tile in the kernel of both products.
int one_pieces(int outputs) { return (outputs + kOneWaves * kColumns - 1) / (kOneWaves * kColumns); }

// Both products in one launch: what one compute unit takes from memory bounds it, a
// launch's end and start the two. A token of 2048 values, rank 8 / 16 / 32, 2048 outputs:
// 7.0 / 6.9 / 8.2 us against 8.2 / 8.4 / 8.8, of 4096 values and rank 32 10.0 against 9.3, of
// 8192 13.3 against 9.5. Rank 64 in two passes: 14.8 against 9.6. On the host a launch is
// 2.5 us.
//
// Its workgroups at work are to have room on the card together, two of rank 16 on a compute
// unit, one of rank 32: each forms v again. 64 tokens of as many adapters, rank 32, to 4096 /
// 8192 / 16384 outputs: 9.3 / 16.8 / 29 us against 10.6 / 14.3 / 18; rank 16 7.3 / 12.3 / 22
// against 9.7 / 13.0 / 15.4. The others only find no tile: 300 / 700 / 1000 tokens of 16
// adapters, rank 16, 1024 values and outputs 7.7 / 10.1 / 13.5 against 12.6 / 13.2 / 13.3.
bool one_launch(int tokens, int hidden, int outputs, int rank, int adapters) {
  if (rank > kOneRank || hidden * rank > kOneValues) return false;
  const int64_t pieces = one_pieces(outputs), tiles = tokens / kTokens + adapters + 1;
  return tokens * pieces <= kOneGroups && (tokens < tiles ? tokens : tiles) * pieces <= (rank <= 16 ? 512 : 256);
}

// With two launches a workgroup of few tokens reads all slots to find its tile, and one is
// launched for every token; the sort is a launch of its own. 250 tokens of 8 adapters of rank
// 64 (2816 to 1408 values) take 19 us either way, 512 of 8 adapters of rank 32 26 and 17.
bool sorts(int tokens) { return tokens > kFewTokens; }

// Workgroups share the hidden dimension in whole turns of 256 values: of few tokens 16 of them
// at most, of many two, whose parts the second launch reads again for every 256 outputs or
// more. Each has as many turns but the last, so that 17 turns are shared by nine.
// 1 / 2 / 4 of them: 4001 tokens of rank 64 (2048 to 4096 values) 38.7 / 37.4 / 39.2 us, 1000 of
// rank 32 (2048 to 2048) 20.6 / 17.3 / 16.0, 1500 of rank 128 (4096 to 4096) 43.9 / 39.8 / 42.7.
int splits_of(int tokens, int hidden) {
  const int turns = (hidden + kTurn - 1) / kTurn, most = sorts(tokens) ? kManySplits : kFewSplits;
  const int each = (turns + most - 1) / most;
  return (turns + each - 1) / each;
}

}  // namespace
}  // namespace cfmoe

extern "C" {

using namespace cfmoe;

CFMOE_API int64_t cfmoe_apply_adapters_scratch_bytes(int32_t hidden_size, int32_t outputs, int32_t rank, int32_t adapters,
                                                     int32_t tokens, int32_t out_is_hidden) {
  if (rank < 8 || rank > kMaxRank || rank % 8) return -fail(CFMOE_EINVAL, "apply_adapters needs a rank that is a multiple of 8, at most 256");
  if (adapters < 1 || adapters > kMaxAdapters) return -fail(CFMOE_EINVAL, "apply_adapters needs 1 to 4096 adapters");
  if (tokens < 0 || tokens > (1 << 24)) return -fail(CFMOE_EINVAL, "apply_adapters needs 0 to 2^24 tokens");
  if (hidden_size < 8 || hidden_size > kMaxSize || hidden_size % 8 || outputs < 8 || outputs > kMaxSize || outputs % 8)
    return -fail(CFMOE_EINVAL, "apply_adapters needs hidden and output sizes that are multiples of 8, at most 65536");
  if (!out_is_hidden && one_launch(tokens, hidden_size, outputs, rank, adapters)) return 0;
  int64_t bytes = splits_of(tokens, hidden_size) * static_cast<int64_t>(tokens) * rank * 4;
  if (sorts(tokens))
    bytes += rounded(4 * (adapters + 1)) + 2 * rounded(4 * static_cast<int64_t>(tokens)) +
             cfmoe_sort_by_expert_scratch_bytes(tokens, 1, adapters);
  return bytes;
}

CFMOE_API int cfmoe_apply_adapters(int32_t hidden_size, int32_t outputs, int32_t rank, int32_t adapters, uint32_t flags,
                                   const void *base, int64_t base_stride, const void *hidden, int64_t hidden_stride,
                                   const void *encoder, const void *decoder, const void *slots, const float *scales,
                                   void *out, int64_t out_stride, void *scratch, int32_t tokens, cfmoe_stream stream) {
  const int64_t bytes = cfmoe_apply_adapters_scratch_bytes(hidden_size, outputs, rank, adapters, tokens, out == hidden);
  if (bytes < 0) return static_cast<int>(-bytes);
  if (base_stride % 8 || hidden_stride % 8 || out_stride % 8 || base_stride < 0 || hidden_stride < 0 || out_stride < outputs)
    return fail(CFMOE_EINVAL, "apply_adapters needs row strides that are multiples of 8");
  if (tokens == 0) return 0;
  if (!base || !hidden || !encoder || !decoder || !slots || !out || (bytes && !scratch)) return fail(CFMOE_EINVAL, "NULL argument");
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
  a.splits = splits_of(tokens, hidden_size);
  // (whole turns: a split ends where the next begins)
  a.share = (hidden_size + a.splits * kTurn - 1) / (a.splits * kTurn) * kTurn;
  const int tiles = (rank + 15) / 16;
  if (bytes == 0) {
    const dim3 grid(tokens, one_pieces(outputs));
    hipLaunchKernelGGL(tiles == 1 ? adapter_one_kernel<1> : adapter_one_kernel<2>, grid, dim3(64 * kOneWaves), 0, stream, a);
    return check_launch("adapter_one");
  }
  const bool sorted = sorts(tokens);
  const int tile = sorted ? kManyTokens : kTokens;
  int most = tokens;  // tiles there can be
  if (sorted) {
    char *at = static_cast<char *>(scratch) + static_cast<int64_t>(a.splits) * tokens * rank * 4;
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
    // one more than whole ones for each adapter, and for the tokens without one
    most = tokens / tile + (adapters + 1 < tokens ? adapters + 1 : tokens);
    if (most > tokens) most = tokens;
  }
  const dim3 block(64 * kWaves);
  const int held = !sorted || tiles == 1 ? 1 : tiles == 2 ? 2 : 4;
  auto start = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(most, (tiles + held - 1) / held, a.splits), block, 0, stream, a);
    return check_launch("adapter_inner");
  };
  if (int rc = !sorted     ? start(adapter_inner_kernel<false, 1>)
               : held == 1 ? start(adapter_inner_kernel<true, 1>)
               : held == 2 ? start(adapter_inner_kernel<true, 2>)
                           : start(adapter_inner_kernel<true, 4>))
    return rc;
  // (4001 tokens of 5 adapters to 4096 outputs: 37.4 us with 1048 workgroups, 42.4 with 2096)
  int columns = (outputs + kWaves * kColumns - 1) / (kWaves * kColumns);
  while (columns > 1 && static_cast<int64_t>(most) * columns > kMostGroups) columns = (columns + 1) / 2;
  const unsigned lds = kParts * tile * parts_row(rank) * 2;
  auto finish = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(most, columns), block, lds, stream, a);
    return check_launch("adapter_out");
  };
  if (rank <= 32) return finish(sorted ? adapter_out_kernel<true, true> : adapter_out_kernel<false, true>);
  return finish(sorted ? adapter_out_kernel<true, false> : adapter_out_kernel<false, false>);
}

}  // extern "C"
