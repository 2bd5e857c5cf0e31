// MI355X (gfx950) router of one MoE layer: hidden rows to expert ids and weights.
//
//   l[t, e] = sum_h x[t, h] r[e, h]                        (x, r BF16)
//   ids[t, :] = the K experts of largest l, largest first; equal logits go to the
//               lowest expert, a NaN counts as larger than any number
//   weights[t, k] = exp(l_k - l_0) / sum_{j < K} exp(l_j - l_0)   (CFMOE_RENORMALISE)
//                   exp(l_k - l_0) / sum_e exp(l_e - l_0)         (otherwise)
//                   times expert_scale[ids[t, k]] where it is given
//
// The ids are those of the exact logits. A first launch forms FP32 logits by matrix
// instructions (router_logits_kernel, router_bulk_kernel for many tokens), and with
// the same operands' magnitudes a bound on how far an FP32 sum can be off;
// router_select_kernel recomputes in FP64 those logits whose order the bound leaves
// open.

#include "cfmoe_device.h"

namespace cfmoe {
namespace {

constexpr int kMaxExperts = 1024;
constexpr int kMaxTop = 64;
constexpr int kMaxHidden = 65536;  // (offsets into the router's rows are 32 bits)
constexpr int kTile = 16;          // experts, and tokens, of a matrix instruction
constexpr int kSplitWaves = 16;    // waves that share a tile's hidden dimension
constexpr int kBulkWaves = 16;     // of a bulk workgroup, two to an expert tile
constexpr int kBulkTokens = 32;
constexpr int kBulkHidden = 2048;  // hidden values in LDS at a time
constexpr int kSelectWaves = 4;    // tokens of a selecting workgroup
constexpr int kPerLane = kMaxExperts / 64;

struct RouteArgs {
  const uint16_t *x, *router;
  const float *expert_scale;
  void *ids, *weights;
  float *logits;     // [T, E]
  float *magnitude;  // [T, expert tiles]: largest sum_h |x r| of the tile's experts
  int hidden, experts, top_k, tokens, tiles, chain;
  bool ids64, weights16, renormalise;
};

__device__ __forceinline__ u32x4 magnitudes(u32x4 v) { return v & 0x7fff7fffu; }

// One tile's logits and the largest of its magnitude sums, for token t of `logits` and
// `magnitude`.
__device__ __forceinline__ void store_logits(const RouteArgs &a, float *logits, float *magnitude, int tile, int t,
                                             f32x4 dot, f32x4 size) {
  const int lane = threadIdx.x & 63, e0 = tile * kTile + lane / 16 * 4;
  // (fmaxf drops a NaN: a row whose magnitudes hold one has NaN logits, which the
  // selection ranks without a bound)
  float largest = fmaxf(fmaxf(size[0], size[1]), fmaxf(size[2], size[3]));
  largest = fmaxf(largest, __shfl_xor(largest, 16));
  largest = fmaxf(largest, __shfl_xor(largest, 32));
  if (t >= a.tokens) return;
  float *out = logits + static_cast<int64_t>(t) * a.experts + e0;
  if (a.experts % 4 == 0) {
    if (e0 < a.experts) *reinterpret_cast<f32x4 *>(out) = dot;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (e0 + i < a.experts) out[i] = dot[i];
  }
  if (lane < 16) magnitude[static_cast<int64_t>(t) * a.tiles + tile] = largest;
}

// The products of steps first, first + stride, .. of a tile's 32-blocks of the hidden
// dimension, four loads ahead.
__device__ __forceinline__ void accumulate(const u32x4 *r, const u32x4 *x, int first, int stride, int steps, f32x4 &dot,
                                           f32x4 &size) {
  constexpr int kAhead = 4;
  for (int s = first; s < steps; s += kAhead * stride) {
    u32x4 rv[kAhead], xv[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int at = min(s + i * stride, steps - 1);
      rv[i] = r[4 * at];
      xv[i] = x[4 * at];
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (s + i * stride >= steps) break;
      dot = mma(rv[i], xv[i], dot);
      size = mma(magnitudes(rv[i]), magnitudes(xv[i]), size);
    }
  }
}

// Few tiles: workgroup = 16 experts x 16 tokens, its waves every sixteenth 32 of the
// hidden dimension, so that one token's router is read by as many loads at once as it
// has (one workgroup for all experts, and the selection behind a barrier, took 20.7 us
// for 128 experts of 2048 where these two launches take 5.2 and 2.7). Latency bounds it:
// the router is 0.5 MB, 0.1 us of HBM.
__global__ __launch_bounds__(64 * kSplitWaves) void router_logits_kernel(RouteArgs a) {
  __shared__ f32x4 sums[2][kSplitWaves][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tile = blockIdx.x % a.tiles, token0 = blockIdx.x / a.tiles * kTile;
  const int row = min(tile * kTile + lane % 16, a.experts - 1);
  const int token = min(token0 + lane % 16, a.tokens - 1);
  const u32x4 *r = reinterpret_cast<const u32x4 *>(a.router + static_cast<int64_t>(row) * a.hidden) + lane / 16;
  const u32x4 *x = reinterpret_cast<const u32x4 *>(a.x + static_cast<int64_t>(token) * a.hidden) + lane / 16;
  f32x4 dot = {0, 0, 0, 0}, size = {0, 0, 0, 0};
  accumulate(r, x, wave, kSplitWaves, a.hidden / 32, dot, size);
  sums[0][wave][lane] = dot;
  sums[1][wave][lane] = size;
  __syncthreads();
  if (wave) return;
#pragma unroll
  for (int w = 1; w < kSplitWaves; ++w) dot += sums[0][w][lane], size += sums[1][w][lane];
  store_logits(a, a.logits, a.magnitude, tile, token0 + lane % 16, dot, size);
}

// Many tiles: workgroup = 32 tokens x 128 experts, two waves to 16 of the experts, each
// with half of the hidden dimension. The tokens' rows pass through LDS, 256 values of
// either half a stage; the loads of all 2048 of a span leave at once and each stage is
// written when its turn comes, so that only the first is waited for. Each wave streams
// its experts' rows past them. 19 us at 1500 tokens of 256 experts of 2048, 23 at 4001,
// where the products alone are 3.4: no rate of the chip bounds it (640 KB a workgroup
// from L2 are 13 bytes a clock). A workgroup fills a compute unit and its waves wait for
// each other at every stage, and half of the matrix work is the bound's magnitudes.
// (64 tokens to a workgroup leave too few workgroups; rows of another stride than
// 4 KB measured the same.)
__global__ __launch_bounds__(64 * kBulkWaves, 4) void router_bulk_kernel(RouteArgs a) {
  constexpr int kCols = kBulkTokens / kTile, kStage = 8, kStages = kBulkHidden / 64 / kStage;
  constexpr int kUnits = kStage * 4;                                   // 16 bytes of a half row's stage
  constexpr int kPart = kBulkTokens * 2 * kUnits / (64 * kBulkWaves);  // of a stage a thread brings
  constexpr int kStride = 2 * kUnits * 16 + 16;  // (equal places of 16 rows in different banks)
  constexpr int kGroup = kBulkWaves / 2;
  __shared__ __align__(16) uint8_t rows[2][kBulkTokens * kStride];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int groups = (a.tiles + kGroup - 1) / kGroup, half = wave / kGroup;
  const int tile = blockIdx.x % groups * kGroup + wave % kGroup, token0 = blockIdx.x / groups * kBulkTokens;
  const uint32_t lane_row = min(tile * kTile + lane % 16, a.experts - 1) * a.hidden * 2 + lane / 16 * 16;
  f32x4 dot[kCols], size[kCols];
#pragma unroll
  for (int n = 0; n < kCols; ++n) dot[n] = size[n] = f32x4{0, 0, 0, 0};
  for (int h0 = 0; h0 < a.hidden; h0 += kBulkHidden) {
    const int steps = min(kBulkHidden, a.hidden - h0) / 64;  // of a half
    const uint8_t *r = reinterpret_cast<const uint8_t *>(a.router) + (h0 + half * steps * 32) * 2;
    u32x4 brought[kStages][kPart], ring[kStage];
#pragma unroll
    for (int i = 0; i < kStage; ++i) ring[i] = *reinterpret_cast<const u32x4 *>(r + 64 * min(i, steps - 1) + lane_row);
#pragma unroll
    for (int c = 0; c < kStages; ++c)
#pragma unroll
      for (int j = 0; j < kPart; ++j) {
        const int i = threadIdx.x + j * 64 * kBulkWaves, token = min(token0 + i / (2 * kUnits), a.tokens - 1);
        // (past the half its end comes again: not multiplied)
        const int at = i / kUnits % 2 * steps * 4 + min(c * kUnits + i % kUnits, steps * 4 - 1);
        brought[c][j] = reinterpret_cast<const u32x4 *>(a.x + static_cast<int64_t>(token) * a.hidden + h0)[at];
      }
#pragma unroll
    for (int c = 0; c < kStages; ++c) {
      if (c * kStage >= steps) break;
#pragma unroll
      for (int j = 0; j < kPart; ++j) {
        const int i = threadIdx.x + j * 64 * kBulkWaves;
        *reinterpret_cast<u32x4 *>(rows[c & 1] + i / (2 * kUnits) * kStride + i % (2 * kUnits) * 16) = brought[c][j];
      }
      // (two buffers: the one written next was read before this barrier)
      __syncthreads();
      const uint8_t *x = rows[c & 1] + lane % 16 * kStride + half * kUnits * 16 + lane / 16 * 16;
#pragma unroll
      for (int i = 0; i < kStage; ++i) {
        // (a step past the half is multiplied by cleared weights: no branch splits the
        // stage's reads)
        const u32x4 rv = ring[i] & (c * kStage + i < steps ? ~0u : 0u), rm = magnitudes(rv);
        ring[i] = *reinterpret_cast<const u32x4 *>(r + 64 * min((c + 1) * kStage + i, steps - 1) + lane_row);
#pragma unroll
        for (int n = 0; n < kCols; ++n) {
          const u32x4 xv = *reinterpret_cast<const u32x4 *>(x + n * kTile * kStride + i * 64);
          dot[n] = mma(rv, xv, dot[n]);
          size[n] = mma(rm, magnitudes(xv), size[n]);
        }
      }
    }
    __syncthreads();
  }
  // the halves' sums
  f32x4 *other = reinterpret_cast<f32x4 *>(rows[0]) + (wave % kGroup * 2 * kCols) * 64 + lane;
  if (half)
#pragma unroll
    for (int n = 0; n < kCols; ++n) other[2 * n * 64] = dot[n], other[(2 * n + 1) * 64] = size[n];
  __syncthreads();
  if (half || tile >= a.tiles) return;
#pragma unroll
  for (int n = 0; n < kCols; ++n)
    store_logits(a, a.logits, a.magnitude, tile, token0 + n * kTile + lane % 16, dot[n] + other[2 * n * 64],
                 size[n] + other[(2 * n + 1) * 64]);
}

// Order of the logits as unsigned integers: -0 equals 0, NaN above all; no logit's is 0.
__device__ __forceinline__ uint32_t order_key(float v) {
  if (v != v) return ~0u;
  const uint32_t bits = __float_as_uint(v + 0.0f);
  return bits >> 31 ? ~bits : bits | 0x80000000u;
}

__device__ __forceinline__ float key_value(uint32_t key) {
  return key == ~0u ? NAN : __uint_as_float(key >> 31 ? key & 0x7fffffffu : ~key);
}

__device__ __forceinline__ uint64_t order_key(double v) {
  if (v != v) return ~0ull;
  const uint64_t bits = __builtin_bit_cast(uint64_t, v + 0.0);
  return bits >> 63 ? ~bits : bits | (1ull << 63);
}

template <int kControl, class T>
__device__ __forceinline__ T moved(T v) {
  return __builtin_bit_cast(T, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), kControl, 0xf, 0xf, true));
}

// A wave's result in every lane: 16 lanes by lane moves (neighbours, pairs, half row
// and row mirrored), the four rows by scalars.
template <class T, class Op>
__device__ __forceinline__ T wave_all(T v, Op op) {
  v = op(v, moved<0xb1>(v));
  v = op(v, moved<0x4e>(v));
  v = op(v, moved<0x141>(v));
  v = op(v, moved<0x140>(v));
  T rows[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    rows[i] = __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 16 * i));
  return op(op(rows[0], rows[1]), op(rows[2], rows[3]));
}

__device__ __forceinline__ float wave_sum(float v) {
  return wave_all(v, [](float a, float b) { return a + b; });
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int m = 1; m < 64; m *= 2) v += __shfl_xor(v, m);
  return v;
}

// Exact dot products of token t's row with two experts' (BF16 products fit FP64 with
// bits to spare; a sum of some thousand is off by less than 2^-40 of its terms).
__device__ __forceinline__ void exact_logits(const RouteArgs &a, int t, int first, int second, double &d0, double &d1) {
  const int lane = threadIdx.x & 63;
  const u32x4 *x = reinterpret_cast<const u32x4 *>(a.x + static_cast<int64_t>(t) * a.hidden);
  const u32x4 *r0 = reinterpret_cast<const u32x4 *>(a.router + static_cast<int64_t>(first) * a.hidden);
  const u32x4 *r1 = reinterpret_cast<const u32x4 *>(a.router + static_cast<int64_t>(second) * a.hidden);
  d0 = d1 = 0.0;
#pragma unroll 2
  for (int i = lane; i < a.hidden / 8; i += 64) {
    const u32x4 xv = x[i], v0 = r0[i], v1 = r1[i];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const double low = bf16_value(xv[w] & 0xffffu), high = __uint_as_float(xv[w] & 0xffff0000u);
      d0 = fma(low, static_cast<double>(bf16_value(v0[w] & 0xffffu)), d0);
      d0 = fma(high, static_cast<double>(__uint_as_float(v0[w] & 0xffff0000u)), d0);
      d1 = fma(low, static_cast<double>(bf16_value(v1[w] & 0xffffu)), d1);
      d1 = fma(high, static_cast<double>(__uint_as_float(v1[w] & 0xffff0000u)), d1);
    }
  }
  d0 = wave_sum(d0);
  d1 = wave_sum(d1);
}

// The `count` largest of the lanes' values (expert 64 j + lane), largest first, ties
// to the lowest expert; the i-th lands in lane i.
template <int kValues>
__device__ __forceinline__ void select(const float (&v)[kValues], int experts, int count, int lane, float &value,
                                       int &expert) {
  uint32_t key[kValues];
#pragma unroll
  for (int j = 0; j < kValues; ++j) key[j] = 64 * j + lane < experts ? order_key(v[j]) : 0;
  uint32_t kept = 0;
  expert = 0;
  for (int i = 0; i < count; ++i) {
    uint32_t best = key[0];
#pragma unroll
    for (int j = 1; j < kValues; ++j) best = max(best, key[j]);
    best = wave_all(best, [](uint32_t a, uint32_t b) { return max(a, b); });
    int at = 0;
#pragma unroll
    for (int j = kValues - 1; j >= 0; --j) {
      const uint64_t equal = __ballot(key[j] == best);
      if (equal) at = 64 * j + __builtin_ctzll(equal);
    }
#pragma unroll
    for (int j = 0; j < kValues; ++j)
      if (at == 64 * j + lane) key[j] = 0;
    if (lane == i) kept = best, expert = at;
  }
  value = key_value(kept);
}

// The same by FP64 values, for rows whose order FP32 leaves open.
template <int kValues>
__device__ __forceinline__ void select(const double (&v)[kValues], int experts, int count, int lane, double &value,
                                       int &expert) {
  uint64_t key[kValues];
#pragma unroll
  for (int j = 0; j < kValues; ++j) key[j] = 64 * j + lane < experts ? order_key(v[j]) : 0;
  value = 0.0;
  expert = 0;
  for (int i = 0; i < count; ++i) {
    uint64_t best = 0;
#pragma unroll
    for (int j = 0; j < kValues; ++j) best = max(best, key[j]);
#pragma unroll
    for (int m = 1; m < 64; m *= 2) best = max(best, static_cast<uint64_t>(__shfl_xor(best, m)));
    int at = 0;
#pragma unroll
    for (int j = kValues - 1; j >= 0; --j) {
      const uint64_t equal = __ballot(key[j] == best);
      if (equal) at = 64 * j + __builtin_ctzll(equal);
    }
    double found = 0.0;
#pragma unroll
    for (int j = 0; j < kValues; ++j)
      if (at == 64 * j + lane) {
        found = v[j];
        key[j] = 0;
      }
    found = __shfl(found, at & 63);
    if (lane == i) value = found, expert = at;
  }
}

// A wave's token t, by its logits `row` and the tiles' magnitudes.
template <int kValues>
__device__ __forceinline__ void select_token(const RouteArgs &a, int t, const float *row, const float *magnitude) {
  const int lane = threadIdx.x & 63;
  float v[kValues];
#pragma unroll
  for (int j = 0; j < kValues; ++j) v[j] = 64 * j + lane < a.experts ? row[64 * j + lane] : -INFINITY;
  const float size = lane < a.tiles ? magnitude[lane] : 0.0f;
  const float largest = wave_all(size, [](float a, float b) { return fmaxf(a, b); });
  // Each of the additions behind a logit rounds (or cuts off) by 2^-23 of a partial
  // sum of at most `largest` at the most; a term goes through at most `chain` of
  // them. Two logits may be off in opposite directions. (The last term covers
  // products below the normal range.)
  const float open = 2.0f * a.chain * 0x1p-23f * largest + 0x1p-110f;

  // the K + 1 largest by FP32, and those whose order with a neighbour is open
  const int wanted = min(a.top_k + 1, a.experts), most = min(wanted, 64);
  float value32;
  int expert;
  select<kValues>(v, a.experts, most, lane, value32, expert);
  const float next = __shfl_down(value32, 1);
  // (written so that a NaN or infinity in between counts as open, and so does a single
  // expert's where FP32 may have overflowed; 64 kept of more: what follows them was not
  // looked at, so that each of those is formed again in FP64, where 63 kept form only the
  // open ones: one token of 128 experts 74 us against 24)
  const bool unsure = (lane + 1 < most && !(value32 - next > open)) || most < wanted || (lane == 0 && !(open < INFINITY));
  const uint64_t unsure_lanes = __ballot(unsure);
  double value = value32;
  // The softmax over all experts adds up FP32 logits, unless some may have overflowed.
  // All are open then: their exact values are in the lanes, or v has them less the first.
  bool overflowed = false;
  if (unsure_lanes != 0) {
    overflowed = !(open < INFINITY);
    const float cut = __shfl(value32, a.top_k - 1);
    int near = 0;  // experts that are kept or might be
#pragma unroll
    for (int j = 0; j < kValues; ++j)
      near += __builtin_popcountll(__ballot(64 * j + lane < a.experts && !(cut - v[j] > open)));
    if (near <= most && most == wanted) {
      // All of them are at hand: the exact logits of the open ones, then each one's
      // rank among the K + 1. (Others are further from their neighbours than either
      // may be off, so their FP32 logits rank right among exact ones.)
      uint64_t todo = unsure_lanes | unsure_lanes << 1;
      while (todo) {
        const int i = __builtin_ctzll(todo);
        todo &= todo - 1;
        const int j = todo ? __builtin_ctzll(todo) : i;
        todo &= todo - 1;
        double di, dj;
        exact_logits(a, t, __builtin_amdgcn_readlane(expert, i), __builtin_amdgcn_readlane(expert, j), di, dj);
        if (lane == i) value = di;
        if (lane == j) value = dj;
      }
      const uint64_t mine = order_key(value);
      int rank = 0;
      for (int j = 0; j < most; ++j) {
        const uint64_t theirs = __shfl(mine, j);
        const int other = __builtin_amdgcn_readlane(expert, j);
        rank += theirs > mine || (theirs == mine && other < expert);
      }
      double ranked = 0.0;
      int ranked_expert = 0;
      for (int j = 0; j < most; ++j) {
        const int to = __builtin_amdgcn_readlane(rank, j), from = __builtin_amdgcn_readlane(expert, j);
        const double moved_value = __shfl(value, j);
        if (lane == to) ranked = moved_value, ranked_expert = from;
      }
      value = ranked;
      expert = ranked_expert;
    } else {
      // more experts lie about the cut: the exact logits of all that might be kept
      double exact[kValues];
#pragma unroll
      for (int j = 0; j < kValues; ++j) {
        exact[j] = v[j];
        uint64_t todo = __ballot(64 * j + lane < a.experts && !(cut - v[j] > open));
        while (todo) {
          const int i = __builtin_ctzll(todo);
          todo &= todo - 1;
          const int k = todo ? __builtin_ctzll(todo) : i;
          todo &= todo - 1;
          double di, dk;
          exact_logits(a, t, 64 * j + i, 64 * j + k, di, dk);
          if (lane == i) exact[j] = di;
          if (lane == k) exact[j] = dk;
        }
      }
      select<kValues>(exact, a.experts, a.top_k, lane, value, expert);
      const double first = __shfl(value, 0);
#pragma unroll
      for (int j = 0; j < kValues; ++j) v[j] = overflowed ? static_cast<float>(exact[j] - first) : v[j];
    }
  }

  const double first = __shfl(value, 0);
  const float share = lane < a.top_k ? expf(static_cast<float>(value - first)) : 0.0f;
  float total;
  if (a.renormalise) {
    total = wave_sum(share);
  } else {
    float part = 0.0f;
    if (overflowed && a.experts <= most) {
      part = lane < a.experts ? expf(static_cast<float>(value - first)) : 0.0f;
    } else {
#pragma unroll
      for (int j = 0; j < kValues; ++j)
        part += 64 * j + lane < a.experts ? expf(overflowed ? v[j] : static_cast<float>(v[j] - first)) : 0.0f;
    }
    total = wave_sum(part);
  }
  if (lane >= a.top_k) return;
  float weight = share / total;
  if (a.expert_scale) weight *= a.expert_scale[expert];
  const int64_t at = static_cast<int64_t>(t) * a.top_k + lane;
  if (a.ids64) static_cast<int64_t *>(a.ids)[at] = expert;
  else static_cast<int32_t *>(a.ids)[at] = expert;
  if (a.weights16) static_cast<uint16_t *>(a.weights)[at] = bf16_bits(weight);
  else static_cast<float *>(a.weights)[at] = weight;
}

// Wave = one token. FP32 logits decide almost all orders; the FP64 dot products of those
// left open are what a call of many tokens pays for ids that do not depend on how a sum
// was split (9 us of 32 at 4001 tokens of 256 experts).
template <int kValues>
__global__ __launch_bounds__(64 * kSelectWaves) void router_select_kernel(RouteArgs a) {
  const int t = blockIdx.x * kSelectWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (t < a.tokens)
    select_token<kValues>(a, t, a.logits + static_cast<int64_t>(t) * a.experts,
                          a.magnitude + static_cast<int64_t>(t) * a.tiles);
}

}  // namespace
}  // namespace cfmoe

extern "C" {

using namespace cfmoe;

CFMOE_API int64_t cfmoe_route_scratch_bytes(int32_t tokens, int32_t experts) {
  if (tokens < 0 || experts < 1 || experts > kMaxExperts) return -fail(CFMOE_EINVAL, "route needs 1 to 1024 experts");
  const int64_t tiles = (experts + kTile - 1) / kTile;
  return static_cast<int64_t>(tokens) * (experts + tiles) * 4;
}

CFMOE_API int cfmoe_route(int32_t hidden_size, int32_t experts, int32_t top_k, uint32_t flags, const void *hidden,
                          const void *router, const float *expert_scale, void *ids, void *weights,
                          void *scratch, int32_t tokens, cfmoe_stream stream) {
  if (hidden_size <= 0 || hidden_size % 128 || hidden_size > kMaxHidden)
    return fail(CFMOE_EINVAL, "route needs a hidden size that is a multiple of 128, at most 65536");
  if (experts < 1 || experts > kMaxExperts) return fail(CFMOE_EINVAL, "route needs 1 to 1024 experts");
  if (top_k < 1 || top_k > kMaxTop || top_k > experts)
    return fail(CFMOE_EINVAL, "route keeps 1 to 64 experts, no more than there are");
  if (tokens < 0) return fail(CFMOE_EINVAL, "route needs a token count of zero or more");
  if (tokens == 0) return 0;
  if (!hidden || !router || !ids || !weights || !scratch) return fail(CFMOE_EINVAL, "NULL argument");
  if ((reinterpret_cast<uintptr_t>(hidden) | reinterpret_cast<uintptr_t>(router) |
       reinterpret_cast<uintptr_t>(scratch)) % 16)
    return fail(CFMOE_EINVAL, "route needs 16-byte aligned hidden rows, router and scratch");
  RouteArgs a;
  a.x = static_cast<const uint16_t *>(hidden);
  a.router = static_cast<const uint16_t *>(router);
  a.expert_scale = expert_scale;
  a.ids = ids;
  a.weights = weights;
  a.tiles = (experts + kTile - 1) / kTile;
  a.logits = static_cast<float *>(scratch);
  a.magnitude = a.logits + static_cast<int64_t>(tokens) * experts;
  a.hidden = hidden_size;
  a.experts = experts;
  a.top_k = top_k;
  a.tokens = tokens;
  a.ids64 = flags & CFMOE_IDS_INT64;
  a.weights16 = flags & CFMOE_WEIGHTS_BF16;
  a.renormalise = flags & CFMOE_RENORMALISE;
  const int64_t tiles = a.tiles * ((static_cast<int64_t>(tokens) + kTile - 1) / kTile);
  if (tiles > 0x1fffff) return fail(CFMOE_EINVAL, "route has too many tokens for one launch");
  // The few-tile kernel reads the router's rows once for 16 tokens, the bulk one for 32
  // from more of the chip's caches, but a workgroup of its takes 18 us however few there
  // are: at 600 tokens of 256 experts (608 tiles) 20.6 us against 25.4, at 1024 of 128
  // (512) 18.2 against 25.3, at 2048 of 128 (1024) 25.8 against 26.4, at 1500 of 256
  // (1504) 33.2 against 27.7, at 3000 of 128 (1504) 33.0 against 26.6, with the selection.
  // `chain`: 32 products inside a matrix instruction, one addition for each of a chain
  // of them, and the waves' sums.
  if (tiles <= 1024) {
    a.chain = 32 + (hidden_size / 32 + kSplitWaves - 1) / kSplitWaves + kSplitWaves;
    hipLaunchKernelGGL(router_logits_kernel, dim3(static_cast<unsigned>(tiles)), dim3(64 * kSplitWaves), 0, stream, a);
  } else {
    a.chain = 32 + hidden_size / 64 + 1;
    const int groups = (a.tiles + kBulkWaves / 2 - 1) / (kBulkWaves / 2) * ((tokens + kBulkTokens - 1) / kBulkTokens);
    hipLaunchKernelGGL(router_bulk_kernel, dim3(groups), dim3(64 * kBulkWaves), 0, stream, a);
  }
  if (int rc = check_launch("router_logits")) return rc;
  auto select = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((tokens + kSelectWaves - 1) / kSelectWaves), dim3(64 * kSelectWaves), 0, stream, a);
  };
  if (experts <= 64) select(router_select_kernel<1>);
  else if (experts <= 128) select(router_select_kernel<2>);
  else if (experts <= 256) select(router_select_kernel<4>);
  else select(router_select_kernel<kPerLane>);
  return check_launch("router_select");
}

}  // extern "C"
