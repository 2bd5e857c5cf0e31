// MI355X (gfx950) router of one MoE layer: hidden rows to expert ids and weights.
//
//   l[t, e] = sum_h x[t, h] r[e, h]                        (x, r BF16)
//   ids[t, :] = the K experts of largest l, largest first; equal logits go to the
//               lowest expert, a NaN counts as larger than any number
//   weights[t, k] = exp(l_k - l_0) / sum_{j < K} exp(l_j - l_0)   (CFMOE_RENORMALISE)
//                   exp(l_k - l_0) / sum_e exp(l_e - l_0)         (otherwise)
//                   times expert_scale[ids[t, k]] where it is given
//
// The ids are those of the exact logits. router_logits_kernel forms FP32 logits by
// matrix instructions, and with the same operands' magnitudes a bound on how far
// an FP32 sum can be off; router_select_kernel recomputes in FP64 those logits
// whose order the bound leaves open.

#include "cfmoe_device.h"

namespace cfmoe {
namespace {

constexpr int kMaxExperts = 1024;
constexpr int kMaxTop = 64;
constexpr int kTile = 16;             // experts, and tokens, of a tile
constexpr int kLogitWaves = 4;        // waves that share a tile's hidden dimension
constexpr int kSelectWaves = 4;       // tokens of a selecting workgroup
constexpr int kPerLane = kMaxExperts / 64;

struct RouteArgs {
  const uint16_t *x, *router;
  const float *expert_scale;
  void *ids, *weights;
  float *logits;     // [T, E]
  float *magnitude;  // [T, expert tiles]: largest sum_h |x r| of the tile's experts
  int hidden, experts, top_k, tokens, tiles;
  bool ids64, weights16, renormalise;
};

__device__ __forceinline__ u32x4 magnitudes(u32x4 v) { return v & 0x7fff7fffu; }

// Workgroup = 16 experts x 16 tokens, its waves a quarter of the hidden dimension
// each (every fourth 32-block of it).
__global__ __launch_bounds__(64 * kLogitWaves) void router_logits_kernel(RouteArgs a) {
  __shared__ f32x4 sums[2][kLogitWaves][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tile = blockIdx.x % a.tiles, token0 = blockIdx.x / a.tiles * kTile;
  const int row = min(tile * kTile + lane % 16, a.experts - 1);
  const int token = min(token0 + lane % 16, a.tokens - 1);
  const u32x4 *r = reinterpret_cast<const u32x4 *>(a.router + static_cast<int64_t>(row) * a.hidden) + lane / 16;
  const u32x4 *x = reinterpret_cast<const u32x4 *>(a.x + static_cast<int64_t>(token) * a.hidden) + lane / 16;
  f32x4 dot = {0, 0, 0, 0}, size = {0, 0, 0, 0};
#pragma unroll 4
  for (int s = wave; s < a.hidden / 32; s += kLogitWaves) {
    const u32x4 rv = r[4 * s], xv = x[4 * s];
    dot = mma(rv, xv, dot);
    size = mma(magnitudes(rv), magnitudes(xv), size);
  }
  sums[0][wave][lane] = dot;
  sums[1][wave][lane] = size;
  __syncthreads();
  if (wave) return;
#pragma unroll
  for (int w = 1; w < kLogitWaves; ++w) dot += sums[0][w][lane], size += sums[1][w][lane];
  const int e0 = tile * kTile + lane / 16 * 4, t = token0 + lane % 16;
  // (fmaxf drops a NaN: a row whose magnitudes hold one has NaN logits, which the
  // selection ranks without a bound)
  float largest = fmaxf(fmaxf(size[0], size[1]), fmaxf(size[2], size[3]));
  largest = fmaxf(largest, __shfl_xor(largest, 16));
  largest = fmaxf(largest, __shfl_xor(largest, 32));
  if (t >= a.tokens) return;
  float *out = a.logits + static_cast<int64_t>(t) * a.experts;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (e0 + i < a.experts) out[e0 + i] = dot[i];
  if (lane < 16) a.magnitude[static_cast<int64_t>(t) * a.tiles + tile] = largest;
}

// Order of the logits as unsigned integers: -0 equals 0, NaN above all.
__device__ __forceinline__ uint64_t order_key(double v) {
  if (v != v) return ~0ull;
  const uint64_t bits = __builtin_bit_cast(uint64_t, v + 0.0);
  return bits >> 63 ? ~bits : bits | (1ull << 63);
}

__device__ __forceinline__ uint64_t wave_max(uint64_t v) {
#pragma unroll
  for (int m = 1; m < 64; m *= 2) {
    const uint64_t other = __shfl_xor(v, m);
    v = v > other ? v : other;
  }
  return v;
}

__device__ __forceinline__ int wave_min(int v) {
#pragma unroll
  for (int m = 1; m < 64; m *= 2) v = min(v, __shfl_xor(v, m));
  return v;
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int m = 1; m < 64; m *= 2) v = fmaxf(v, __shfl_xor(v, m));
  return v;
}

template <class T>
__device__ __forceinline__ T wave_sum(T v) {
#pragma unroll
  for (int m = 1; m < 64; m *= 2) v += __shfl_xor(v, m);
  return v;
}

// One selection: the `count` largest of the lanes' values (expert 64 j + lane),
// largest first, ties to the lowest expert; value and expert i land in lane i.
template <int kValues>
__device__ __forceinline__ void select(const double (&v)[kValues], int experts, int count, int lane,
                                       double &value, int &expert) {
  uint64_t key[kValues];
#pragma unroll
  for (int j = 0; j < kValues; ++j) key[j] = 64 * j + lane < experts ? order_key(v[j]) : 0;
  value = 0.0;
  expert = 0;
  for (int i = 0; i < count; ++i) {
    uint64_t best = 0;
#pragma unroll
    for (int j = 0; j < kValues; ++j) best = best > key[j] ? best : key[j];
    best = wave_max(best);
    int at = kMaxExperts;
#pragma unroll
    for (int j = kValues - 1; j >= 0; --j) at = key[j] == best ? 64 * j + lane : at;
    at = wave_min(at);
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

// Wave = one token.
template <int kValues>
__global__ __launch_bounds__(64 * kSelectWaves) void router_select_kernel(RouteArgs a) {
  const int lane = threadIdx.x & 63;
  const int t = blockIdx.x * kSelectWaves + (threadIdx.x >> 6);
  if (t >= a.tokens) return;
  const float *row = a.logits + static_cast<int64_t>(t) * a.experts;
  double v[kValues];
#pragma unroll
  for (int j = 0; j < kValues; ++j) v[j] = 64 * j + lane < a.experts ? row[64 * j + lane] : -INFINITY;
  float largest = 0.0f;
  for (int i = lane; i < a.tiles; i += 64)
    largest = fmaxf(largest, a.magnitude[static_cast<int64_t>(t) * a.tiles + i]);
  largest = wave_max(largest);
  // Each of the additions behind a logit rounds (or cuts off) by 2^-23 of a partial
  // sum of at most `largest` at the most: 32 inside a matrix instruction, one for
  // each instruction of a wave's chain, and the waves' own. Two logits may be off
  // in opposite directions. (The last term covers products below the normal range.)
  const int chain = (a.hidden / 32 + kLogitWaves - 1) / kLogitWaves;
  const double open = 2.0 * (32 + chain + kLogitWaves) * 0x1p-23 * largest + 0x1p-110;

  // the K + 1 largest by FP32, the smallest kept logit, and whose order is open
  const int wanted = min(a.top_k + 1, a.experts);
  const int most = min(wanted, 64);
  double value;
  int expert;
  select<kValues>(v, a.experts, most, lane, value, expert);
  const double cut = __shfl(value, a.top_k - 1);
  const double next = __shfl_down(value, 1);
  // (written so that a NaN or infinity in between counts as open)
  bool unsure = lane + 1 < most && !(value - next > open);
  if (most < wanted) unsure = true;  // (64 kept: what follows them was not looked at)
  if (__ballot(unsure) != 0) {
    // recompute every logit that lies within `open` of another that matters
    bool contested[kValues];
#pragma unroll
    for (int j = 0; j < kValues; ++j) contested[j] = 64 * j + lane < a.experts && !(cut - v[j] > open);
    const u32x4 *x = reinterpret_cast<const u32x4 *>(a.x + static_cast<int64_t>(t) * a.hidden);
#pragma unroll
    for (int j = 0; j < kValues; ++j) {
      uint64_t todo = __ballot(contested[j]);
      while (todo) {
        const int owner = __builtin_ctzll(todo);
        todo &= todo - 1;
        const u32x4 *r =
            reinterpret_cast<const u32x4 *>(a.router + static_cast<int64_t>(64 * j + owner) * a.hidden);
        double sum = 0.0;
        for (int i = lane; i < a.hidden / 8; i += 64) {
          const u32x4 rv = r[i], xv = x[i];
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            sum = fma(static_cast<double>(bf16_value(rv[w] & 0xffffu)),
                      static_cast<double>(bf16_value(xv[w] & 0xffffu)), sum);
            sum = fma(static_cast<double>(__uint_as_float(rv[w] & 0xffff0000u)),
                      static_cast<double>(__uint_as_float(xv[w] & 0xffff0000u)), sum);
          }
        }
        sum = wave_sum(sum);
        if (lane == owner) v[j] = sum;
      }
    }
    select<kValues>(v, a.experts, a.top_k, lane, value, expert);
  }

  const double first = __shfl(value, 0);
  const float share = lane < a.top_k ? expf(static_cast<float>(value - first)) : 0.0f;
  float total;
  if (a.renormalise) {
    total = wave_sum(share);
  } else {
    float part = 0.0f;
#pragma unroll
    for (int j = 0; j < kValues; ++j)
      part += 64 * j + lane < a.experts ? expf(static_cast<float>(v[j] - first)) : 0.0f;
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
  if (hidden_size <= 0 || hidden_size % 128) return fail(CFMOE_EINVAL, "route needs a hidden size that is a multiple of 128");
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
  const int64_t groups = static_cast<int64_t>(a.tiles) * ((tokens + kTile - 1) / kTile);
  if (groups > 0x7fffffffL / (64 * kLogitWaves)) return fail(CFMOE_EINVAL, "route has too many tokens for one launch");
  hipLaunchKernelGGL(router_logits_kernel, dim3(static_cast<unsigned>(groups)), dim3(64 * kLogitWaves), 0, stream, a);
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
