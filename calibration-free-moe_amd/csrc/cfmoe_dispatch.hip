// MI355X (gfx950): tokens laid out by expert, and back.
//
// A token t has K pairs (t, k) with expert ids[t, k]. A pair is kept where its id lies in
// [0, E) and its token is not padding. Rows are the kept pairs by expert, pairs of one
// expert in the batch's order, and behind them the dropped pairs, in that order too:
//
//   offsets[e]    first row of expert e; offsets[E] rows are kept
//   pairs[row]    t K + k of the row's pair
//   places[t, k]  row of the pair, or -1 - row of a dropped one
//
//   gather    rows[row] = x[t], 0 for dropped pairs
//   combine   out[t] = sum_k w[t, k] rows[place], kept pairs in slot order, FP32, rounded once
//   backward  of gather: dx[t] = sum_k drows[place], which is combine without weights
//             of combine: drows[place] = w[t, k] dout[t], 0 for dropped pairs,
//                         dw[t, k] = sum_h dout[t, h] rows[place, h]
//
// What a dropped pair's row or weight holds is never read, so it may hold a NaN.
//
// All but the order is one pass over rows, bound by memory. 4096 and 8191 tokens of eight
// BF16 rows of 2048, new ones each time: laid out 24 and 59 us (151 and 302 MB, 6.2 and 5.1
// TB/s), summed 26 and 58 (5.7 and 5.2), the sum's gradients 116 (570 MB, 4.9 TB/s). Rows
// that are read once are loaded past the caches, which keep the others: 8192 tokens, the
// same ones again and again, 73 -> 46 us the sum, 103 -> 87 its gradients; stores past them
// made a sum that follows slower (104 -> 112 both).

#include "cfmoe_rows.h"

namespace cfmoe {
namespace {

constexpr int kMaxExperts = 4096;
constexpr int kMaxTop = 64;
constexpr int64_t kMaxPairs = INT64_C(1) << 30;
constexpr int kSortWaves = 16;
constexpr int kSortBlocks = 64;       // workgroups that share the pairs of a large call
constexpr int kCountBytes = 63 << 10; // a workgroup's counts, per wave and expert
constexpr int kHeld = 4;              // keys of a lane that stay in registers
constexpr int kThreads = 256;
constexpr int kSlots = 8;             // rows of a token in flight at once

// ---------------------------------------------------------------------------
// order of the pairs

struct OrderArgs {
  const void *ids;
  const uint8_t *padding;
  int32_t *offsets, *places, *pairs;
  int32_t *counts;  // [workgroups, E + 1], or NULL where one workgroup has all pairs
  int pairs_total, top_k, experts;
  int range;  // pairs of one wave
  bool ids64;
};

__device__ __forceinline__ int key_of(const OrderArgs &a, int pair) {
  int64_t id = a.ids64 ? static_cast<const int64_t *>(a.ids)[pair] : static_cast<const int32_t *>(a.ids)[pair];
  if (a.padding && a.padding[pair / a.top_k]) id = a.experts;
  return id >= 0 && id < a.experts ? static_cast<int>(id) : a.experts;
}

// Pairs of this wave: [low, high).
__device__ __forceinline__ void range_of(const OrderArgs &a, int waves, int &low, int &high) {
  const int64_t first = (static_cast<int64_t>(blockIdx.x) * waves + (threadIdx.x >> 6)) * a.range;
  low = static_cast<int>(first < a.pairs_total ? first : a.pairs_total);
  high = static_cast<int>(first + a.range < a.pairs_total ? first + a.range : a.pairs_total);
}

// The first keys of the wave's range, -1 past its end.
__device__ __forceinline__ void hold_keys(const OrderArgs &a, int low, int high, int (&held)[kHeld]) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int j = 0; j < kHeld; ++j) held[j] = low + 64 * j + lane < high ? key_of(a, low + 64 * j + lane) : -1;
}

// Takes 64 keys, one a lane (-1: none), into the wave's running `next` rows of each key:
// lanes of one key find each other by a ballot for each of its bits, and each gets its key's
// next row and the number of its fellows in lower lanes. No atomic, so no order but the lanes'.
__device__ __forceinline__ int take_keys(const OrderArgs &a, int *next, int key) {
  const int lane = threadIdx.x & 63, bits = 32 - __builtin_clz(a.experts);
  const bool live = key >= 0;
  uint64_t fellows = __ballot(live);
  for (int b = 0; b < bits; ++b) {
    const uint64_t set = __ballot((key >> b) & 1);
    fellows &= (key >> b) & 1 ? set : ~set;
  }
  const int below = __builtin_popcountll(fellows & ((UINT64_C(1) << lane) - 1));
  int row = 0;
  // (the lanes of a wave read before its last fellow writes, in program order)
  if (live) row = next[key] + below;
  wave_in_step();
  if (live && below + 1 == __builtin_popcountll(fellows)) next[key] = row + 1;
  wave_in_step();
  return row;
}

// The keys' counts of each workgroup's pairs, for a call of several.
__global__ __launch_bounds__(64 * kSortWaves) void order_count_kernel(OrderArgs a) {
  extern __shared__ int shared[];
  const int width = a.experts + 1, waves = blockDim.x >> 6, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  int low, high, held[kHeld];
  range_of(a, waves, low, high);
  hold_keys(a, low, high, held);
  for (int i = threadIdx.x; i < waves * width; i += blockDim.x) shared[i] = 0;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kHeld; ++j)
    if (low + 64 * j < high) take_keys(a, shared + wave * width, held[j]);
  for (int p = low + 64 * kHeld; p < high; p += 64) take_keys(a, shared + wave * width, p + lane < high ? key_of(a, p + lane) : -1);
  __syncthreads();
  for (int e = threadIdx.x; e < width; e += blockDim.x) {
    int total = 0;
    for (int w = 0; w < waves; ++w) total += shared[w * width + e];
    a.counts[static_cast<int64_t>(blockIdx.x) * width + e] = total;
  }
}

// Stable counting sort. A wave has a range of consecutive pairs: it counts their keys in
// LDS, the counts become first rows (a scan over the keys, then over workgroups and waves),
// and a pair's row is its key's first row of the wave and its rank there, which the counting
// gave; pairs that the lanes do not hold from then are ranked again. Round trips and barriers
// bound it: 3.5 us for one token, 4.7 for 1048 pairs in one workgroup, 4.6 and 6.4 in two
// launches for 32768 in 32. (Counting by LDS atomics took 9.3 us for 4001 pairs of five
// keys, which now take 6.1.)
__global__ __launch_bounds__(64 * kSortWaves) void order_kernel(OrderArgs a) {
  extern __shared__ int shared[];
  __shared__ int wave_sums[kSortWaves];
  const int width = a.experts + 1, waves = blockDim.x >> 6;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  int *totals = shared, *before = shared + width, *counts = shared + 2 * width + wave * width;
  int low, high, held[kHeld], rank[kHeld];
  range_of(a, waves, low, high);
  hold_keys(a, low, high, held);
  for (int i = threadIdx.x; i < (waves + 2) * width; i += blockDim.x) shared[i] = 0;
  __syncthreads();
  if (a.counts) {  // (a wave some of the workgroups, all their loads on the way together)
    for (int e = lane; e < width; e += 64) {
      int total = 0, earlier = 0;
#pragma unroll 4
      for (int b = wave; b < static_cast<int>(gridDim.x); b += waves) {
        const int c = a.counts[static_cast<int64_t>(b) * width + e];
        total += c;
        earlier += b < static_cast<int>(blockIdx.x) ? c : 0;
      }
      if (total) atomicAdd(&totals[e], total);
      if (earlier) atomicAdd(&before[e], earlier);
    }
  }
#pragma unroll
  for (int j = 0; j < kHeld; ++j)
    if (low + 64 * j < high) rank[j] = take_keys(a, counts, held[j]);
  for (int p = low + 64 * kHeld; p < high; p += 64) take_keys(a, counts, p + lane < high ? key_of(a, p + lane) : -1);
  __syncthreads();

  // thread i scans `each` consecutive keys
  const int each = (width + blockDim.x - 1) / blockDim.x;
  const int first = threadIdx.x * each, last = min(first + each, width);
  int sum = 0;
  for (int e = first; e < last; ++e) {
    if (!a.counts) {
      int total = 0;
      for (int w = 0; w < waves; ++w) total += shared[(2 + w) * width + e];
      totals[e] = total;
    }
    sum += totals[e];
  }
  int scan = sum;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const int below = __shfl_up(scan, m);
    if (lane >= m) scan += below;
  }
  if (lane == 63) wave_sums[wave] = scan;
  __syncthreads();
  int row = scan - sum;
  for (int w = 0; w < wave; ++w) row += wave_sums[w];
  for (int e = first; e < last; ++e) {
    if (blockIdx.x == 0) a.offsets[e] = row;
    int next = row + before[e];
    for (int w = 0; w < waves; ++w) {
      const int c = shared[(2 + w) * width + e];
      shared[(2 + w) * width + e] = next;
      next += c;
    }
    row += totals[e];
  }
  __syncthreads();

  auto place = [&](int p, int key, int r) {
    a.places[p] = key < a.experts ? r : -1 - r;
    a.pairs[r] = p;
  };
  // (all of a wave's ranks are read before its later pairs move the rows on)
#pragma unroll
  for (int j = 0; j < kHeld; ++j)
    if (held[j] >= 0) place(low + 64 * j + lane, held[j], counts[held[j]] + rank[j]);
  if (low + 64 * kHeld >= high) return;
  // rows of the pairs not held: behind the wave's held ones
  wave_in_step();
#pragma unroll
  for (int j = 0; j < kHeld; ++j) take_keys(a, counts, held[j]);
  for (int p = low + 64 * kHeld; p < high; p += 64) {
    const int key = p + lane < high ? key_of(a, p + lane) : -1;
    const int r = take_keys(a, counts, key);
    if (key >= 0) place(p + lane, key, r);
  }
}

// Waves of a sorting workgroup at most: 16, fewer where the counts of many experts need the
// LDS. That costs much: 65536 pairs of 512 / 1024 / 2048 / 4096 experts take 15 / 26 / 70 / 391
// us in both launches, of 16 / 8 / 4 / 1 waves, each of which reads as many more of the 64
// workgroups' counts.
int most_waves(int experts) {
  int waves = kSortWaves;
  while ((waves + 2) * (experts + 1) * 4 > kCountBytes) waves /= 2;
  return waves;
}

// One workgroup while its lanes hold all keys, else up to 64 of a key a lane: 4096 pairs are
// 6.1 us in one, 32768 took 4.7 and 10.5 in eight of four keys a lane.
int sort_blocks(int64_t pairs, int experts) {
  const int64_t lanes = 64 * most_waves(experts);
  if (pairs <= lanes * kHeld) return 1;
  const int64_t blocks = (pairs + lanes - 1) / lanes;
  return static_cast<int>(blocks < kSortBlocks ? blocks : kSortBlocks);
}

// ---------------------------------------------------------------------------
// rows of the pairs, and back

struct RowsArgs {
  const void *from;     // [T, H] (gather, combine's backward) or [T K, H] (combine)
  const void *rows;     // combine's backward: [T K, H]
  const int32_t *places;
  const void *weights;  // [T, K] or NULL
  void *out;            // gather and combine's backward: [T K, H], combine: [T, H]
  void *grad_weights;   // [T, K]
  int tokens, top_k, hidden;
  bool weights16;
};

// The slots of one token: lane k of each of its waves reads slot k's place and weight, and
// hands them to all lanes, so that a token's rows are on their way after one round trip.
struct Slots {
  int place;
  float weight;

  __device__ __forceinline__ Slots(const RowsArgs &a, int t) : place(INT32_MAX), weight(1.0f) {
    const int k = threadIdx.x & 63;
    if (k >= a.top_k) return;
    const int64_t pair = static_cast<int64_t>(t) * a.top_k + k;
    place = a.places[pair];
    if (a.weights)
      weight = a.weights16 ? bf16_value(static_cast<const uint16_t *>(a.weights)[pair])
                           : static_cast<const float *>(a.weights)[pair];
    // (a place past the rows, which no order holds, is skipped)
    const int row = place >= 0 ? place : -1 - place;
    if (row >= static_cast<int64_t>(a.tokens) * a.top_k) place = INT32_MAX;
  }
  __device__ __forceinline__ int at(int k) const { return __builtin_amdgcn_readlane(place, k); }
  __device__ __forceinline__ float weight_at(int k) const {
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(weight), k));
  }
};

__device__ __forceinline__ bool kept(int place) { return place >= 0 && place != INT32_MAX; }

// A token's lanes: all of a workgroup, or one wave of it where the rows are short.
template <int kWaves, typename F>
__device__ __forceinline__ void for_tokens(const RowsArgs &a, F f) {
  constexpr int kTokens = kThreads / 64 / kWaves;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t step = static_cast<int64_t>(gridDim.x) * kTokens;
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * kTokens + wave / kWaves; t < a.tokens; t += step)
    f(static_cast<int>(t), wave % kWaves, static_cast<int>(threadIdx.x & 63));
}

// In the kernels below all lanes of a wave go through a row together, those past its end
// with the row's last values, which they neither store nor count: a slot's place is read
// from its lane by the others while that lane is at work.

// rows[place] = x[t]: a token's row is read once and written K times.
template <bool kFp32, Rows kRows, int kWaves>
__global__ __launch_bounds__(kThreads) void gather_kernel(RowsArgs a) {
  using L = Lane<kFp32, kRows>;
  for_tokens<kWaves>(a, [&](int t, int part, int lane) {
    const Slots slots(a, t);
    for (int base = 64 * part * L::kValues; base < a.hidden; base += 64 * kWaves * L::kValues) {
      const int column = base + lane * L::kValues, h = L::first(column, a.hidden);
      float v[L::kValues], zero[L::kValues] = {};
      L::values(L::load(a.from, static_cast<int64_t>(t) * a.hidden + h), v);
      for (int k = 0; k < a.top_k; ++k) {
        const int place = slots.at(k);
        if (place == INT32_MAX) continue;
        const int64_t row = place >= 0 ? place : -1 - place;
        if (column < a.hidden) L::store(a.out, row * a.hidden + h, place >= 0 ? v : zero);
      }
    }
  });
}

// out[t] = sum over kept slots of w rows[place]: kSlots rows are on their way together.
template <bool kFp32, Rows kRows, int kWaves>
__global__ __launch_bounds__(kThreads) void combine_kernel(RowsArgs a) {
  using L = Lane<kFp32, kRows>;
  for_tokens<kWaves>(a, [&](int t, int part, int lane) {
    const Slots slots(a, t);
    for (int base = 64 * part * L::kValues; base < a.hidden; base += 64 * kWaves * L::kValues) {
      const int column = base + lane * L::kValues, h = L::first(column, a.hidden);
      float sum[L::kValues] = {};
      for (int k0 = 0; k0 < a.top_k; k0 += kSlots) {
        typename L::Raw raw[kSlots] = {};
#pragma unroll
        for (int j = 0; j < kSlots; ++j) {
          const int place = k0 + j < a.top_k ? slots.at(k0 + j) : -1;
          if (kept(place)) raw[j] = L::template load<true>(a.from, static_cast<int64_t>(place) * a.hidden + h);
        }
#pragma unroll
        for (int j = 0; j < kSlots; ++j) {
          if (k0 + j >= a.top_k || !kept(slots.at(k0 + j))) continue;
          const float w = slots.weight_at(k0 + j);
          float v[L::kValues];
          L::values(raw[j], v);
#pragma unroll
          for (int i = 0; i < L::kValues; ++i) sum[i] = fmaf(w, v[i], sum[i]);
        }
      }
      if (column < a.hidden) L::store(a.out, static_cast<int64_t>(t) * a.hidden + h, sum);
    }
  });
}

// drows[place] = w dout[t] and dw = dout[t] . rows[place], kSlots slots at a time.
template <bool kFp32, Rows kRows, int kWaves>
__global__ __launch_bounds__(kThreads) void combine_backward_kernel(RowsArgs a) {
  using L = Lane<kFp32, kRows>;
  __shared__ float parts[kWaves][kSlots];
  for_tokens<kWaves>(a, [&](int t, int part, int lane) {
    const Slots slots(a, t);
    for (int k0 = 0; k0 < a.top_k; k0 += kSlots) {
      float dot[kSlots] = {};
      // (whole: no lane of the wave is past the row's end)
      auto take = [&](int column, auto whole) {
        constexpr bool kInside = decltype(whole)::value;
        const int h = kInside ? column : L::first(column, a.hidden), others = column - h;
        const bool in = kInside || column < a.hidden;
        float grad[L::kValues];
        typename L::Raw raw[kSlots] = {};
        L::values(L::load(a.from, static_cast<int64_t>(t) * a.hidden + h), grad);
        if (a.grad_weights) {
#pragma unroll
          for (int j = 0; j < kSlots; ++j) {
            const int place = k0 + j < a.top_k ? slots.at(k0 + j) : -1;
            if (kept(place)) raw[j] = L::template load<true>(a.rows, static_cast<int64_t>(place) * a.hidden + h);
          }
#pragma unroll
          for (int j = 0; j < kSlots; ++j) {
            if (k0 + j >= a.top_k || !kept(slots.at(k0 + j))) continue;
            float v[L::kValues], more = dot[j];
            L::values(raw[j], v);
#pragma unroll
            for (int i = 0; i < L::kValues; ++i) {
              const float next = fmaf(grad[i], v[i], more);
              more = !kInside && i < others ? more : next;
            }
            dot[j] = in ? more : dot[j];
          }
        }
        if (!a.out) return;
#pragma unroll
        for (int j = 0; j < kSlots; ++j) {
          const int place = k0 + j < a.top_k ? slots.at(k0 + j) : INT32_MAX;
          if (place == INT32_MAX) continue;
          const float w = slots.weight_at(k0 + j);
          float g[L::kValues];
#pragma unroll
          for (int i = 0; i < L::kValues; ++i) g[i] = place >= 0 ? w * grad[i] : 0.0f;
          const int64_t row = place >= 0 ? place : -1 - place;
          if (in) L::store(a.out, row * a.hidden + h, g);
        }
      };
      for (int base = 64 * part * L::kValues; base < a.hidden; base += 64 * kWaves * L::kValues) {
        const int column = base + lane * L::kValues;
        if (base + 64 * L::kValues <= a.hidden) take(column, std::true_type());
        else take(column, std::false_type());
      }
      if (!a.grad_weights) continue;
#pragma unroll
      for (int j = 0; j < kSlots; ++j) dot[j] = wave_total(dot[j]);
      if (kWaves > 1) {
#pragma unroll
        for (int j = 0; j < kSlots; ++j)
          if (lane == j) parts[part][j] = dot[j];
        __syncthreads();
      }
      if (part == 0 && lane < kSlots && k0 + lane < a.top_k) {
        float total = 0.0f;
        if (kWaves > 1) {
#pragma unroll
          for (int w = 0; w < kWaves; ++w) total += parts[w][lane];
        } else {
#pragma unroll
          for (int j = 0; j < kSlots; ++j) total = lane == j ? dot[j] : total;
        }
        const int64_t pair = static_cast<int64_t>(t) * a.top_k + k0 + lane;
        if (a.weights16) static_cast<uint16_t *>(a.grad_weights)[pair] = bf16_bits(total);
        else static_cast<float *>(a.grad_weights)[pair] = total;
      }
      if (kWaves > 1) __syncthreads();
    }
  });
}

int check_rows(const RowsArgs &a) {
  if (a.hidden < 1 || a.hidden > (1 << 20)) return fail(CFMOE_EINVAL, "rows need a hidden size from 1 to 2^20");
  if (a.top_k < 1 || a.top_k > kMaxTop) return fail(CFMOE_EINVAL, "rows need 1 to 64 pairs a token");
  if (a.tokens < 0 || static_cast<int64_t>(a.tokens) * a.top_k > kMaxPairs)
    return fail(CFMOE_EINVAL, "rows need 0 to 2^30 pairs");
  return 0;
}

// A wave takes a token of up to two lanes' worth, a workgroup of four a longer one. 8192
// tokens of 8 rows, BF16, the same ones again and again, one wave against four: laying out
// rows of 264 / 1024 / 2048 9.4 / 24.1 / 55.2 us and 11.4 / 24.0 / 47.1, their sum 9.8 / 23.3 /
// 57.6 and 11.5 / 23.9 / 45.9, its gradients 21.0 / 47.4 / 98.9 and 41.2 / 48.3 / 87.4.
#define CFMOE_ROWS_LAUNCH(KERNEL, fp32, a, stream)                                                          \
  do {                                                                                                      \
    const Rows rows = rows_of((a).hidden, fp32);                                                            \
    const int values = rows == kSingle ? 1 : (fp32) ? 4 : 8;                                                \
    const bool wide = (a).hidden > 128 * values;                                                            \
    const int64_t groups = wide ? (a).tokens : (static_cast<int64_t>((a).tokens) + 3) / 4;                  \
    const dim3 grid(static_cast<unsigned>(groups < (1 << 20) ? groups : (1 << 20)));                        \
    auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, stream, a); };     \
    auto typed = [&](auto narrow, auto full) { launch(wide ? full : narrow); };                             \
    if (rows == kSingle) launch((fp32) ? KERNEL<true, kSingle, 1> : KERNEL<false, kSingle, 1>);             \
    else if ((fp32) && rows == kWhole) typed(KERNEL<true, kWhole, 1>, KERNEL<true, kWhole, 4>);             \
    else if (fp32) typed(KERNEL<true, kRagged, 1>, KERNEL<true, kRagged, 4>);                               \
    else if (rows == kWhole) typed(KERNEL<false, kWhole, 1>, KERNEL<false, kWhole, 4>);                     \
    else typed(KERNEL<false, kRagged, 1>, KERNEL<false, kRagged, 4>);                                       \
  } while (0)

}  // namespace
}  // namespace cfmoe

extern "C" {

using namespace cfmoe;

CFMOE_API int64_t cfmoe_sort_by_expert_scratch_bytes(int32_t tokens, int32_t top_k, int32_t experts) {
  if (tokens < 0 || top_k < 1 || top_k > kMaxTop || static_cast<int64_t>(tokens) * top_k > kMaxPairs)
    return -fail(CFMOE_EINVAL, "sort_by_expert needs 0 to 2^30 pairs, 1 to 64 a token");
  if (experts < 1 || experts > kMaxExperts) return -fail(CFMOE_EINVAL, "sort_by_expert needs 1 to 4096 experts");
  const int blocks = sort_blocks(static_cast<int64_t>(tokens) * top_k, experts);
  return blocks <= 1 ? 0 : static_cast<int64_t>(blocks) * (experts + 1) * 4;
}

CFMOE_API int cfmoe_sort_by_expert(int32_t experts, int32_t top_k, uint32_t flags, const void *ids,
                                   const uint8_t *padding, int32_t *offsets, int32_t *places, int32_t *pairs,
                                   void *scratch, int32_t tokens, cfmoe_stream stream) {
  const int64_t bytes = cfmoe_sort_by_expert_scratch_bytes(tokens, top_k, experts);
  if (bytes < 0) return static_cast<int>(-bytes);
  if (!offsets || (tokens && (!ids || !places || !pairs)) || (bytes && !scratch)) return fail(CFMOE_EINVAL, "NULL argument");
  OrderArgs a;
  a.ids = ids;
  a.padding = padding;
  a.offsets = offsets;
  a.places = places;
  a.pairs = pairs;
  a.counts = bytes ? static_cast<int32_t *>(scratch) : nullptr;
  a.pairs_total = tokens * top_k;
  a.top_k = top_k;
  a.experts = experts;
  a.ids64 = flags & CFMOE_IDS_INT64;
  // (no pairs: one workgroup writes the offsets, all zero)
  const int blocks = sort_blocks(a.pairs_total, experts);
  int waves = most_waves(experts);
  if (blocks == 1)
    while (waves > 1 && a.pairs_total <= 32 * waves) waves /= 2;
  const int64_t share = (a.pairs_total + static_cast<int64_t>(blocks) * waves - 1) / (static_cast<int64_t>(blocks) * waves);
  a.range = static_cast<int>((share + 63) / 64 * 64);
  const unsigned lds = static_cast<unsigned>((waves + 2) * (experts + 1) * 4);
  if (a.counts) {
    hipLaunchKernelGGL(order_count_kernel, dim3(blocks), dim3(64 * waves), lds, stream, a);
    if (int rc = check_launch("order_count")) return rc;
  }
  hipLaunchKernelGGL(order_kernel, dim3(blocks), dim3(64 * waves), lds, stream, a);
  return check_launch("order");
}

CFMOE_API int cfmoe_gather_rows(int32_t hidden_size, int32_t top_k, uint32_t flags, const void *hidden,
                                const int32_t *places, void *rows, int32_t tokens, cfmoe_stream stream) {
  RowsArgs a = {};
  a.from = hidden;
  a.places = places;
  a.out = rows;
  a.tokens = tokens;
  a.top_k = top_k;
  a.hidden = hidden_size;
  if (int rc = check_rows(a)) return rc;
  if (tokens == 0) return 0;
  if (!hidden || !places || !rows) return fail(CFMOE_EINVAL, "NULL argument");
  CFMOE_ROWS_LAUNCH(gather_kernel, (flags & CFMOE_FP32) != 0, a, stream);
  return check_launch("gather_rows");
}

CFMOE_API int cfmoe_combine_rows(int32_t hidden_size, int32_t top_k, uint32_t flags, const void *rows,
                                 const int32_t *places, const void *weights, void *out, int32_t tokens,
                                 cfmoe_stream stream) {
  RowsArgs a = {};
  a.from = rows;
  a.places = places;
  a.weights = weights;
  a.out = out;
  a.tokens = tokens;
  a.top_k = top_k;
  a.hidden = hidden_size;
  a.weights16 = flags & CFMOE_WEIGHTS_BF16;
  if (int rc = check_rows(a)) return rc;
  if (tokens == 0) return 0;
  if (!rows || !places || !out) return fail(CFMOE_EINVAL, "NULL argument");
  CFMOE_ROWS_LAUNCH(combine_kernel, (flags & CFMOE_FP32) != 0, a, stream);
  return check_launch("combine_rows");
}

CFMOE_API int cfmoe_combine_rows_backward(int32_t hidden_size, int32_t top_k, uint32_t flags, const void *grad_out,
                                          const void *rows, const int32_t *places, const void *weights,
                                          void *grad_rows, void *grad_weights, int32_t tokens,
                                          cfmoe_stream stream) {
  RowsArgs a = {};
  a.from = grad_out;
  a.rows = rows;
  a.places = places;
  a.weights = weights;
  a.out = grad_rows;
  a.grad_weights = grad_weights;
  a.tokens = tokens;
  a.top_k = top_k;
  a.hidden = hidden_size;
  a.weights16 = flags & CFMOE_WEIGHTS_BF16;
  if (int rc = check_rows(a)) return rc;
  if (tokens == 0 || (!grad_rows && !grad_weights)) return 0;
  if (!grad_out || !places || (grad_weights && !rows)) return fail(CFMOE_EINVAL, "NULL argument");
  CFMOE_ROWS_LAUNCH(combine_backward_kernel, (flags & CFMOE_FP32) != 0, a, stream);
  return check_launch("combine_rows_backward");
}

}  // extern "C"
