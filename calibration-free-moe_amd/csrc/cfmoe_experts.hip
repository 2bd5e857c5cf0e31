// MI355X (gfx950) whole MoE layer for a batch of few tokens.
//
//   out[t] = sum_k w[t, k] D_e (phi(G_e x_t) * (U_e x_t)),  e = ids[t, k]
//
// A (token, slot) pair is one row of its expert's products. The layer's time is
// that of reading every touched expert's weights once, so each workgroup owns a
// piece of one expert's weights and computes it for all of that expert's pairs, 16 to
// a matrix instruction's columns. Three launches, and one ahead of them for more than
// 64 pairs:
//
//   sort  the pairs of each expert, in runs (experts_sort_kernel)
//   up    act[p, c] = w phi(g) u, g and u in FP32 (experts_rows_kernel)
//   down  partial[p, h] = FP32 sum over the channels (experts_down_kernel and
//         experts_down_many_kernel over channel-major BF16 rows, experts_rows_kernel
//         over 4-bit rows)
//   join  out[t, h] = bf16(sum over t's slots, in order) (experts_join_kernel)
//
// Few tokens over 4-bit rows have down and join in one (experts_fp4_tokens_kernel).
//
// Measured with 128 experts of 2048 x 768, top 8, in microseconds (floor = the touched
// weights at 6.0 TB/s):                sort   up   down  join  floor
//   1 token, BF16                        -    13     7     4    12.6
//   1 token, 4 bits                      -     7     7     -     3.3
//   32 tokens, BF16                      5   124    68     5   179
//   256 tokens, Zipf(1.2), BF16          5   168   110     7   197
//   128 tokens, 4 bits                   5    51    37     5    53.6
// Large BF16 calls of uniform routing read at 4.5 to 5.1 TB/s over all their launches (up
// rows at 4.7 to 5.2, down rows at 4.3 to 4.8), the skewed one, whose experts of many
// pairs take several runs, at 4.2 (4.6 and 3.7), the 4-bit one at 3.3 (4.3 and 2.7). Small
// calls are the launches and one pass of memory latency each.
//
// A pair whose id lies outside [0, E) or whose token is padded belongs to no
// expert: nothing computes it, and the join leaves it out.
//
// The second product's matrix operand is BF16, so an activation (router weight and
// all) is held as two BF16 numbers, high = v cut off and low = bf16(v - high), 2^-16 of
// it off at most, and multiplied twice: the output's error stays that of its own
// rounding (one BF16 activation made it 1.45 times that). It costs BF16 layers nothing
// to 3 us in 100 and the 4-bit down product of many tokens a third (128 tokens 31 us and
// 43, since then 37); one token has columns to spare.

#include <algorithm>
#include <type_traits>

#include "cfmoe_device.h"

namespace cfmoe {
namespace {

constexpr int kWaves = 8;
constexpr int kThreads = 64 * kWaves;
constexpr int kMaxPairs = 8192;
constexpr int kMaxLength = 4096;  // of a row: 16 operand loads of eight waves
constexpr int kColumns = 16;      // pairs of a matrix instruction
constexpr int kRows = 16;         // weight rows of one
constexpr int kDownOutputs = 64;  // outputs of a BF16 down workgroup
constexpr int kJoinThreads = 256;

struct ExpertArgs {
  const uint16_t *x;
  const void *ids, *weights;
  const uint8_t *padding;
  const uint8_t *gate_up, *gate_up_scales, *down, *down_scales;
  uint16_t *act;   // [pairs, act_row]
  float *partial;  // [pairs, hidden]
  uint16_t *out;
  int tokens, top_k, pairs, experts, hidden, width;
  int groups;   // workgroups of an item
  int tiles;    // row tiles of an item
  int share;    // row tiles of a workgroup
  int splits;   // waves that share a row's products (experts_rows_kernel)
  bool ids64, weights16, gelu, by_pair;
  const struct Run *runs;   // of the sorted pairs, or NULL
  const uint16_t *sorted;
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

// A uniform base and a lane's 32-bit offset: one register an address.
template <class T>
__device__ __forceinline__ T load_at(const void *base, uint32_t offset) {
  return *reinterpret_cast<const T *>(static_cast<const uint8_t *>(base) + offset);
}

// Some pairs of one expert: the item of a workgroup. Up to 64 pairs each wave looks at
// all of the batch's itself: an item is a pair (by_pair) or an expert, has all of the
// expert's pairs, and of the pairs' items only an expert's first has any. (A single
// token's pairs are left apart: its experts differ, or one named twice is read twice.)
// Larger batches are sorted by a launch of their own (5 us; at 64 pairs, which need none,
// 106 us are 111 with it), whose items are runs of at most kMaxRun pairs: an expert that many tokens share takes several workgroups, one behind
// the other on its rows.
constexpr int kMaxRun = 64;

struct Run {
  int32_t expert, begin, count, unused;
};

struct Pairs {
  int expert, count;
  uint64_t found;
  int listed;  // the lane's pair of a sorted run

  __device__ __forceinline__ explicit Pairs(const ExpertArgs &a, int z) {
    const int lane = threadIdx.x & 63;
    if (a.runs) {
      const Run run = a.runs[z];
      expert = __builtin_amdgcn_readfirstlane(run.expert);
      count = __builtin_amdgcn_readfirstlane(run.count);
      listed = lane < count ? a.sorted[run.begin + lane] : 0;
      return;
    }
    const int e = lane < a.pairs ? pair_expert(a, lane) : -1;
    expert = a.by_pair ? __builtin_amdgcn_readlane(e, z) : z;
    found = __ballot(e == expert);
    if (a.tokens == 1 && a.by_pair) found = 1ull << z;
    const bool first = !a.by_pair || (found & ((1ull << z) - 1)) == 0;
    count = expert >= 0 && first ? __builtin_popcountll(found) : 0;
  }

  // The list into LDS. (Every wave writes the same list, and reads what it wrote.)
  __device__ __forceinline__ void list(const ExpertArgs &a, uint16_t *out) const {
    const int lane = threadIdx.x & 63;
    if (a.runs) {
      if (lane < count) out[lane] = listed;
    } else if (found >> lane & 1) {
      out[__builtin_popcountll(found & ((1ull << lane) - 1))] = lane;
    }
  }
};

// The sort: one workgroup counts the experts' pairs in LDS, adds the counts and the
// runs up, and writes the pairs expert by expert and the runs, the rest of them empty.
// (The order of an expert's pairs is that of the atomics: a pair's results are those of
// its own column of a product, whichever it is.)
constexpr int kSortThreads = 1024;
constexpr int kMaxExperts = 4096;

__global__ __launch_bounds__(kSortThreads) void experts_sort_kernel(ExpertArgs a, Run *runs, uint16_t *sorted,
                                                                    int items, int most) {
  constexpr int kEach = kMaxExperts / kSortThreads;
  __shared__ int counts[kMaxExperts];
  __shared__ int wave_pairs[kSortThreads / 64], wave_runs[kSortThreads / 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int e = threadIdx.x; e < a.experts; e += kSortThreads) counts[e] = 0;
  __syncthreads();
  for (int p = threadIdx.x; p < a.pairs; p += kSortThreads) {
    const int e = pair_expert(a, p);
    if (e >= 0) atomicAdd(&counts[e], 1);
  }
  __syncthreads();
  // thread = kEach experts in a row
  int mine[kEach], pairs = 0, parts = 0;
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const int e = threadIdx.x * kEach + j;
    mine[j] = e < a.experts ? counts[e] : 0;
    pairs += mine[j];
    parts += (mine[j] + most - 1) / most;
  }
  int pairs_to = pairs, parts_to = parts;  // inclusive sums
  for (int m = 1; m < 64; m *= 2) {
    const int p = __shfl_up(pairs_to, m), q = __shfl_up(parts_to, m);
    pairs_to += lane >= m ? p : 0;
    parts_to += lane >= m ? q : 0;
  }
  if (lane == 63) wave_pairs[wave] = pairs_to, wave_runs[wave] = parts_to;
  __syncthreads();
  int at = pairs_to - pairs, run = parts_to - parts, total = 0;
  for (int w = 0; w < kSortThreads / 64; ++w) {
    at += w < wave ? wave_pairs[w] : 0;
    run += w < wave ? wave_runs[w] : 0;
    total += wave_runs[w];
  }
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const int e = threadIdx.x * kEach + j;
    if (e >= a.experts) break;
    counts[e] = at;  // where the expert's next pair goes
    for (int n = 0; n < mine[j]; n += most) runs[run++] = Run{e, at + n, min(most, mine[j] - n), 0};
    at += mine[j];
  }
  for (int i = total + threadIdx.x; i < items; i += kSortThreads) runs[i] = Run{0, 0, 0, 0};
  __syncthreads();
  for (int p = threadIdx.x; p < a.pairs; p += kSortThreads) {
    const int e = pair_expert(a, p);
    if (e >= 0) sorted[atomicAdd(&counts[e], 1)] = p;
  }
}

__device__ __forceinline__ float activated(float gate, float up, bool gelu) {
  const float inner = gelu ? 1.5957691216057308f * (gate + 0.044715f * gate * gate * gate) : gate;
  return gate / (1.0f + __expf(-inner)) * up;
}

// A pair's activations are pieces of eight channels, their high parts and then their low
// ones: a piece is a matrix operand's load of one lane. For 4-bit rows the pieces of each
// 128 channels stand as the four lanes of a pair read them, 32 block + 8 q at piece
// 4 q + block.
template <bool kFp4>
constexpr __host__ __device__ int act_row(int width) { return kFp4 ? (width + 127) / 128 * 256 : 2 * width; }
template <bool kFp4>
__device__ __forceinline__ uint32_t act_place(uint32_t piece) {
  return 16 * (kFp4 ? (piece & ~15u) + piece % 4 * 4 + piece / 4 % 4 : piece);
}

// A value's high part: the BF16 number next below it in size, so that the rest is never 0
// and has its sign. (Against an infinite weight a rest of 0 or of the other sign makes a
// NaN of what is infinite. To nearest, the high part of a value above 3.39e38 would be
// infinite; the rest off by 2^-17 of the value where it is 2^-16 now.) An infinity's is
// the largest number. Below 2^-132 both parts are 2^-133, the least BF16 number.
__device__ __forceinline__ void split(float v, uint32_t &high, float &low) {
  const uint32_t sign = __float_as_uint(v) & 0x80000000u, size = __float_as_uint(v) & 0x7fffffffu;
  const uint32_t least = min(size, 1u) << 16;
  const uint32_t part = max(__builtin_elementwise_sub_sat(size, 1u) & 0xffff0000u, least);
  // (a NaN stays in the high part: it is quiet, its bits well above infinity's)
  const float rest = fmaxf(__uint_as_float(size) - __uint_as_float(part), __uint_as_float(least));
  high = part | sign;
  low = __uint_as_float(__float_as_uint(rest) | sign);
}

// Both parts of a piece at element `to`, of which lane l, l + 16, l + 32 and l + 48 have
// two channels each: after two swaps, of half waves and of odd with even quarters, two
// words that stand side by side. (A store for each part took a sixth of the up product's
// time.)
__device__ __forceinline__ void store_activations(const ExpertArgs &a, uint32_t to, float first, float second) {
  uint32_t high0, high1;
  float low0, low1;
  split(first, high0, low0);
  split(second, high1, low1);
  const auto halves = __builtin_amdgcn_permlane32_swap(high0 >> 16 | high1, bf16_pair(low0, low1), false, false);
  const auto words = __builtin_amdgcn_permlane16_swap(halves[0], halves[1], false, false);
  *reinterpret_cast<u32x2 *>(a.act + (to + (threadIdx.x & 63) / 16 * 4)) = u32x2{words[0], words[1]};
}

// v + the v of the lane eight columns on or back: a pair's high and low parts.
__device__ __forceinline__ float parts_sum(float v) {
  constexpr int kRotate8 = 0x128;  // of 16 lanes
  return v + __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), kRotate8, 0xf, 0xf, true));
}

// What a row product is of.
enum Product { kUpBf16, kUpFp4, kDownFp4 };

// Weight rows times the pairs' vectors. `splits` waves share a row's products, the
// others take further row tiles, and the sums of a round, kBatch tiles of each wave, meet
// in LDS. A wave keeps its piece of the pairs' vectors in registers as matrix operands,
// kSteps products of 32 for kCols x kPairs pairs, and multiplies its rows by them (a
// column past the last pair repeats it; nothing of it is stored).
//
// BF16: a lane's 16 bytes are eight values, step j the wave's j-th 32. FP4: they
// are a whole block of 32, lane group g taking block g of 128 values, so that
// steps 4 i .. 4 i + 3 are the four words of the wave's i-th block. The scales of
// all the workgroup's rows go to LDS first: they are rows of length / 32 bytes, of
// which a wave wants a few bytes each (byte loads from memory took a third of the
// up product's time, 87 us of it 27 at 1024 pairs, 128 experts of 2048 x 768).
//
// Unless kFull a wave may hold fewer loads than the kernel has: it repeats its last
// one with every bit cleared, weights and vectors both, so that what a row holds
// cannot reach the sum a second time.
template <Product kProduct, int kSteps, bool kFull, int kCols, int kBatch>
struct RowPass {
  static constexpr bool kFp4 = kProduct != kUpBf16, kDown = kProduct == kDownFp4;
  static constexpr int kLoads = kFp4 ? kSteps / 4 : kSteps;
  // pairs of a column tile: the down product's high parts are columns 0-7, their low parts 8-15
  static constexpr int kPairs = kDown ? kColumns / 2 : kColumns;

  template <class Ready>
  static __device__ __forceinline__ void run(const ExpertArgs &a, int expert, int first, int last,
                                             const uint16_t *list, int count, int base, f32x4 *sums,
                                             const uint8_t *scales, Ready ready) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int split = wave % a.splits, sub = wave / a.splits, subs = kWaves / a.splits;
    const int length = kDown ? a.width : a.hidden;
    const int units = kFp4 ? (length + 127) / 128 : length / 32;
    const int begin = units * split / a.splits, steps = units * (split + 1) / a.splits - begin;
    const int rounds = (last - first + subs * kBatch - 1) / (subs * kBatch);
    const uint32_t row_bytes = kFp4 ? length / 2 : length * 2, scale_bytes = length / 32;
    // the lane's row of a tile: in the up product gate and up row of a channel in turn
    const uint32_t row = kDown ? lane % 16 : (lane & 1) * a.width + lane % 16 / 2;
    const uint32_t lane_row = row * row_bytes + lane / 16 * 16;
    const uint32_t kept_row = kDown ? lane % 16 : (lane & 1) * (a.share * (kRows / 2)) + lane % 16 / 2;
    const uint8_t *lane_scales = scales + kept_row * scale_bytes + 4 * begin;

    // load i is one of the wave's own (in 4 bits a row's last 128 values may end at a
    // block), and where it starts, in units of 64 bytes from the wave's first
    auto own = [&](int i) {
      const bool inside = i < steps && (!kFp4 || 4 * (begin + i) + lane / 16 < length / 32);
      return kFull || inside ? ~0u : 0u;
    };
    // (steps >= 1: cut_of takes no more waves than there are units)
    auto unit = [&](int i) { return kFull ? i : min(i, steps - 1); };

    u32x4 words[kBatch][kLoads];
    auto load = [&](int r, int of) {
      const int tile = min(first + (r * kBatch + of) * subs + sub, last - 1);
      const int64_t row0 = kDown ? static_cast<int64_t>(expert) * a.hidden + tile * kRows
                                 : static_cast<int64_t>(expert) * 2 * a.width + tile * (kRows / 2);
      const uint8_t *w = (kDown ? a.down : a.gate_up) + row0 * row_bytes + begin * 64;
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const bool whole = kFull || !kFp4 || own(unit(i));
        words[of][i] = load_at<u32x4>(w + unit(i) * 64, whole ? lane_row : lane_row - lane / 16 * 16);
      }
    };
#pragma unroll
    for (int of = 0; of < kBatch; ++of) load(0, of);
    ready();
    u32x4 b[kCols][kSteps];
#pragma unroll
    for (int n = 0; n < kCols; ++n) {
      const uint32_t pair = list[min(base + n * kPairs + lane % kPairs, count - 1)];
      const uint32_t vector = kDown ? pair * (2 * act_row<kFp4>(a.width)) + lane % 16 / kPairs * 16 : pair / a.top_k * a.hidden * 2;
#pragma unroll
      for (int j = 0; j < kSteps; ++j) {
        // (element 32 block + 8 (j % 4) in 4 bits, block 4 i + lane / 16)
        const int i = unit(kFp4 ? j / 4 : j);
        const uint32_t place = kDown   ? (begin + i) * 512 + j % 4 * 128 + lane / 16 * 32
                               : kFp4 ? (4 * (begin + i) + (own(i) ? lane / 16 : 0)) * 64 + j % 4 * 16
                                      : (begin + i) * 64 + lane / 16 * 16;
        b[n][j] = load_at<u32x4>(kDown ? a.act : a.x, vector + place) & own(kFp4 ? j / 4 : j);
      }
    }
    // What a wave adds up and stores: of a round's subs x kSums sums every eighth; its
    // column tile is the same in each. Two column tiles of the down product make one sum,
    // high and low parts' columns added first.
    constexpr int kSums = kDown ? 1 : kCols, kStored = kDown ? kCols * kPairs : kColumns;
    const int column = base + wave % kSums * kColumns + lane % kStored;
    const bool stores = column < count && lane % 16 < kStored;
    const uint32_t pair = list[min(column, count - 1)];
    const uint32_t to = kDown ? pair * a.hidden + lane / 16 * 4 : pair * act_row<kFp4>(a.width);
    const float weight = kDown ? 0.0f : pair_weight(a, pair);

    auto product = [&](int r, int of) {
      f32x4 d[kCols];
#pragma unroll
      for (int n = 0; n < kCols; ++n) d[n] = f32x4{0, 0, 0, 0};
      const int kept = min((r * kBatch + of) * subs + sub, last - 1 - first) * (kDown ? kRows : kRows / 2) * scale_bytes;
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const u32x4 w = words[of][i] & own(i);
        if constexpr (kFp4) {
          const uint32_t byte = lane_scales[kept + 4 * unit(i) + (own(unit(i)) ? lane / 16 : 0)];
          const float by = __uint_as_float((byte & own(i)) << 23);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const u32x4 values = fp4_values(w[q], by);
#pragma unroll
            for (int n = 0; n < kCols; ++n) d[n] = mma(values, b[n][4 * i + q], d[n]);
          }
        } else {
#pragma unroll
          for (int n = 0; n < kCols; ++n) d[n] = mma(w, b[n][i], d[n]);
        }
      }
      // (the sums alternate between two buffers: what a round overwrites was read
      // before the last barrier)
      f32x4 *in = sums + ((r & 1) * kBatch + of) * (kWaves * kSums * 64) + lane;
      if constexpr (kDown) {
        f32x4 both;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          // (both sums by all lanes: one reads a lane of the other half)
          const float first = parts_sum(d[0][e]), second = parts_sum(d[kCols - 1][e]);
          both[e] = kCols == 2 && (lane & 8) ? second : first;
        }
        in[wave * 64] = both;
      } else {
#pragma unroll
        for (int n = 0; n < kCols; ++n) in[(wave * kCols + n) * 64] = d[n];
      }
    };
    auto add = [&](int r) {
      __syncthreads();
      for (int i = wave; i < kBatch * subs * kSums; i += kWaves) {
        const int tile = first + r * kBatch * subs + i / kSums;
        if (!stores || tile >= last) break;
        const f32x4 *in = sums + ((r & 1) * kBatch + i / (subs * kSums)) * (kWaves * kSums * 64) + lane;
        f32x4 v = in[(i / kSums % subs * a.splits * kSums + i % kSums) * 64];
        for (int w = 1; w < a.splits; ++w) v += in[((i / kSums % subs * a.splits + w) * kSums + i % kSums) * 64];
        if (kDown)
          *reinterpret_cast<f32x4 *>(a.partial + (to + tile * kRows)) = v;
        else
          store_activations(a, to + act_place<kFp4>(tile), weight * activated(v[0], v[1], a.gelu),
                            weight * activated(v[2], v[3], a.gelu));
      }
    };
    // The rows' registers are free once multiplied: the next round's loads leave before
    // this one's sums are added up. (Rounds on their way ahead of that, with a barrier
    // for each, measured the same or worse: two to eight of one load a wave made the
    // 4-bit down product 41 to 59 us, 1024 pairs, where kBatch 1 made it 43.)
    for (int r = 0; r + 1 < rounds; ++r) {
#pragma unroll
      for (int of = 0; of < kBatch; ++of) {
        product(r, of);
        load(r + 1, of);
      }
      add(r);
    }
#pragma unroll
    for (int of = 0; of < kBatch; ++of) product(rounds - 1, of);
    add(rounds - 1);
    __syncthreads();
  }
};

// Waves of a SIMD that the registers have to leave room for: two a workgroup. Three
// workgroups for the 4-bit up product of few pairs, which holds little (one token of
// 2048 x 768, three workgroups to a compute unit in all: 14.1 us the call, 15.2 with two).
constexpr int least_waves(Product product, int steps, bool full, int columns, int batch) {
  if (product == kUpFp4 && steps <= 8 && full && columns == 1 && batch == 1) return 6;
  return columns <= 2 && steps <= 8 ? 4 : 2;
}

// Workgroup = `share` row tiles of one item, for all of its pairs, up to kMaxCols x 16
// at a time. Dynamic LDS: the scales of its rows.
template <Product kProduct, int kSteps, bool kFull, int kMaxCols, int kBatch>
__global__ __launch_bounds__(kThreads, least_waves(kProduct, kSteps, kFull, kMaxCols, kBatch)) void experts_rows_kernel(ExpertArgs a) {
  constexpr bool kFp4 = kProduct != kUpBf16, kDown = kProduct == kDownFp4;
  __shared__ f32x4 sums[2 * kBatch * kWaves * (kDown ? 1 : kMaxCols) * 64];
  __shared__ uint16_t list[kMaxRun];
  extern __shared__ __align__(16) uint8_t lds[];
  const Pairs pairs(a, blockIdx.x / a.groups);
  const int count = pairs.count, expert = pairs.expert;
  if (count == 0) return;
  const int first = blockIdx.x % a.groups * a.share, last = min(first + a.share, a.tiles);
  const uint32_t scale_bytes = kFp4 ? (kDown ? a.width : a.hidden) / 32 : 0;

  // 16 bytes a thread of the scales of rows first .. last - 1 (gate rows, then up)
  const int tile_rows = kDown ? kRows : kRows / 2, parts = kDown ? 1 : 2;
  const int chunks = (last - first) * tile_rows * scale_bytes / 16, kept = a.share * tile_rows * scale_bytes / 16;
  const uint8_t *scales = (kDown ? a.down_scales + static_cast<int64_t>(expert) * a.hidden * scale_bytes
                                 : a.gate_up_scales + static_cast<int64_t>(expert) * 2 * a.width * scale_bytes) +
                          first * tile_rows * scale_bytes;
  for (int i = threadIdx.x; kFp4 && i < parts * kept; i += kThreads) {
    const int part = i / kept, chunk = i - part * kept;
    if (chunk < chunks)
      reinterpret_cast<u32x4 *>(lds)[i] = load_at<u32x4>(scales, part * a.width * scale_bytes + chunk * 16);
  }

  constexpr int kPairs = RowPass<kProduct, kSteps, kFull, 1, kBatch>::kPairs;
  for (int base = 0; base < count;) {
    const int left = count - base;
    auto ready = [&] {
      if (base == 0) pairs.list(a, list);
      if (kFp4 && base == 0) __syncthreads();  // the scales
    };
    if (kMaxCols >= 4 && left > 2 * kPairs) {
      if constexpr (kMaxCols >= 4)
        RowPass<kProduct, kSteps, kFull, 4, kBatch>::run(a, expert, first, last, list, count, base, sums, lds, ready);
      base += 4 * kPairs;
    } else if (kMaxCols >= 2 && left > kPairs) {
      if constexpr (kMaxCols >= 2)
        RowPass<kProduct, kSteps, kFull, 2, kBatch>::run(a, expert, first, last, list, count, base, sums, lds, ready);
      base += 2 * kPairs;
    } else {
      RowPass<kProduct, kSteps, kFull, 1, kBatch>::run(a, expert, first, last, list, count, base, sums, lds, ready);
      base += kPairs;
    }
  }
}

// Channel-major down rows hold an output per element, where the matrix operand
// wants eight channels of one output: a lane loads eight channels' rows at its
// four outputs and turns the 8 x 4 piece in registers. Output 4 (l % 16) + j of
// the tile is row l % 16 of product j.
__device__ __forceinline__ void turn(const u32x2 (&rows)[8], u32x4 (&turned)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t select = j & 1 ? 0x07060302u : 0x05040100u;
#pragma unroll
    for (int c = 0; c < 4; ++c)
      turned[j][c] = __builtin_amdgcn_perm(rows[2 * c + 1][j / 2], rows[2 * c][j / 2], select);
  }
}

// How the layer's 32-channel steps, every eighth to a wave, meet kSteps of them.
enum Steps {
  kExact,    // kSteps for each wave
  kRagged,   // some waves one fewer: a step past the last repeats it, every bit cleared
  kHalfStep  // and the last step is 16 channels: its second half repeats the first, cleared
};

template <Steps kMode>
struct DownLane {
  uint32_t row_bytes, channel, row;  // the lane's channel and row from a step's start on
  int steps;
  bool half;

  __device__ __forceinline__ explicit DownLane(const ExpertArgs &a)
      : row_bytes(2 * a.hidden), steps((a.width + 31) / 32) {
    const int lane = threadIdx.x & 63;
    half = lane >= 32;
    channel = lane / 16 * 8;
    row = channel * row_bytes + lane % 16 * 8;
  }
  __device__ __forceinline__ int at(int step) const { return kMode == kExact ? step : min(step, steps - 1); }
  __device__ __forceinline__ bool short_of(int step) const { return kMode == kHalfStep && at(step) == steps - 1 && half; }
  template <class T>
  __device__ __forceinline__ T own(T v, int step) const {
    if (kMode == kExact) return v;
    return v & (step < steps && !short_of(step) ? ~0u : 0u);
  }
  // a part of a pair's activations, high (0) or low (1)
  __device__ __forceinline__ u32x4 vector(const ExpertArgs &a, uint32_t pair, int part, int step) const {
    const uint32_t offset = (pair * a.width + channel) * 4 + part * 16;
    return own(load_at<u32x4>(reinterpret_cast<const uint8_t *>(a.act) + 128 * at(step),
                              short_of(step) ? offset - 64 : offset), step);
  }
  __device__ __forceinline__ void rows(u32x2 (&to)[8], const uint8_t *down, int step) const {
    const uint8_t *from = down + static_cast<int64_t>(32 * at(step)) * row_bytes;
    const uint32_t offset = short_of(step) ? row - 16 * row_bytes : row;
#pragma unroll
    for (int i = 0; i < 8; ++i) to[i] = load_at<u32x2>(from + i * row_bytes, offset);
  }
};

// Workgroup = `share` x 64 outputs of one expert, the waves an eighth of its channels
// each (kSteps products of 32 at most; wider layers take several chunks), 16 pairs at
// a time. The pairs' vectors stay in registers; a step's rows are loaded for the next
// 64 outputs as soon as they are turned. Reading the rows bounds it, a channel's piece
// 128 bytes: 13 rows over 128 experts of 2816 x 704 (72 of them touched) 58 us; one token
// over eight of 2048 x 768 7 us for 25 MB, most of it the first loads' latency.
template <int kSteps, Steps kMode>
__global__ __launch_bounds__(kThreads, kSteps <= 3 ? 4 : 2) void experts_down_kernel(ExpertArgs a) {
  __shared__ f32x4 sums[2 * kWaves * 4 * 64];
  __shared__ uint16_t list[kMaxRun];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Pairs pairs(a, blockIdx.x / a.groups);
  const int count = pairs.count;
  if (count == 0) return;
  const int first = blockIdx.x % a.groups * a.share, rounds = min(a.share, a.tiles - first);
  const DownLane<kMode> place(a);
  const uint8_t *down =
      a.down + (static_cast<int64_t>(pairs.expert) * a.width * a.hidden + first * kDownOutputs) * 2;
  for (int base = 0; base < count; base += kColumns) {
    for (int chunk = 0; chunk < place.steps; chunk += kWaves * kSteps) {
      auto step = [&](int s) { return chunk + s * kWaves + wave; };
      u32x2 rows[kSteps][8];
#pragma unroll
      for (int s = 0; s < kSteps; ++s) place.rows(rows[s], down, step(s));
      if (base == 0 && chunk == 0) pairs.list(a, list);
      const int column = base + lane % 16;
      const uint32_t pair = list[min(column, count - 1)];
      u32x4 b[kSteps][2];
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
        for (int part = 0; part < 2; ++part) b[s][part] = place.vector(a, pair, part, step(s));
      auto round = [&](int r, auto more) {
        f32x4 d[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) d[j] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
          u32x4 w[4];
          // (cleared rows: what they hold must not meet a cleared vector as 0 x infinity)
#pragma unroll
          for (int i = 0; i < 8; ++i) rows[s][i] = place.own(rows[s][i], step(s));
          turn(rows[s], w);
          if (decltype(more)::value) place.rows(rows[s], down + (r + 1) * (2 * kDownOutputs), step(s));
#pragma unroll
          for (int j = 0; j < 4; ++j) d[j] = mma(w[j], b[s][0], d[j]);
#pragma unroll
          for (int j = 0; j < 4; ++j) d[j] = mma(w[j], b[s][1], d[j]);
        }
        // a lane holds outputs 16 g + 4 i + j of its pair, g = l / 16; the sums alternate
        // between two buffers, and the waves' two halves in adding them up
        f32x4 *in = sums + (r & 1) * (kWaves * 4 * 64);
#pragma unroll
        for (int i = 0; i < 4; ++i) in[(wave * 4 + i) * 64 + lane] = f32x4{d[0][i], d[1][i], d[2][i], d[3][i]};
        __syncthreads();
        if ((wave ^ (r & 1) * 4) < 4) {
          const int i = wave % 4;
          f32x4 v = in[i * 64 + lane];
#pragma unroll
          for (int k = 1; k < kWaves; ++k) v += in[(k * 4 + i) * 64 + lane];
          if (column < count) {
            f32x4 *out = reinterpret_cast<f32x4 *>(
                a.partial + (pair * a.hidden + (first + r) * kDownOutputs + lane / 16 * 16 + i * 4));
            *out = chunk ? *out + v : v;
          }
        }
      };
      for (int r = 0; r + 1 < rounds; ++r) round(r, std::true_type{});
      round(rounds - 1, std::false_type{});
      __syncthreads();
    }
  }
}

// Many pairs an expert: workgroup = 64 outputs of one expert, whose weights stay in
// registers for all of its pairs, 16 at a time. 64 tokens over 64 experts of 2048 x 1024
// 62 us for 268 MB (4.4 TB/s); every further 16 pairs cost their vectors' loads and two
// barriers, nothing of memory but their partials (256 Zipf tokens over 128 experts of
// 2048 x 768 108 us).
template <int kSteps, Steps kMode>
__global__ __launch_bounds__(kThreads, kSteps <= 3 ? 4 : 2) void experts_down_many_kernel(ExpertArgs a) {
  __shared__ f32x4 sums[kWaves * 4 * 64];
  __shared__ uint16_t list[kMaxRun];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Pairs pairs(a, blockIdx.x / a.groups);
  const int count = pairs.count, expert = pairs.expert;
  if (count == 0) return;
  const int row0 = blockIdx.x % a.groups * kDownOutputs;
  const DownLane<kMode> place(a);
  const uint8_t *down = a.down + (static_cast<int64_t>(expert) * a.width * a.hidden + row0) * 2;
  for (int chunk = 0; chunk < place.steps; chunk += kWaves * kSteps) {
    u32x4 w[kSteps][4];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int step = chunk + s * kWaves + wave;
      u32x2 rows[8];
      place.rows(rows, down, step);
#pragma unroll
      for (int i = 0; i < 8; ++i) rows[i] = place.own(rows[i], step);
      turn(rows, w[s]);
    }
    if (chunk == 0) pairs.list(a, list);
    for (int base = 0; base < count; base += kColumns) {
      const uint32_t pair = list[min(base + lane % 16, count - 1)];
      u32x4 b[kSteps][2];
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
        for (int part = 0; part < 2; ++part) b[s][part] = place.vector(a, pair, part, chunk + s * kWaves + wave);
      f32x4 d[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) d[j] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
#pragma unroll
        for (int j = 0; j < 4; ++j) d[j] = mma(w[s][j], b[s][0], d[j]);
#pragma unroll
        for (int j = 0; j < 4; ++j) d[j] = mma(w[s][j], b[s][1], d[j]);
      }
      // a lane holds outputs 16 g + 4 r + j of its pair, g = l / 16
#pragma unroll
      for (int r = 0; r < 4; ++r)
        sums[(wave * 4 + r) * 64 + lane] = f32x4{d[0][r], d[1][r], d[2][r], d[3][r]};
      __syncthreads();
      if (threadIdx.x < 256) {
        f32x4 v = sums[threadIdx.x];
#pragma unroll
        for (int k = 1; k < kWaves; ++k) v += sums[k * 256 + threadIdx.x];
        const int column = base + lane % 16;
        if (column < count) {
          f32x4 *out = reinterpret_cast<f32x4 *>(a.partial + (static_cast<uint32_t>(list[column]) * a.hidden + row0 +
                                                 lane / 16 * 16 + wave * 4));
          *out = chunk ? *out + v : v;
        }
      }
      __syncthreads();
    }
  }
}

// Few tokens over 4-bit rows: workgroup = 16 outputs of one token, its waves the
// token's slots (every eighth), so that the slots' sum needs no launch of its own. An
// expert that several tokens name is read for each of them, and fewer slots than waves
// leave some idle. A pair's high and low parts are columns in turn.
//
// Whole calls in a graph, in us, this kernel against the down and join kernels:
//                          top 1         top 2         top 4         top 8
//   128 of 2048 x 768    8:  13, 15   10:  27, 30   12:  40, 43    6:  38, 43
//                       16:  24, 25   16:  34, 33   16:  49, 48   10:  58, 55
//   64 of 2048 x 1024    8:  15, 18    8:  22, 24    8:  33, 34    4:  33, 35
//                       12:  21, 23   10:  29, 28   10:  39, 39    5:  41, 40
//   64 of 4096 x 2048    3:  21, 21    2:  25, 26    2:  36, 36    1:  37, 39
//    (top 1 to 4 of 16)  5:  33, 30    4:  34, 33    4:  53, 47    2:  61, 58
//   1024 of 1024 x 128  16:   8, 10   16:  10, 12   16:  12, 14   16:  22, 24
//                       32:  12, 11   32:  15, 14   32:  23, 22   32:  33, 29
// (tokens: us). So it is taken up to 10 MB of rows for each slot a token has, four at the
// most, and up to 1280 workgroups, what the chip holds at a time.
constexpr int kFewGroups = 1280;
constexpr int64_t kFewBytes = 10000000;
__global__ __launch_bounds__(kThreads) void experts_fp4_tokens_kernel(ExpertArgs a) {
  constexpr int kAhead = 4;
  __shared__ f32x4 sums[kWaves][2][4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int t = blockIdx.x / a.tiles, row = blockIdx.x % a.tiles * kRows;
  const int blocks = a.width / 32, steps = (blocks + 3) / 4;
  f32x4 d = {0, 0, 0, 0};
  for (int k = wave; k < a.top_k; k += kWaves) {
    const int pair = t * a.top_k + k;
    const int expert = __builtin_amdgcn_readfirstlane(pair_expert(a, pair));
    if (expert < 0) continue;
    const int64_t row0 = static_cast<int64_t>(expert) * a.hidden + row;
    const uint8_t *words = a.down + row0 * (a.width / 2), *scales = a.down_scales + row0 * blocks;
    const uint8_t *act = reinterpret_cast<const uint8_t *>(a.act + static_cast<uint32_t>(pair) * act_row<true>(a.width));
    for (int s = 0; s < steps; s += kAhead) {
      u32x4 word[kAhead];
      u32x4 b[kAhead][4];
      uint32_t scale[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        // (past the last block it comes again, cleared)
        const uint32_t block = min(4 * (s + i) + lane / 16, blocks - 1);
        const uint32_t own = 4 * (s + i) + lane / 16 < blocks ? ~0u : 0u;
        word[i] = load_at<u32x4>(words, lane % 16 * (a.width / 2) + block * 16) & own;
        scale[i] = load_at<uint8_t>(scales, lane % 16 * blocks + block) & own;
#pragma unroll
        for (int q = 0; q < 4; ++q) b[i][q] = load_at<u32x4>(act, min(s + i, steps - 1) * 512 + q * 128 + lane / 16 * 32 + lane % 2 * 16) & own;
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) d = mma(fp4_values(word[i][q], __uint_as_float(scale[i] << 23)), b[i][q], d);
    }
  }
  // (all 16 columns are the one token's, high and low parts in turn)
  if (lane % 16 < 2) sums[wave][lane % 2][lane / 16] = d;
  __syncthreads();
  if (threadIdx.x < 4) {
    f32x4 v = {0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) v += sums[w][0][threadIdx.x] + sums[w][1][threadIdx.x];
    *reinterpret_cast<u32x2 *>(a.out + (static_cast<uint32_t>(t) * a.hidden + row + threadIdx.x * 4)) =
        u32x2{bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3])};
  }
}

// Thread = four outputs of one token: its slots' partials in order. Latency, 4 to 7 us:
// 256 tokens of top 8 and 2048 outputs are 16 MB, from the caches that the down product
// wrote.
__global__ __launch_bounds__(kJoinThreads) void experts_join_kernel(ExpertArgs a) {
  constexpr int kAhead = 8;
  const int groups = a.hidden / 4;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kJoinThreads + threadIdx.x;
  const int t = static_cast<int>(i / groups), h = static_cast<int>(i % groups) * 4;
  if (t >= a.tokens) return;
  f32x4 sum = {0, 0, 0, 0};
  const float *row = a.partial + static_cast<int64_t>(t) * a.top_k * a.hidden + h;
  for (int k = 0; k < a.top_k; k += kAhead) {
    f32x4 v[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      // (a slot that no expert computed holds whatever the scratch held)
      const int slot = min(k + j, a.top_k - 1);
      v[j] = *reinterpret_cast<const f32x4 *>(row + static_cast<int64_t>(slot) * a.hidden);
      const bool routed = k + j < a.top_k && pair_expert(a, t * a.top_k + slot) >= 0;
#pragma unroll
      for (int r = 0; r < 4; ++r) v[j][r] = routed ? v[j][r] : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) sum += v[j];
  }
  const u32x2 out = {bf16_pair(sum[0], sum[1]), bf16_pair(sum[2], sum[3])};
  *reinterpret_cast<u32x2 *>(a.out + static_cast<int64_t>(t) * a.hidden + h) = out;
}

int validate(int hidden, int width, int experts, int top_k, uint32_t flags, int tokens) {
  if (hidden <= 0 || hidden % 128 || hidden > kMaxLength)
    return fail(CFMOE_EINVAL, "routed_experts needs a hidden size that is a multiple of 128, at most 4096");
  const int grain = flags & CFMOE_FP4 ? 32 : 16;
  if (width <= 0 || width % grain || width > kMaxLength)
    return fail(CFMOE_EINVAL, "routed_experts needs a width that is a multiple of 16 (of 32 with 4-bit weights), at most 4096");
  if (experts < 1 || experts > kMaxExperts) return fail(CFMOE_EINVAL, "routed_experts needs 1 to 4096 experts");
  if (top_k < 1 || top_k > 64) return fail(CFMOE_EINVAL, "routed_experts needs 1 to 64 experts per token");
  if (tokens < 0 || static_cast<int64_t>(tokens) * top_k > kMaxPairs)
    return fail(CFMOE_EINVAL, "routed_experts takes at most 8192 routed pairs per call");
  return 0;
}

// How a row of `units` operand loads (32 BF16 values, or 128 in 4 bits) is cut: the
// waves that share it, and each one's loads, one of the counts that kernels exist
// for. Fewest idle loads first, then the most waves. The 4-bit down product takes one
// load a wave where that leaves none idle (width 1024, 512 pairs of 64 experts, 23 us
// against 27 of two; width 768 40 against 38), and two where eight waves can: three want
// more registers than two workgroups have (46 against 43).
struct Cut {
  int splits, loads;
};

Cut cut_of(int units, bool fp4, bool down) {
  Cut best = {0, 0};
  for (int splits = kWaves; splits >= 1; splits /= 2)
    for (int loads : {down && splits == units ? 1 : fp4 ? 2 : 8, fp4 ? 2 : 8, fp4 ? 3 : 12, fp4 ? 4 : 16})
      if (loads * splits >= units && !(down && loads > 2 && units <= 2 * kWaves) &&
          (!best.splits || loads * splits < best.loads * best.splits))
        best = {splits, loads};
  return best;
}

// The most runs of at most `most` pairs that `pairs` pairs of `experts` can make.
int run_items(int experts, int pairs, int most) { return std::min(experts, pairs) + pairs / most; }

int64_t act_bytes(int width, int pairs, bool fp4) {  // (a row is a multiple of 64 bytes)
  return static_cast<int64_t>(pairs) * (fp4 ? act_row<true>(width) : act_row<false>(width)) * 2;
}

template <int kSteps>
auto down_kernel(bool many, Steps mode) {
  if (many)
    return mode == kExact    ? experts_down_many_kernel<kSteps, kExact>
           : mode == kRagged ? experts_down_many_kernel<kSteps, kRagged>
                             : experts_down_many_kernel<kSteps, kHalfStep>;
  return mode == kExact    ? experts_down_kernel<kSteps, kExact>
         : mode == kRagged ? experts_down_kernel<kSteps, kRagged>
                           : experts_down_kernel<kSteps, kHalfStep>;
}

// Tiles of a wave between two barriers, where its workgroup has as many: what the
// registers hold with two workgroups to a compute unit, of 4-bit rows only. (128 tokens
// over 128 experts of 2048 x 768: up product 52 us against 55, down 38 against 43; 64
// tokens over 64 of 2048 x 1024: 34 against 40, 23 against 28.)
template <Product kProduct, int kSteps>
constexpr int batch_tiles(bool wide) {
  if (kProduct == kUpBf16 || kSteps > 8) return 1;
  return kProduct == kDownFp4 ? (kSteps == 8 ? 2 : 4) : wide ? 2 : 4;
}

template <Product kProduct, int kSteps>
auto rows_kernel(bool full, bool wide, int tiles) {
  // Column tiles of a wide call's. BF16: as many as the registers hold with one
  // workgroup to a compute unit. 4 bits: two, with which there are still two workgroups
  // (four leave room for one: 256 Zipf tokens 103 us against 80).
  constexpr int kWide = kProduct == kUpBf16 ? (kSteps == 8 ? 4 : kSteps == 12 ? 2 : 1)
                                            : (kProduct == kDownFp4 || kSteps <= 8 ? 2 : 1);
  constexpr int kNarrow = kProduct == kDownFp4 ? 2 : 1;
  constexpr int kBatch = batch_tiles<kProduct, kSteps>(false), kWideBatch = batch_tiles<kProduct, kSteps>(true);
  // (one width alone fills three loads of eight waves in the 4-bit down product: it takes
  // the general kernel)
  constexpr bool kFull = kProduct != kDownFp4 || kSteps != 12;
  if (wide)
    return tiles >= kWideBatch ? full ? experts_rows_kernel<kProduct, kSteps, kFull, kWide, kWideBatch>
                                      : experts_rows_kernel<kProduct, kSteps, false, kWide, kWideBatch>
                               : full ? experts_rows_kernel<kProduct, kSteps, kFull, kWide, 1>
                                      : experts_rows_kernel<kProduct, kSteps, false, kWide, 1>;
  return tiles >= kBatch ? full ? experts_rows_kernel<kProduct, kSteps, kFull, kNarrow, kBatch>
                                : experts_rows_kernel<kProduct, kSteps, false, kNarrow, kBatch>
                         : full ? experts_rows_kernel<kProduct, kSteps, kFull, kNarrow, 1>
                                : experts_rows_kernel<kProduct, kSteps, false, kNarrow, 1>;
}

template <Product kProduct>
int launch_rows(ExpertArgs a, int items, bool wide, cfmoe_stream stream) {
  constexpr bool kFp4 = kProduct != kUpBf16, kDown = kProduct == kDownFp4;
  const int length = kDown ? a.width : a.hidden;
  const int units = kFp4 ? (length + 127) / 128 : length / 32;
  const Cut cut = cut_of(units, kFp4, kDown);
  const int steps = cut.loads * (kFp4 ? 4 : 1);
  const bool full = units == cut.splits * cut.loads && length % 128 == 0;
  a.splits = cut.splits;
  a.tiles = kDown ? a.hidden / kRows : a.width / (kRows / 2);
  // Enough workgroups to fill the chip, then fewer loads of the pairs' vectors. Items are
  // counted as the most runs there can be, all that the host knows of a sorted call: up to
  // a third of the workgroups find theirs empty and end. (Narrow
  // BF16 kernels, three workgroups to a compute unit: 2048 for 1024 make 16 tokens over
  // 128 experts 94 us of 96, 32 over 64 97 of 99, those of 2816 x 704 135 of 129.)
  const int subs = kWaves / cut.splits;
  a.share = subs;
  while (static_cast<int64_t>(items) * a.tiles / (2 * a.share) >= (kFp4 || wide ? 1024 : 2048) && a.share < 8 * subs) a.share *= 2;
  a.groups = (a.tiles + a.share - 1) / a.share;
  const int tiles = a.share / subs;  // of a wave
  auto kernel = steps <= 8    ? rows_kernel<kProduct, 8>(full, wide, tiles)
                : steps <= 12 ? rows_kernel<kProduct, 12>(full, wide, tiles)
                              : rows_kernel<kProduct, 16>(full, wide, tiles);
  if constexpr (kDown)
    if (steps <= 4) kernel = rows_kernel<kProduct, 4>(full, wide, tiles);
  const unsigned scales = kFp4 ? a.share * kRows * (length / 32) : 0;
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(a.groups) * items), dim3(kThreads), scales, stream, a);
  return check_launch(kDown ? "experts_down" : "experts_up");
}

}  // namespace
}  // namespace cfmoe

extern "C" {

using namespace cfmoe;

CFMOE_API int64_t cfmoe_routed_experts_scratch_bytes(int32_t hidden_size, int32_t width, int32_t experts,
                                                     int32_t top_k, uint32_t flags, int32_t tokens) {
  if (int rc = validate(hidden_size, width, experts, top_k, flags, tokens)) return -rc;
  const int pairs = tokens * top_k;
  // activations, partials, and for more than 64 pairs the runs and the sorted pairs
  const int64_t sorted = pairs > 64 ? run_items(experts, pairs, 16) * sizeof(Run) + pairs * 2 : 0;
  return act_bytes(width, pairs, flags & CFMOE_FP4) + static_cast<int64_t>(pairs) * hidden_size * 4 + sorted;
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
  for (const void *p : {gate_up, down, hidden, static_cast<const void *>(out), static_cast<const void *>(scratch),
                        static_cast<const void *>(gate_up_scales), static_cast<const void *>(down_scales)})
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
  a.act = static_cast<uint16_t *>(scratch);
  a.partial = reinterpret_cast<float *>(static_cast<uint8_t *>(scratch) + act_bytes(width, a.pairs, fp4));
  a.ids64 = flags & CFMOE_IDS_INT64;
  a.weights16 = flags & CFMOE_WEIGHTS_BF16;
  a.gelu = flags & CFMOE_GELU;
  a.by_pair = a.pairs <= experts;
  // A wide call's sorted runs are of 64 pairs over BF16 rows and 32 over 4-bit rows, the
  // others' of 16, and its up product takes several column tiles at a time: only where
  // its registers hold them (rows_kernel). It pays where experts have more than 16 pairs,
  // and costs where most have few. Whole calls in a graph, wide against narrow, in us, by
  // pairs an expert on average (uniform routing, and Zipf(1.2)):
  //   BF16, 64 experts of 2048 x 1024   6: 170, 168 (164, 162)    8: 175, 183 (171, 174)
  //                                    16: 189, 195 (199, 214)   32: 218, 265 (230, 272)
  //         128 of 2048 x 768           6: 249, 235 (229, 224)    8: 257, 251 (240, 237)
  //                                    12: 270, 268 (264, 272)   16: 283, 291 (284, 298)
  //         64 of 1536 x 768            6: 109, 112 (111, 108)    8: 113, 114 (119, 116)
  //         32 of 4096 x 1024 (one column tile)                  16: 222, 200 (239, 222)
  // 4-bit rows' down product has no wide form, so that their calls gain later, and only
  // where eight waves share an up row:
  //         128 of 2048 x 768          16: 131, 127 (139, 133)   28: 178, 181 (183, 182)
  //                                    48: 258, 268 (255, 268)   64: 319, 340 (316, 339)
  //         64 of 2048 x 1024          24: 104, 103 (106, 102)   64: 191, 206 (190, 206)
  //         64 of 1024 x 512 (four)    16:  49,  40  (53,  42)   48:  69,  61  (69,  62)
  const Cut up = cut_of(fp4 ? hidden_size / 128 : hidden_size / 32, fp4, false);
  const bool wide = fp4 ? up.splits == kWaves && up.loads <= 2 && a.pairs >= 28 * experts
                        : up.loads <= 12 && a.pairs >= 8 * experts;
  int items = a.by_pair ? a.pairs : experts;
  a.runs = nullptr;
  a.sorted = nullptr;
  if (a.pairs > 64) {
    const int most = !wide ? 16 : fp4 ? 32 : kMaxRun;
    items = run_items(experts, a.pairs, most);
    Run *runs = reinterpret_cast<Run *>(static_cast<uint8_t *>(scratch) + act_bytes(width, a.pairs, fp4) +
                                        static_cast<int64_t>(a.pairs) * hidden_size * 4);
    uint16_t *sorted = reinterpret_cast<uint16_t *>(runs + run_items(experts, a.pairs, 16));
    hipLaunchKernelGGL(experts_sort_kernel, dim3(1), dim3(kSortThreads), 0, stream, a, runs, sorted, items, most);
    if (int rc = check_launch("experts_sort")) return rc;
    a.runs = runs;
    a.sorted = sorted;
  }

  if (int rc = fp4 ? launch_rows<kUpFp4>(a, items, wide, stream) : launch_rows<kUpBf16>(a, items, wide, stream)) return rc;
  const int64_t read = static_cast<int64_t>(a.pairs) * hidden_size * (width / 2);
  if (fp4 && a.by_pair && tokens * (hidden_size / kRows) <= kFewGroups && read <= kFewBytes * std::min(top_k, 4)) {
    a.tiles = hidden_size / kRows;  // (experts_fp4_tokens_kernel: both sides)
    hipLaunchKernelGGL(experts_fp4_tokens_kernel, dim3(static_cast<unsigned>(a.tiles) * tokens), dim3(kThreads), 0,
                       stream, a);
    return check_launch("experts_down");
  }
  if (fp4) {
    if (int rc = launch_rows<kDownFp4>(a, items, false, stream)) return rc;
  } else {
    a.tiles = hidden_size / kDownOutputs;
    a.share = 1;
    const bool many = wide;
    while (!many && static_cast<int64_t>(items) * a.tiles / (2 * a.share) >= 256 && a.share < 4) a.share *= 2;
    a.groups = (a.tiles + a.share - 1) / a.share;
    const int steps = (width + 31) / 32, each = (steps + kWaves - 1) / kWaves;
    const int held = each <= 2 ? 2 : each <= 4 ? each : 8;
    const Steps mode = width % 32 ? kHalfStep : steps % (kWaves * held) ? kRagged : kExact;
    const auto kernel = held == 2   ? down_kernel<2>(many, mode)
                        : held == 3 ? down_kernel<3>(many, mode)
                        : held == 4 ? down_kernel<4>(many, mode)
                                    : down_kernel<8>(many, mode);
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(a.groups) * items), dim3(kThreads), 0, stream, a);
    if (int rc = check_launch("experts_down")) return rc;
  }

  const int64_t threads = static_cast<int64_t>(tokens) * (hidden_size / 4);
  hipLaunchKernelGGL(experts_join_kernel, dim3(static_cast<unsigned>((threads + kJoinThreads - 1) / kJoinThreads)),
                     dim3(kJoinThreads), 0, stream, a);
  return check_launch("experts_join");
}

}  // extern "C"
