// MI355X (gfx950): the norms before and after a block, its gate and the residual's scale.
//
// Of rows x (the residual stream) and b (a block's output), with i(v) = 1 / sqrt(mean(v^2) + eps):
//
//   n = b i(b) p        behind the block, p its weights; n = b without them
//   j = s x + g n       s a number, g nothing, [H], [T, 1] or [T, H]
//   y = j i(j) w        before the next block, w its weights
//
// and backward, with G = dL/dj of both outputs, b^ = b i(b), j^ = j i(j), means over a row:
//
//   G  = dj + i(j) (dy w - j^ mean(dy w j^))      dw = sum_t dy j^
//   dx = s G      dg = G n, summed where g was spread
//   dn = G g      dp = sum_t dn b^
//   db = i(b) (dn p - b^ mean(dn p b^))           db = dn without p
//
// A norm alone is the case without b: j = x, and only y is written. A row is read once and
// stays in registers between the sums; y is of j before it is rounded, and the backward
// pass forms j again from what forward read, so that no rounding but the outputs' own is in
// them. Squares are summed in FP32; a row whose sum passes FP32 is summed again 2^-80 times
// as large, which leaves no number to overflow, beside 2^-160 epsilon: of 1e30 still 2e-5 of
// the mean where a row of 8192 begins to pass, of 1e27 and less nothing that FP32 holds.

#include "cfmoe_rows.h"

namespace cfmoe {
namespace {

constexpr int kMaxHidden = 8192;
constexpr int kEach = 8;  // values of a row that a thread holds
// Waves of a launch at most: 24 to a compute unit (16 / 24 / 32: 27.5 / 26.5 / 27.7 us), and 12
// in at most 1024 workgroups.
constexpr int kForwardWaves = 24 * 256;
constexpr int kBackwardWaves = 12 * 256;
constexpr float kSmall = 0x1p-80f;

enum Gate { kNone, kChannel, kRow, kFull };

struct JoinArgs {
  const void *hidden, *block, *post, *gate, *next;
  void *joined, *out;
  float *statistics;  // [T, 2]: i(b) and i(j); -v stands for 2^-80 v
  const void *grad_joined, *grad_out;
  void *grad_hidden, *grad_block, *grad_gate;
  float *partial;  // [workgroups, sums, H]: dw, dp and the channel gate's dg, those there are
  int tokens, size, sums;
  float scale, epsilon;
  Gate form;
  bool post32, gate32, next32, grad_post, grad_next;
};

template <bool kFp32, Rows kRows, int kWaves>
struct Row {
  using L = Lane<kFp32, kRows>;
  static constexpr int kValues = L::kValues;
  static constexpr int kParts = kEach / kValues;
  static constexpr int kThreads = 64 * kWaves;

  // Eight values of a row on their way.
  struct Raw {
    typename L::Raw part[kParts];
  };

  // Column from which a thread's part p counts its values, and the one its values begin at.
  __device__ static int column(int p) { return (p * kThreads + static_cast<int>(threadIdx.x)) * kValues; }
  __device__ static int first(int p, int size) { return L::first(column(p), size); }

  // Whether the thread counts its value i in a sum.
  __device__ static bool counts(int i, int size) {
    return kRows != kRagged || i % kValues >= L::others(column(i / kValues), size);
  }

  __device__ static void load(const void *rows, int64_t row, int size, Raw &raw) {
#pragma unroll
    for (int p = 0; p < kParts; ++p)
      if (column(p) < size) raw.part[p] = L::load(rows, row * size + first(p, size));
  }

  // Zero past the end.
  __device__ static void values(const Raw &raw, int size, float *v) {
#pragma unroll
    for (int p = 0; p < kParts; ++p) {
      L::values(raw.part[p], v + p * kValues);
#pragma unroll
      for (int i = 0; i < kValues; ++i) v[p * kValues + i] = column(p) < size ? v[p * kValues + i] : 0.0f;
    }
  }

  __device__ static void store(void *rows, int64_t row, int size, const float *v) {
#pragma unroll
    for (int p = 0; p < kParts; ++p)
      if (column(p) < size) L::store(rows, row * size + first(p, size), v + p * kValues);
  }

  // Weights [H] of the rows' type or FP32; zero past the end.
  __device__ static void weights(const void *w, bool fp32, int size, float *v) {
#pragma unroll
    for (int p = 0; p < kParts; ++p) {
      float *part = v + p * kValues;
      if (column(p) >= size) {
#pragma unroll
        for (int i = 0; i < kValues; ++i) part[i] = 0.0f;
      } else if (!kFp32 && fp32) {
        using F = Lane<true, kRows>;
#pragma unroll
        for (int i = 0; i < kValues; i += F::kValues) F::values(F::load(w, first(p, size) + i), part + i);
      } else {
        L::values(L::load(w, first(p, size)), part);
      }
    }
  }
};

// A row's gate, [T, 1].
template <bool kFp32>
__device__ __forceinline__ float row_gate(const JoinArgs &a, int64_t row) {
  return kFp32 || a.gate32 ? static_cast<const float *>(a.gate)[row]
                           : bf16_value(static_cast<const uint16_t *>(a.gate)[row]);
}

// Sums over the workgroup, in every thread, always in the same order. `turn` changes with
// each call, so that one barrier is enough: who writes a half again has passed the barrier
// of the call between, which all reach after they read it.
template <int kWaves, int kSums>
__device__ __forceinline__ void group_totals(float (&v)[kSums], float (*shared)[2][kWaves], int &turn) {
#pragma unroll
  for (int s = 0; s < kSums; ++s) v[s] = wave_total(v[s]);
  if constexpr (kWaves > 1) {
    turn ^= 1;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int s = 0; s < kSums; ++s) shared[turn][s][threadIdx.x >> 6] = v[s];
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < kSums; ++s) {
      v[s] = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) v[s] += shared[turn][s][w];
    }
  }
}

// 1 / sqrt(mean(v^2) + eps); negative, it is that of 2^-80 v.
template <typename R, int kWaves>
__device__ __forceinline__ float inverse_root(const float *values, const JoinArgs &a, float (*shared)[2][kWaves], int &turn) {
  float sum[1] = {0.0f}, v[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) v[i] = R::counts(i, a.size) ? values[i] : 0.0f;
#pragma unroll
  for (int i = 0; i < kEach; ++i) sum[0] = fmaf(v[i], v[i], sum[0]);
  group_totals<kWaves, 1>(sum, shared, turn);
  const float size = static_cast<float>(a.size);
  if (sum[0] <= 3.4e38f) return 1.0f / sqrtf(sum[0] / size + a.epsilon);
  sum[0] = 0.0f;
#pragma unroll
  for (int i = 0; i < kEach; ++i) sum[0] = fmaf(v[i] * kSmall, v[i] * kSmall, sum[0]);
  group_totals<kWaves, 1>(sum, shared, turn);
  return -1.0f / sqrtf(sum[0] / size + a.epsilon * kSmall * kSmall);
}

__device__ __forceinline__ float unit(float v, float inverse) {
  return inverse < 0.0f ? v * kSmall * -inverse : v * inverse;
}

// times 1 / sqrt(...) itself
__device__ __forceinline__ float times_inverse(float v, float inverse) {
  return inverse < 0.0f ? v * -inverse * kSmall : v * inverse;
}

// Workgroup = rows in steps of the grid, a thread eight values of each. The weights are
// read once, and the next row is on its way while this one's sums are formed: 8192 rows of
// 2048 BF16 values with both norms 35 us without either, 26.5 to 29 with (134 MB, 4.6 to 5.1
// TB/s; a copy of that size reaches 5.5). A row alone is 2.9 us, a launch and two round trips.
template <bool kFp32, Rows kRows, int kWaves>
__global__ __launch_bounds__(64 * kWaves) void join_kernel(JoinArgs a) {
  using R = Row<kFp32, kRows, kWaves>;
  __shared__ float shared[2][2][kWaves];
  int turn = 0;
  typename R::Raw x = {}, b = {}, g = {};
  float spread = 0.0f;
  auto fetch = [&](int64_t t) {
    R::load(a.hidden, t, a.size, x);
    if (a.block) R::load(a.block, t, a.size, b);
    if (a.form == kFull) R::load(a.gate, t, a.size, g);
    if (a.form == kRow) spread = row_gate<kFp32>(a, t);
  };
  fetch(blockIdx.x);
  float post[kEach], next[kEach], gate[kEach];
  if (a.post) R::weights(a.post, a.post32, a.size, post);
  if (a.next) R::weights(a.next, a.next32, a.size, next);
  if (a.form == kChannel) R::weights(a.gate, a.gate32, a.size, gate);
  for (int64_t t = blockIdx.x; t < a.tokens; t += gridDim.x) {
    float j[kEach], n[kEach], first = 0.0f, second = 0.0f;
    R::values(x, a.size, j);
    if (a.block) R::values(b, a.size, n);
    if (a.form == kFull) R::values(g, a.size, gate);
    if (a.form == kRow) {
#pragma unroll
      for (int i = 0; i < kEach; ++i) gate[i] = spread;
    }
    if (t + gridDim.x < a.tokens) fetch(t + gridDim.x);
    if (a.block) {
      if (a.post) {
        first = inverse_root<R, kWaves>(n, a, shared, turn);
#pragma unroll
        for (int i = 0; i < kEach; ++i) n[i] = unit(n[i], first) * post[i];
      }
      if (a.form != kNone) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) n[i] *= gate[i];
      }
#pragma unroll
      for (int i = 0; i < kEach; ++i) j[i] = fmaf(a.scale, j[i], n[i]);
      R::store(a.joined, t, a.size, j);
    }
    if (a.next) {
      second = inverse_root<R, kWaves>(j, a, shared, turn);
#pragma unroll
      for (int i = 0; i < kEach; ++i) n[i] = next[i] * unit(j[i], second);
      R::store(a.out, t, a.size, n);
    }
    if (a.statistics && threadIdx.x == 0) {
      a.statistics[2 * t] = first;
      a.statistics[2 * t + 1] = second;
    }
  }
}

// Workgroup = rows in steps of the grid; the sums over rows stay in registers and leave as
// one partial row each, which join_sums_kernel adds up: no atomics, so that a call gives
// the same bits every time. 8192 rows of 2048 BF16 values with both norms and a gate per
// channel: 41 us (201 MB, 4.9 TB/s) and 4.8 for the three sums. Rows of hidden and block are
// read whatever is asked for: the gradient of a plain sum, which needs neither, takes 21 us.
template <bool kFp32, Rows kRows, int kWaves>
__global__ __launch_bounds__(64 * kWaves) void join_backward_kernel(JoinArgs a) {
  using R = Row<kFp32, kRows, kWaves>;
  __shared__ float shared[2][2][kWaves];
  int turn = 0;
  const float part = 1.0f / static_cast<float>(a.size);
  typename R::Raw x = {}, b = {}, g = {}, dj = {}, dy = {};
  float spread = 0.0f, first = 0.0f, second = 0.0f;
  auto fetch = [&](int64_t t) {
    R::load(a.hidden, t, a.size, x);
    if (a.block) R::load(a.block, t, a.size, b);
    if (a.grad_joined) R::load(a.grad_joined, t, a.size, dj);
    if (a.grad_out) R::load(a.grad_out, t, a.size, dy);
    if (a.form == kFull) R::load(a.gate, t, a.size, g);
    if (a.form == kRow) spread = row_gate<kFp32>(a, t);
    if (a.post) first = a.statistics[2 * t];
    if (a.grad_out) second = a.statistics[2 * t + 1];
  };
  fetch(blockIdx.x);
  float post[kEach], next[kEach], gate[kEach];
  if (a.post) R::weights(a.post, a.post32, a.size, post);
  if (a.grad_out) R::weights(a.next, a.next32, a.size, next);
  if (a.form == kChannel) R::weights(a.gate, a.gate32, a.size, gate);
  float sum_next[kEach] = {}, sum_post[kEach] = {}, sum_gate[kEach] = {};
  for (int64_t t = blockIdx.x; t < a.tokens; t += gridDim.x) {
    // (unit: the block's rows over their root, or as they are)
    float j[kEach], unit_block[kEach], grad[kEach], y[kEach];
    const float inverse_block = first, inverse = second;
    R::values(x, a.size, j);
    if (a.block) R::values(b, a.size, unit_block);
    if (a.form == kFull) R::values(g, a.size, gate);
    if (a.form == kRow) {
#pragma unroll
      for (int i = 0; i < kEach; ++i) gate[i] = spread;
    }
    if (a.grad_out) R::values(dy, a.size, y);
    if (a.grad_joined) {
      R::values(dj, a.size, grad);
    } else {
#pragma unroll
      for (int i = 0; i < kEach; ++i) grad[i] = 0.0f;
    }
    if (t + gridDim.x < a.tokens) fetch(t + gridDim.x);
    if (a.block) {
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        if (a.post) unit_block[i] = unit(unit_block[i], inverse_block);
        float n = a.post ? unit_block[i] * post[i] : unit_block[i];
        if (a.form != kNone) n *= gate[i];
        j[i] = fmaf(a.scale, j[i], n);
      }
    }
    if (a.grad_out) {
      float mean[1] = {0.0f};
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        j[i] = unit(j[i], inverse);
        sum_next[i] = fmaf(y[i], j[i], sum_next[i]);
        y[i] *= next[i];
        if (R::counts(i, a.size)) mean[0] = fmaf(y[i], j[i], mean[0]);
      }
      group_totals<kWaves, 1>(mean, shared, turn);
      mean[0] *= part;
#pragma unroll
      for (int i = 0; i < kEach; ++i) grad[i] += times_inverse(fmaf(-j[i], mean[0], y[i]), inverse);
    }
    if (a.grad_hidden) {
#pragma unroll
      for (int i = 0; i < kEach; ++i) y[i] = a.scale * grad[i];
      R::store(a.grad_hidden, t, a.size, y);
    }
    if (!a.block) continue;
    float totals[2] = {0.0f, 0.0f};
    if (a.grad_gate) {
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        y[i] = grad[i] * (a.post ? unit_block[i] * post[i] : unit_block[i]);
        if (R::counts(i, a.size)) totals[0] += y[i];
        sum_gate[i] += y[i];
      }
      if (a.form == kFull) R::store(a.grad_gate, t, a.size, y);
    }
    if (a.form != kNone) {
#pragma unroll
      for (int i = 0; i < kEach; ++i) grad[i] *= gate[i];
    }
    if (a.post) {
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        sum_post[i] = fmaf(grad[i], unit_block[i], sum_post[i]);
        grad[i] *= post[i];
        if (R::counts(i, a.size)) totals[1] = fmaf(grad[i], unit_block[i], totals[1]);
      }
    }
    const bool row_sum = a.grad_gate && a.form == kRow;
    if (a.post || row_sum) group_totals<kWaves, 2>(totals, shared, turn);
    if (row_sum && threadIdx.x == 0) {
      if (kFp32 || a.gate32) static_cast<float *>(a.grad_gate)[t] = totals[0];
      else static_cast<uint16_t *>(a.grad_gate)[t] = bf16_bits(totals[0]);
    }
    if (!a.grad_block) continue;
    if (a.post) {
#pragma unroll
      for (int i = 0; i < kEach; ++i)
        grad[i] = times_inverse(fmaf(-unit_block[i], totals[1] * part, grad[i]), inverse_block);
    }
    R::store(a.grad_block, t, a.size, grad);
  }
  if (!a.partial) return;
  float *rows = a.partial + static_cast<int64_t>(blockIdx.x) * a.sums * a.size;
  auto leave = [&](const float *v) {
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int p = i / R::kValues;
      if (R::column(p) < a.size && R::counts(i, a.size)) rows[R::first(p, a.size) + i % R::kValues] = v[i];
    }
    rows += a.size;
  };
  if (a.grad_next) leave(sum_next);
  if (a.grad_post) leave(sum_post);
  if (a.grad_gate && a.form == kChannel) leave(sum_gate);
}

struct SumsArgs {
  const float *partial;
  void *to[3];
  bool fp32[3];
  int groups, sums, size;
};

constexpr int kSumWaves = 16;
constexpr int kSumChains = 8;

// Sums in pairs of neighbours.
template <int kCount>
__device__ __forceinline__ float paired(const float *v) {
  if constexpr (kCount == 1) return v[0];
  else return paired<kCount / 2>(v) + paired<kCount / 2>(v + kCount / 2);
}

// Wave = every 16th of the partial rows of 64 columns, in eight sums that are added in pairs, as
// the waves' are: of 1024 partial rows a value passes 8 + 3 + 4 roundings and not the 64 + 16
// of sums in order (515 FP32 rows and both norms: gradients 1.2e-7 off, in order 1.5e-7).
__global__ __launch_bounds__(64 * kSumWaves) void join_sums_kernel(SumsArgs a) {
  __shared__ float sums[kSumWaves][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = blockIdx.x * 64 + lane, which = blockIdx.y;
  float chains[kSumChains] = {};
  if (c < a.size) {
    const float *from = a.partial + static_cast<int64_t>(which) * a.size + c;
    const int64_t step = static_cast<int64_t>(a.sums) * a.size;
    int g = wave;
    for (; g + kSumWaves * (kSumChains - 1) < a.groups; g += kSumWaves * kSumChains) {
      float v[kSumChains];  // (all on the way together)
#pragma unroll
      for (int i = 0; i < kSumChains; ++i) v[i] = from[(g + kSumWaves * i) * step];
#pragma unroll
      for (int i = 0; i < kSumChains; ++i) chains[i] += v[i];
    }
#pragma unroll
    for (int i = 0; i < kSumChains - 1; ++i, g += kSumWaves)
      if (g < a.groups) chains[i] += from[g * step];
  }
  sums[wave][lane] = paired<kSumChains>(chains);
  __syncthreads();
  if (wave || c >= a.size) return;
  float waves[kSumWaves];
#pragma unroll
  for (int w = 0; w < kSumWaves; ++w) waves[w] = sums[w][lane];
  const float sum = paired<kSumWaves>(waves);
  if (a.fp32[which]) static_cast<float *>(a.to[which])[c] = sum;
  else static_cast<uint16_t *>(a.to[which])[c] = bf16_bits(sum);
}

int check_join(int hidden_size, int tokens, float epsilon) {
  if (hidden_size < 1 || hidden_size > kMaxHidden) return fail(CFMOE_EINVAL, "join_block needs a hidden size from 1 to 8192");
  if (tokens < 0) return fail(CFMOE_EINVAL, "join_block needs a token count of zero or more");
  if (!(epsilon >= 1e-30f && epsilon <= 1e30f)) return fail(CFMOE_EINVAL, "join_block needs an epsilon from 1e-30 to 1e30");
  return 0;
}

// Waves of a row: the fewest of these whose threads hold it.
int row_waves(int size) {
  for (int waves : {1, 2, 4, 8})
    if (size <= 64 * kEach * waves) return waves;
  return 16;
}

// Workgroups of a backward call. Each leaves a partial row of every sum: 512 / 768 / 1024 /
// 2048 of them take 8192 rows of 2048 in 50.2 / 49.6 / 51.3 / 59.8 us, 512 / 1024 take 2000
// rows of 4096 in 30.8 / 41.4 (384: 29.8), 8000 of 512 in 31.3 / 23.1.
int backward_groups(int size, int tokens) {
  const int waves = row_waves(size);
  const int groups = waves < 3 ? 1024 : kBackwardWaves / waves;
  return tokens < groups ? tokens : groups;
}

template <typename F>
int dispatch_row(int size, bool fp32, F f) {
  const Rows rows = rows_of(size, fp32);
  if (rows == kSingle) return fp32 ? f(Row<true, kSingle, 1>()) : f(Row<false, kSingle, 1>());
  auto typed = [&](auto waves) {
    constexpr int kWaves = decltype(waves)::value;
    if (fp32) return rows == kWhole ? f(Row<true, kWhole, kWaves>()) : f(Row<true, kRagged, kWaves>());
    return rows == kWhole ? f(Row<false, kWhole, kWaves>()) : f(Row<false, kRagged, kWaves>());
  };
  switch (row_waves(size)) {
    case 1: return typed(std::integral_constant<int, 1>());
    case 2: return typed(std::integral_constant<int, 2>());
    case 4: return typed(std::integral_constant<int, 4>());
    case 8: return typed(std::integral_constant<int, 8>());
    default: return typed(std::integral_constant<int, 16>());
  }
}

template <bool kFp32, Rows kRows, int kWaves>
int launch_join(Row<kFp32, kRows, kWaves>, const JoinArgs &a, hipStream_t stream) {
  constexpr int kGroups = kForwardWaves / kWaves;
  const int groups = a.tokens < kGroups ? a.tokens : kGroups;
  hipLaunchKernelGGL((join_kernel<kFp32, kRows, kWaves>), dim3(groups), dim3(64 * kWaves), 0, stream, a);
  return check_launch("join_block");
}

template <bool kFp32, Rows kRows, int kWaves>
int launch_backward(Row<kFp32, kRows, kWaves>, const JoinArgs &a, hipStream_t stream) {
  hipLaunchKernelGGL((join_backward_kernel<kFp32, kRows, kWaves>), dim3(backward_groups(a.size, a.tokens)), dim3(64 * kWaves), 0,
                     stream, a);
  return check_launch("join_block_backward");
}

Gate gate_of(uint32_t flags) {
  return flags & CFMOE_GATE_CHANNEL ? kChannel : flags & CFMOE_GATE_ROW ? kRow : flags & CFMOE_GATE_FULL ? kFull : kNone;
}

}  // namespace
}  // namespace cfmoe

extern "C" {

using namespace cfmoe;

CFMOE_API int cfmoe_join_block(int32_t hidden_size, uint32_t flags, const void *hidden, const void *block,
                               const void *post_weight, const void *gate, float residual_scale,
                               const void *next_weight, float epsilon, void *joined, void *next, float *statistics,
                               int32_t tokens, cfmoe_stream stream) {
  if (int rc = check_join(hidden_size, tokens, epsilon)) return rc;
  if (tokens == 0) return 0;
  JoinArgs a = {};
  a.form = gate_of(flags);
  if (!hidden || (block ? !joined : !next_weight) || (next_weight && !next) || (a.form != kNone && !gate))
    return fail(CFMOE_EINVAL, "NULL argument");
  if (!block && (post_weight || a.form != kNone)) return fail(CFMOE_EINVAL, "join_block takes a post weight or a gate with a block only");
  a.hidden = hidden;
  a.block = block;
  a.post = post_weight;
  a.gate = a.form != kNone ? gate : nullptr;
  a.next = next_weight;
  a.joined = joined;
  a.out = next;
  a.statistics = statistics;
  a.tokens = tokens;
  a.size = hidden_size;
  a.scale = residual_scale;
  a.epsilon = epsilon;
  const bool fp32 = flags & CFMOE_FP32;
  a.post32 = fp32 || flags & CFMOE_POST_FP32;
  a.gate32 = fp32 || flags & CFMOE_GATE_FP32;
  a.next32 = fp32 || flags & CFMOE_NEXT_FP32;
  if (a.form == kFull && !fp32 && flags & CFMOE_GATE_FP32)
    return fail(CFMOE_EINVAL, "join_block needs a gate per value in the rows' type");
  return dispatch_row(hidden_size, fp32, [&](auto row) { return launch_join(row, a, stream); });
}

CFMOE_API int64_t cfmoe_join_block_backward_scratch_bytes(int32_t hidden_size, int32_t sums, int32_t tokens) {
  if (hidden_size < 1 || hidden_size > kMaxHidden || sums < 0 || sums > 3 || tokens < 0)
    return -fail(CFMOE_EINVAL, "join_block needs a hidden size from 1 to 8192, up to 3 sums and 0 or more tokens");
  return static_cast<int64_t>(backward_groups(hidden_size, tokens)) * sums * hidden_size * 4;
}

CFMOE_API int cfmoe_join_block_backward(int32_t hidden_size, uint32_t flags, const void *hidden, const void *block,
                                        const void *post_weight, const void *gate, float residual_scale,
                                        const void *next_weight, const float *statistics, const void *grad_joined,
                                        const void *grad_next, void *grad_hidden, void *grad_block,
                                        void *grad_post_weight, void *grad_gate, void *grad_next_weight, void *scratch,
                                        int32_t tokens, cfmoe_stream stream) {
  if (int rc = check_join(hidden_size, tokens, 1.0f)) return rc;
  JoinArgs a = {};
  a.form = gate_of(flags);
  const bool fp32 = flags & CFMOE_FP32;
  SumsArgs s = {};
  if (grad_next_weight) s.fp32[s.sums] = fp32 || flags & CFMOE_NEXT_FP32, s.to[s.sums++] = grad_next_weight;
  if (grad_post_weight) s.fp32[s.sums] = fp32 || flags & CFMOE_POST_FP32, s.to[s.sums++] = grad_post_weight;
  if (grad_gate && a.form == kChannel) s.fp32[s.sums] = fp32 || flags & CFMOE_GATE_FP32, s.to[s.sums++] = grad_gate;
  if ((tokens && (!hidden || (a.form != kNone && !gate) || (grad_next && !next_weight) ||
                  ((post_weight || grad_next) && !statistics) || (s.sums && !scratch))) ||
      (grad_next_weight && tokens && !grad_next) || (grad_post_weight && !post_weight) || (grad_gate && a.form == kNone))
    return fail(CFMOE_EINVAL, "NULL argument");
  if (tokens && !block && (post_weight || a.form != kNone || grad_block || grad_joined))
    return fail(CFMOE_EINVAL, "join_block takes a post weight or a gate with a block only");
  if (a.form == kFull && !fp32 && flags & CFMOE_GATE_FP32)
    return fail(CFMOE_EINVAL, "join_block needs a gate per value in the rows' type");
  a.hidden = hidden;
  a.block = block;
  a.post = post_weight;
  a.gate = a.form != kNone ? gate : nullptr;
  a.next = next_weight;
  a.statistics = const_cast<float *>(statistics);
  a.grad_joined = grad_joined;
  a.grad_out = grad_next;
  a.grad_hidden = grad_hidden;
  a.grad_block = grad_block;
  a.grad_gate = grad_gate;
  a.partial = s.sums ? static_cast<float *>(scratch) : nullptr;
  a.tokens = tokens;
  a.size = hidden_size;
  a.sums = s.sums;
  a.scale = residual_scale;
  a.post32 = fp32 || flags & CFMOE_POST_FP32;
  a.gate32 = fp32 || flags & CFMOE_GATE_FP32;
  a.next32 = fp32 || flags & CFMOE_NEXT_FP32;
  a.grad_post = grad_post_weight;
  a.grad_next = grad_next_weight;
  if (tokens) {
    if (int rc = dispatch_row(hidden_size, fp32, [&](auto row) { return launch_backward(row, a, stream); })) return rc;
  }
  if (!s.sums) return 0;
  s.partial = a.partial;
  s.groups = backward_groups(hidden_size, tokens);
  s.size = hidden_size;
  hipLaunchKernelGGL(join_sums_kernel, dim3((hidden_size + 63) / 64, s.sums), dim3(64 * kSumWaves), 0, stream, s);
  return check_launch("join_block_sums");
}

}  // extern "C"
