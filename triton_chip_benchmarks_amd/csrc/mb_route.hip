// Routing of tokens to experts: choice and weights with their gradient, the
// sort of the choices by expert, and the weighted sum of the experts' outputs
// with its gradients.
#include <type_traits>

#include "mb_elem.h"

namespace mb {
namespace {

constexpr uint32_t kMostExperts = 1024, kMostTop = 64;
constexpr float kNegInf = -__builtin_inff();


// Orders a wave's LDS writes before its later LDS reads.
__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
}

// Scores s of a token's logits, lane l of its team holding experts l * V ..
// l * V + V - 1; logits past the last expert and masked ones (-inf) are -inf and
// score 0. So does a sigmoid's logit below -88.7, whose e^-l is infinite; `far`
// takes e^l there, which fp32 still holds.
template <int V, int TEAM>
__device__ __forceinline__ void scores_of(const float (&logit)[V], bool softmax, bool far, float (&score)[V]) {
  if (!softmax) {
#pragma unroll
    for (int i = 0; i < V; ++i) score[i] = 1.0f / (1.0f + expf(-logit[i]));
    if (far) {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (score[i] == 0.0f) score[i] = expf(logit[i]);
    }
    return;
  }
  float top = kNegInf;
#pragma unroll
  for (int i = 0; i < V; ++i) top = fmaxf(top, logit[i]);
  top = team_max<TEAM>(top);
  if (top == kNegInf) top = 0.0f;  // nothing but masked experts
  float total = 0.0f;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    score[i] = expf(logit[i] - top);
    total += score[i];
  }
  total = team_add<TEAM>(total);
#pragma unroll
  for (int i = 0; i < V; ++i) score[i] = total == 0.0f ? 0.0f : score[i] / total;
}

// A lane's V consecutive elements of a row, at any element's address.
template <class T, int V>
struct __attribute__((packed, aligned(sizeof(T)))) LaneValues {
  T at[V];
};

template <class T, int V>
__device__ __forceinline__ void load_logits(const T* __restrict__ row, uint32_t experts, int lane, float (&logit)[V]) {
  const uint32_t first = lane * V;
  if (first + V <= experts) {
    const LaneValues<T, V> values = *reinterpret_cast<const LaneValues<T, V>*>(row + first);
#pragma unroll
    for (int i = 0; i < V; ++i) logit[i] = widen(values.at[i]);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) logit[i] = first + i < experts ? widen(row[first + i]) : kNegInf;
  }
}

// A team of TEAM lanes a token: a wave, or, for many tokens, a quarter of one.
// Selection values: score + bias; -inf where masked (a logit of -inf) or outside
// the kept groups; a NaN counts as -1e38, below any score and a finite sum with
// another, so that a token of NaNs still gets different experts, with NaN weights.
//
// Bound by the instructions of `top` rounds of a maximum over the team, which
// cost the same for one token a wave as for four: 16384 tokens of 128 experts,
// top 8, 15.6 us a wave each, 9.7 a quarter each. Few tokens are bound by the
// latency of one: 16 of 256 experts 5.7 us a wave each, of which a launch is
// about three.
template <class T, int V, int TEAM>
__global__ void __launch_bounds__(256)
    route_kernel(const T* __restrict__ logits, uint32_t tokens, uint32_t experts, uint64_t row_stride,
                 const float* __restrict__ bias, uint32_t top, bool softmax, uint32_t groups, uint32_t top_groups,
                 bool renormalize, float scale, int32_t* __restrict__ chosen, float* __restrict__ weights) {
  constexpr int TOKENS = 256 / TEAM;
  __shared__ float values_lds[TOKENS][TEAM * V];
  __shared__ float groups_lds[TOKENS][TEAM];
  struct Choice {
    int32_t expert;
    float score;
  };
  __shared__ Choice choices[TOKENS][TEAM];
  const int lane = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
  const uint32_t token = blockIdx.x * TOKENS + team;
  if (token >= tokens) return;
  float logit[V], score[V], value[V];
  load_logits(logits + token * row_stride, experts, lane, logit);
  auto choose = [&](bool far) __attribute__((always_inline)) {
    scores_of<V, TEAM>(logit, softmax, far, score);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const uint32_t e = lane * V + i;
      value[i] = score[i] + (bias && e < experts ? bias[e] : 0.0f);
      if (value[i] != value[i]) value[i] = -1e38f;
      if (logit[i] == kNegInf) value[i] = kNegInf;
    }
    choices[team][lane] = Choice{-1, 0.0f};
    if (groups > 1) {
      const uint32_t size = experts / groups;
#pragma unroll
      for (int i = 0; i < V; ++i) values_lds[team][lane * V + i] = value[i];
      wave_lds_fence();
      float first = kNegInf, second = kNegInf;
      if (static_cast<uint32_t>(lane) < groups) {
#pragma unroll 8
        for (uint32_t i = 0; i < size; ++i) {
          const float v = values_lds[team][lane * size + i];
          second = fmaxf(second, fminf(first, v));
          first = fmaxf(first, v);
        }
      }
      const float mine = first + (second == kNegInf ? 0.0f : second);
      groups_lds[team][lane] = mine;
      wave_lds_fence();
      // A group is kept if fewer than top_groups come before it: larger ones, or
      // as large ones of a lower index.
      uint32_t before = 0;
#pragma unroll 8
      for (uint32_t g = 0; g < groups; ++g) {
        const float other = groups_lds[team][g];
        before += other > mine || (other == mine && g < static_cast<uint32_t>(lane));
      }
      const bool kept = static_cast<uint32_t>(lane) < groups && before < top_groups;
      const uint64_t mask = __ballot(kept) >> (threadIdx.x % 64 - lane);
      uint32_t group = lane * V / size, inside = lane * V % size;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if (!(mask >> (group & 63) & 1)) value[i] = kNegInf;
        if (++inside == size) inside = 0, ++group;
      }
    }
    for (uint32_t j = 0; j < top; ++j) {
      float best = value[0];
#pragma unroll
      for (int i = 1; i < V; ++i) best = fmaxf(best, value[i]);
      const float largest = team_max<TEAM>(best);
      // The first lane that has it, and there the first value.
      const uint64_t winners = __ballot(best == largest) >> (threadIdx.x % 64 - lane);
      const bool mine = __builtin_ctzll(winners | uint64_t{1} << 63) == lane && largest != kNegInf;
      bool open = mine;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if (open && value[i] == largest) {
          open = false;
          value[i] = kNegInf;
          choices[team][j] = Choice{static_cast<int32_t>(lane * V + i), score[i]};
        }
      }
    }
    wave_lds_fence();
    return choices[team][lane];
  };
  Choice choice = choose(false);
  // Once more, with `far` scores, for a token with a choice that scored 0 (a comparison of every logit with -88
  // would cost 16384 tokens of 256 experts 0.6 us of 14).
  const uint64_t zeros = softmax ? 0 : __ballot(choice.expert >= 0 && choice.score == 0.0f);
  if (__builtin_expect(zeros != 0, 0))
    choice = choose((zeros >> (threadIdx.x % 64 - lane) & ~uint64_t{0} >> (64 - TEAM)) != 0);
  float weight = choice.score;
  if (renormalize) {
    const float total = team_add<TEAM>(choice.score);
    weight = total == 0.0f ? 0.0f : weight / total;
  }
  if (static_cast<uint32_t>(lane) < top) {
    chosen[static_cast<uint64_t>(token) * top + lane] = choice.expert;
    weights[static_cast<uint64_t>(token) * top + lane] = weight * scale;
  }
}

// Gradient of route's weights with respect to the logits, a team a token. With
// w_j = r s_j / Z over the chosen (Z = 1 unless renormalised) and g their
// gradient, d s_j = r (g_j - sum_i g_i s_i / Z) / Z, then through the scores:
// softmax d l = s (d s - sum d s s), sigmoid d l = d s s (1 - s). Renormalised,
// s d s is r (g_j - sum_i g_i p_i) p_j with the shares p = s / Z. The choice
// itself has no gradient.
template <class T, int V, int TEAM>
__global__ void __launch_bounds__(256)
    route_backward_kernel(const T* __restrict__ logits, uint32_t tokens, uint32_t experts, uint64_t row_stride,
                          const int32_t* __restrict__ chosen, const float* __restrict__ d_weights, uint32_t top,
                          bool softmax, bool renormalize, float scale, T* __restrict__ d_logits) {
  constexpr int TOKENS = 256 / TEAM;
  __shared__ float lds[TOKENS][TEAM * V];
  const int lane = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
  const uint32_t token = blockIdx.x * TOKENS + team;
  if (token >= tokens) return;
  int expert = -1;
  float d = 0.0f;
  if (static_cast<uint32_t>(lane) < top) {
    expert = chosen[static_cast<uint64_t>(token) * top + lane];
    d = d_weights[static_cast<uint64_t>(token) * top + lane] * scale;
  }
  float logit[V], score[V];
  load_logits(logits + token * row_stride, experts, lane, logit);
  if (softmax) scores_of<V, TEAM>(logit, true, false, score);
  if (static_cast<uint32_t>(expert) >= experts) expert = -1, d = 0.0f;
#pragma unroll
  for (int i = 0; i < V; ++i) lds[team][lane * V + i] = softmax ? score[i] : logit[i];
  wave_lds_fence();
  const float held = expert >= 0 ? lds[team][expert] : kNegInf;
  wave_lds_fence();
  float s = expert >= 0 ? held : 0.0f, rest = 1.0f;
  if (!softmax) {
    // s and 1 - s of a sigmoid, both from e^-|l|: the difference is 6% off at a logit of 16 and 0 at 17.5.
    const float power = expf(-fabsf(held)), larger = 1.0f / (1.0f + power), smaller = power * larger;
    s = held < 0.0f ? smaller : larger;
    rest = held < 0.0f ? larger : smaller;
  }
  if (renormalize) {
    const float total = team_add<TEAM>(s);
    // By shares: a lone choice, whose weight is constant, has a gradient of exactly zero, and nothing
    // overflows where the scores are small (1 / total is infinite for scores below 2^-128).
    const float share = total == 0.0f ? 0.0f : s / total;
    const float mean = team_add<TEAM>(d * share);
    d = expert < 0 || total == 0.0f ? 0.0f : (d - mean) * share;
  }
  const float common = softmax && !renormalize ? team_add<TEAM>(d * s) : 0.0f;
  if (!softmax) d = (renormalize ? d : d * s) * rest;
#pragma unroll
  for (int i = 0; i < V; ++i) lds[team][lane * V + i] = 0.0f;
  wave_lds_fence();
  if (expert >= 0) lds[team][expert] = d;
  wave_lds_fence();
  LaneValues<T, V> out;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    // The gradient itself, but softmax scores that are not renormalised: there every logit has one, of the common
    // sum. A NaN logit, or softmax score, still gives NaN.
    const float ds = lds[team][lane * V + i];
    float dl;
    if (softmax)
      dl = renormalize ? fmaf(score[i], 0.0f, ds) : score[i] * (ds - common);
    else
      dl = logit[i] != logit[i] ? logit[i] : ds;
    out.at[i] = static_cast<T>(dl);
  }
  T* to = d_logits + static_cast<uint64_t>(token) * experts + lane * V;
  if (static_cast<uint32_t>(lane) * V + V <= experts) {
    *reinterpret_cast<LaneValues<T, V>*>(to) = out;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (lane * V + i < static_cast<int>(experts)) to[i] = out.at[i];
  }
}

// ---- dispatch ----------------------------------------------------------------

constexpr int kDispatchWaves = 16, kDispatchRounds = 4;
constexpr uint32_t kDispatchItems = kDispatchWaves * kDispatchRounds * 64;  // entries of a workgroup

// Lanes whose expert equals this lane's; none for a lane without one.
__device__ __forceinline__ uint64_t same_expert(int expert, uint32_t bits) {
  uint64_t mask = __ballot(expert >= 0);
  for (uint32_t b = 0; b < bits; ++b) {
    const bool set = expert >> b & 1;
    const uint64_t with = __ballot(set);
    mask &= set ? with : ~with;
  }
  return expert < 0 ? 0 : mask;
}

// A wave's entries: `rounds` of 64 consecutive ones from `base` on.
struct DispatchEntries {
  uint32_t base;
  int rounds;
  int expert[kDispatchRounds];     // -1 without one
  uint64_t same[kDispatchRounds];  // lanes of the round with the same expert
};

// Loads a wave's entries and adds them to its own row of the histogram.
__device__ __forceinline__ void count_entries(const int32_t* __restrict__ chosen, uint32_t entries, uint32_t experts,
                                              uint32_t bits, int wave, int lane, DispatchEntries& mine,
                                              uint32_t* hist) {
  // A launch of one workgroup shares few entries out over its waves.
  const uint32_t here = min(kDispatchItems, entries - min(entries, blockIdx.x * kDispatchItems));
  mine.rounds = static_cast<int>((here + kDispatchWaves * 64 - 1) / (kDispatchWaves * 64));
  mine.base = blockIdx.x * kDispatchItems + wave * mine.rounds * 64;
#pragma unroll
  for (int r = 0; r < kDispatchRounds; ++r) {
    const uint32_t i = mine.base + r * 64 + lane;
    const int e = r < mine.rounds && i < entries ? chosen[i] : -1;
    mine.expert[r] = static_cast<uint32_t>(e) < experts ? e : -1;
  }
  for (uint32_t i = threadIdx.x; i < kDispatchWaves * experts; i += 1024) hist[i] = 0;
  __syncthreads();
  uint32_t* row = hist + wave * experts;
#pragma unroll
  for (int r = 0; r < kDispatchRounds; ++r) {
    mine.same[r] = 0;
    if (r >= mine.rounds) continue;
    const uint64_t same = mine.same[r] = same_expert(mine.expert[r], bits);
    if (same && __builtin_ctzll(same) == lane) row[mine.expert[r]] += __builtin_popcountll(same);
    wave_lds_fence();
  }
  __syncthreads();
}

// Counts of each expert's entries, one row a workgroup.
__global__ void __launch_bounds__(1024)
    dispatch_count_kernel(const int32_t* __restrict__ chosen, uint32_t entries, uint32_t experts, uint32_t bits,
                          uint32_t* __restrict__ counts) {
  extern __shared__ uint32_t hist[];  // [waves][experts]
  DispatchEntries mine;
  count_entries(chosen, entries, experts, bits, threadIdx.x >> 6, threadIdx.x & 63, mine, hist);
  for (uint32_t e = threadIdx.x; e < experts; e += 1024) {
    uint32_t total = 0;
#pragma unroll
    for (int w = 0; w < kDispatchWaves; ++w) total += hist[w * experts + e];
    counts[static_cast<uint64_t>(blockIdx.x) * experts + e] = total;
  }
}

// Bound by latencies: 256 entries of 128 experts take 3.3 us, 131072 of 256 (32
// workgroups) 9.1 after 5.1 of counting. With 128 workgroups of a quarter of
// the entries each, reading 128 rows of counts takes 5 us more.
//
// Places every entry: an expert's entries follow those of the experts before
// it, its own of earlier workgroups, waves, rounds and lanes. `counts` are the
// rows of dispatch_count_kernel; NULL in a launch of one workgroup.
__global__ void __launch_bounds__(1024)
    dispatch_place_kernel(const int32_t* __restrict__ chosen, uint32_t entries, uint32_t experts, uint32_t bits,
                          const uint32_t* __restrict__ counts, int32_t* __restrict__ offsets,
                          int32_t* __restrict__ order, int32_t* __restrict__ slots) {
  extern __shared__ uint32_t hist[];  // [waves][experts]
  __shared__ uint32_t wave_total[kDispatchWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // Thread e: the expert's entries in all workgroups, and in earlier ones.
  const uint32_t e = threadIdx.x;
  uint32_t total = 0, before = 0;
  if (e < experts && counts) {
#pragma unroll 16  // loads in flight
    for (uint32_t b = 0; b < gridDim.x; ++b) {
      const uint32_t c = counts[static_cast<uint64_t>(b) * experts + e];
      before += b < blockIdx.x ? c : 0;
      total += c;
    }
  }
  DispatchEntries mine;
  count_entries(chosen, entries, experts, bits, wave, lane, mine, hist);
  if (e < experts && !counts) {
#pragma unroll
    for (int w = 0; w < kDispatchWaves; ++w) total += hist[w * experts + e];
  }
  uint32_t scan = total;
#pragma unroll
  for (int offset = 1; offset < 64; offset <<= 1) {
    const uint32_t v = __shfl_up(scan, offset, 64);
    if (lane >= offset) scan += v;
  }
  if (lane == 63) wave_total[wave] = scan;
  __syncthreads();
  uint32_t all = 0, start = scan - total;
#pragma unroll
  for (int w = 0; w < kDispatchWaves; ++w) {
    if (w < wave) start += wave_total[w];
    all += wave_total[w];
  }
  if (e < experts) {
    if (blockIdx.x == 0) offsets[e] = static_cast<int32_t>(start);
    uint32_t at = start + before, c[kDispatchWaves];
#pragma unroll  // all reads before the writes, which the compiler cannot tell apart
    for (int w = 0; w < kDispatchWaves; ++w) c[w] = hist[w * experts + e];
#pragma unroll
    for (int w = 0; w < kDispatchWaves; ++w) {
      hist[w * experts + e] = at;
      at += c[w];
    }
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) offsets[experts] = static_cast<int32_t>(all);
  __syncthreads();
  uint32_t* next = hist + wave * experts;
#pragma unroll
  for (int r = 0; r < kDispatchRounds; ++r) {
    if (r >= mine.rounds) continue;
    const uint32_t i = mine.base + r * 64 + lane;
    const uint64_t same = mine.same[r];
    const uint32_t rank = __builtin_popcountll(same & ((uint64_t{1} << lane) - 1));
    uint32_t slot = 0;
    if (same) slot = next[mine.expert[r]] + rank;
    wave_lds_fence();
    if (same && rank == 0) next[mine.expert[r]] += __builtin_popcountll(same);
    wave_lds_fence();
    if (i < entries) {
      slots[i] = same ? static_cast<int32_t>(slot) : -1;
      if (same) order[slot] = static_cast<int32_t>(i);
      if (i >= all) order[i] = -1;  // places of entries without an expert, at the end
    }
  }
}

// ---- combine -----------------------------------------------------------------

// Rows of one token's slots whose loads are in flight together.
constexpr int kCombineRows = 8;

// out[t] = sum over j of weights[t][j] * y[slots[t][j]], in the order of j. One
// wave a token and 512 columns, eight a lane.
template <class T, bool STREAM>
__global__ void __launch_bounds__(256)
    combine_kernel(const T* __restrict__ y, uint32_t y_rows, const int32_t* __restrict__ slots,
                   const float* __restrict__ weights, T* __restrict__ out, uint32_t tokens, uint32_t top, uint32_t n) {
  const uint32_t strips = (n + 511) / 512;
  const uint32_t task = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
  const uint32_t token = task / strips;
  if (token >= tokens) return;
  // Lane j holds entry j: the loads of all slots and weights go out together. Lanes past the row stay for their
  // entries, on the row's last columns.
  const uint32_t lane = threadIdx.x & 63, own = task % strips * 512 + lane * 8;
  const uint32_t column = min(own, (n - 1) / 8 * 8);
  uint32_t my_slot = ~0u;
  float my_weight = 0.0f;
  if (lane < top) {
    my_slot = static_cast<uint32_t>(slots[uint64_t{token} * top + lane]);
    my_weight = weights[uint64_t{token} * top + lane];
  }
  const int count = static_cast<int>(min(8u, n - column));
  float sum[8] = {};
  for (uint32_t j0 = 0; j0 < top; j0 += kCombineRows) {
    Raw8<T> raw[kCombineRows];
    uint32_t slot[kCombineRows];
#pragma unroll
    for (int j = 0; j < kCombineRows; ++j) {
      slot[j] = j0 + j < top ? __builtin_amdgcn_readlane(my_slot, j0 + j) : ~0u;
      if (slot[j] < y_rows) raw[j].load(y + uint64_t{slot[j]} * n + column, count);
    }
#pragma unroll
    for (int j = 0; j < kCombineRows; ++j) {
      if (slot[j] >= y_rows) continue;
      const float weight = __builtin_bit_cast(
          float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, my_weight), j0 + j));
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[i] = fmaf(weight, raw[j][i], sum[i]);
    }
  }
  if (column == own) store8<STREAM>(out + uint64_t{token} * n + column, sum, count);
}

constexpr int kGradientRows = 4;

// d_y[slots[t][j]] = weights[t][j] * d_out[t] and d_weights[t][j] = the product
// of d_out[t] and y[slots[t][j]]. One workgroup a token, 2048 columns at a time;
// a part of d_out serves kGradientRows slots.
template <class T, bool STREAM>
__global__ void __launch_bounds__(256)
    combine_backward_kernel(const T* __restrict__ d_out, const T* __restrict__ y, uint32_t y_rows,
                            const int32_t* __restrict__ slots, const float* __restrict__ weights, T* __restrict__ d_y,
                            float* __restrict__ d_weights, uint32_t top, uint32_t n) {
  __shared__ float parts[4][kGradientRows];
  const uint32_t token = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (uint32_t j0 = 0; j0 < top; j0 += kGradientRows) {
    const uint64_t entry = uint64_t{token} * top + j0;
    const uint32_t rows = min(static_cast<uint32_t>(kGradientRows), top - j0);
    uint32_t slot[kGradientRows];
    float weight[kGradientRows], dot[kGradientRows];
#pragma unroll
    for (int j = 0; j < kGradientRows; ++j) {
      slot[j] = j < static_cast<int>(rows) ? static_cast<uint32_t>(slots[entry + j]) : ~0u;
      weight[j] = slot[j] < y_rows ? weights[entry + j] : 0.0f;
      dot[j] = 0.0f;
    }
    for (uint32_t column = threadIdx.x * 8; column < n; column += 2048) {
      const int count = static_cast<int>(min(8u, n - column));
      Raw8<T> g, v[kGradientRows];
      g.load(d_out + uint64_t{token} * n + column, count);
#pragma unroll
      for (int j = 0; j < kGradientRows; ++j)
        if (slot[j] < y_rows) v[j].load(y + uint64_t{slot[j]} * n + column, count);
#pragma unroll
      for (int j = 0; j < kGradientRows; ++j) {
        if (slot[j] >= y_rows) continue;
        float d[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          dot[j] = fmaf(g[i], v[j][i], dot[j]);
          d[i] = weight[j] * g[i];
        }
        store8<STREAM>(d_y + uint64_t{slot[j]} * n + column, d, count);
      }
    }
#pragma unroll
    for (int j = 0; j < kGradientRows; ++j) {
      const float sum = wave_add(dot[j]);
      if (lane == 0) parts[wave][j] = sum;
    }
    __syncthreads();
    if (threadIdx.x < rows)
      d_weights[entry + threadIdx.x] = (parts[0][threadIdx.x] + parts[1][threadIdx.x]) +
                                       (parts[2][threadIdx.x] + parts[3][threadIdx.x]);
    __syncthreads();
  }
}

#define MB_ROUTE_REGISTER_V(T, NAME, V, TEAM)                                               \
  MB_REGISTER_KERNEL("route_" NAME "_" #TEAM "x" #V, (route_kernel<T, V, TEAM>));          \
  MB_REGISTER_KERNEL("route_backward_" NAME "_" #TEAM "x" #V, (route_backward_kernel<T, V, TEAM>))
#define MB_ROUTE_REGISTER(T, NAME)                                                            \
  MB_ROUTE_REGISTER_V(T, NAME, 1, 64);                                                        \
  MB_ROUTE_REGISTER_V(T, NAME, 2, 64);                                                        \
  MB_ROUTE_REGISTER_V(T, NAME, 4, 64);                                                        \
  MB_ROUTE_REGISTER_V(T, NAME, 8, 64);                                                        \
  MB_ROUTE_REGISTER_V(T, NAME, 16, 64);                                                       \
  MB_ROUTE_REGISTER_V(T, NAME, 4, 16);                                                        \
  MB_ROUTE_REGISTER_V(T, NAME, 8, 16);                                                        \
  MB_ROUTE_REGISTER_V(T, NAME, 16, 16);                                                       \
  MB_REGISTER_KERNEL("combine_" NAME, (combine_kernel<T, false>));                            \
  MB_REGISTER_KERNEL("combine_" NAME "_stream", (combine_kernel<T, true>));                   \
  MB_REGISTER_KERNEL("combine_backward_" NAME, (combine_backward_kernel<T, false>));          \
  MB_REGISTER_KERNEL("combine_backward_" NAME "_stream", (combine_backward_kernel<T, true>))
MB_ROUTE_REGISTER(float, "f32");
MB_ROUTE_REGISTER(_Float16, "f16");
MB_ROUTE_REGISTER(__bf16, "bf16");
MB_REGISTER_KERNEL("dispatch_count", dispatch_count_kernel);
MB_REGISTER_KERNEL("dispatch_place", dispatch_place_kernel);

int check_logits(const char* entry, int dtype, const void* logits, uint64_t logits_bytes, uint32_t tokens,
                 uint32_t experts, uint64_t row_stride, uint32_t top) {
  const uint32_t item = elem_bytes(dtype);
  if (!item) return fail(MB_ERR_INVALID, "%s: unknown element type %d", entry, dtype);
  if (experts == 0 || experts > kMostExperts)
    return fail(MB_ERR_INVALID, "%s: %u experts outside 1..%u", entry, experts, kMostExperts);
  if (top == 0 || top > kMostTop || top > experts)
    return fail(MB_ERR_INVALID, "%s: top %u outside 1..%u of %u experts", entry, top, kMostTop, experts);
  if (tokens > (1u << 24)) return fail(MB_ERR_UNSUPPORTED, "%s: at most %u tokens", entry, 1u << 24);
  if (tokens == 0) return MB_OK;
  if (logits == nullptr || row_stride > UINT64_MAX / 8 / tokens ||
      logits_bytes < strided_bytes(tokens, experts, row_stride, item))
    return fail(MB_ERR_INVALID, "%s: logits are NULL or too small for %u tokens of %u experts", entry, tokens, experts);
  if (!aligned(logits, item))
    return fail(MB_ERR_ALIGNMENT, "%s: logits must lie on their elements' %u bytes", entry, item);
  return MB_OK;
}

int check_chosen(const char* entry, const void* chosen, uint64_t chosen_bytes, const void* weights,
                 uint64_t weights_bytes, uint64_t entries) {
  if (chosen == nullptr || weights == nullptr || chosen_bytes < entries * 4 || weights_bytes < entries * 4)
    return fail(MB_ERR_INVALID, "%s: experts or weights are NULL or too small for %llu entries", entry,
                (unsigned long long)entries);
  if (!aligned(chosen, 4) || !aligned(weights, 4))
    return fail(MB_ERR_ALIGNMENT, "%s: experts and weights must lie on 4 bytes", entry);
  return MB_OK;
}

// f(values a lane, lanes a token): a quarter of a wave a token where there are
// enough tokens to fill the chip's SIMDs so, and 16 lanes hold the experts, the
// choices and the groups; else a wave.
template <class F>
void for_experts(uint32_t tokens, uint32_t experts, uint32_t top, uint32_t groups, F&& f) {
  const bool quarter = tokens >= 4096 && experts <= 256 && top <= 16 && groups <= 16;
  auto call = [&](auto v, auto team) { f(v, team); };
  using Wave = std::integral_constant<int, 64>;
  using Row = std::integral_constant<int, 16>;
  if (quarter && experts <= 64)
    call(std::integral_constant<int, 4>{}, Row{});
  else if (quarter && experts <= 128)
    call(std::integral_constant<int, 8>{}, Row{});
  else if (quarter)
    call(std::integral_constant<int, 16>{}, Row{});
  else if (experts <= 64)
    call(std::integral_constant<int, 1>{}, Wave{});
  else if (experts <= 128)
    call(std::integral_constant<int, 2>{}, Wave{});
  else if (experts <= 256)
    call(std::integral_constant<int, 4>{}, Wave{});
  else if (experts <= 512)
    call(std::integral_constant<int, 8>{}, Wave{});
  else
    call(std::integral_constant<int, 16>{}, Wave{});
}

uint64_t dispatch_blocks(uint64_t entries) { return (entries + kDispatchItems - 1) / kDispatchItems; }

}  // namespace
}  // namespace mb

extern "C" {

int mb_route(int dtype, const void* logits, uint64_t logits_bytes, uint32_t tokens, uint32_t experts,
             uint64_t row_stride, const float* bias, uint64_t bias_bytes, uint32_t top, uint32_t scores,
             uint32_t groups, uint32_t top_groups, uint32_t renormalize, float scale, int32_t* chosen,
             uint64_t chosen_bytes, float* weights, uint64_t weights_bytes, void* stream) {
  const char* entry = "mb_route";
  if (int rc = mb::check_logits(entry, dtype, logits, logits_bytes, tokens, experts, row_stride, top)) return rc;
  if (scores > MB_SCORES_SIGMOID) return mb::fail(MB_ERR_INVALID, "%s: unknown scores %u", entry, scores);
  if (groups == 0 || groups > 64 || experts % groups || top_groups == 0 || top_groups > groups)
    return mb::fail(MB_ERR_INVALID, "%s: %u of %u groups: 1 to 64 groups that divide the %u experts", entry,
                    top_groups, groups, experts);
  if (top > experts / groups * top_groups)
    return mb::fail(MB_ERR_INVALID, "%s: top %u exceeds the %u experts of %u groups", entry, top,
                    experts / groups * top_groups, top_groups);
  if (bias && (bias_bytes < uint64_t{experts} * 4 || !mb::aligned(bias, 4)))
    return mb::fail(MB_ERR_INVALID, "%s: the bias must hold %u floats, on 4 bytes", entry, experts);
  if (tokens == 0) return MB_OK;
  if (int rc = mb::check_chosen(entry, chosen, chosen_bytes, weights, weights_bytes, uint64_t{tokens} * top))
    return rc;
  MB_FOR_DTYPE(dtype, mb::for_experts(tokens, experts, top, groups, [&](auto v, auto team) {
    constexpr uint32_t kTokens = 256 / decltype(team)::value;
    mb::route_kernel<T, decltype(v)::value, decltype(team)::value><<<(tokens + kTokens - 1) / kTokens, dim3(256), 0, static_cast<hipStream_t>(stream)>>>(
        static_cast<const T*>(logits), tokens, experts, row_stride, bias, top, scores == MB_SCORES_SOFTMAX,
        top_groups == groups ? 1 : groups, top_groups, renormalize != 0, scale, chosen, weights);
  }));
  return mb::launch_status("route");
}

int mb_route_backward(int dtype, const void* logits, uint64_t logits_bytes, uint32_t tokens, uint32_t experts,
                      uint64_t row_stride, const int32_t* chosen, uint64_t chosen_bytes, const float* d_weights,
                      uint64_t d_weights_bytes, uint32_t top, uint32_t scores, uint32_t renormalize, float scale,
                      void* d_logits, uint64_t d_logits_bytes, void* stream) {
  const char* entry = "mb_route_backward";
  if (int rc = mb::check_logits(entry, dtype, logits, logits_bytes, tokens, experts, row_stride, top)) return rc;
  if (scores > MB_SCORES_SIGMOID) return mb::fail(MB_ERR_INVALID, "%s: unknown scores %u", entry, scores);
  if (tokens == 0) return MB_OK;
  if (int rc = mb::check_chosen(entry, chosen, chosen_bytes, d_weights, d_weights_bytes, uint64_t{tokens} * top))
    return rc;
  const uint32_t item = mb::elem_bytes(dtype);
  if (d_logits == nullptr || d_logits_bytes < uint64_t{tokens} * experts * item)
    return mb::fail(MB_ERR_INVALID, "%s: d_logits are NULL or too small for %u tokens of %u experts", entry, tokens,
                    experts);
  if (!mb::aligned(d_logits, item))
    return mb::fail(MB_ERR_ALIGNMENT, "%s: d_logits must lie on their elements' %u bytes", entry, item);
  MB_FOR_DTYPE(dtype, mb::for_experts(tokens, experts, top, 1, [&](auto v, auto team) {
    constexpr uint32_t kTokens = 256 / decltype(team)::value;
    mb::route_backward_kernel<T, decltype(v)::value, decltype(team)::value><<<(tokens + kTokens - 1) / kTokens, dim3(256), 0, static_cast<hipStream_t>(stream)>>>(
        static_cast<const T*>(logits), tokens, experts, row_stride, chosen, d_weights, top,
        scores == MB_SCORES_SOFTMAX, renormalize != 0, scale, static_cast<T*>(d_logits));
  }));
  return mb::launch_status("route_backward");
}

uint64_t mb_dispatch_workspace(uint64_t entries, uint32_t experts) {
  const uint64_t blocks = mb::dispatch_blocks(entries);
  return blocks > 1 ? blocks * experts * 4 : 0;
}

int mb_dispatch(const int32_t* chosen, uint64_t chosen_bytes, uint64_t entries, uint32_t experts, int32_t* offsets,
                uint64_t offsets_bytes, int32_t* order, uint64_t order_bytes, int32_t* slots, uint64_t slots_bytes,
                void* workspace, uint64_t workspace_bytes, void* stream) {
  const char* entry = "mb_dispatch";
  if (experts == 0 || experts > mb::kMostExperts)
    return mb::fail(MB_ERR_INVALID, "%s: %u experts outside 1..%u", entry, experts, mb::kMostExperts);
  if (entries > (1u << 24)) return mb::fail(MB_ERR_UNSUPPORTED, "%s: at most %u entries", entry, 1u << 24);
  if (offsets == nullptr || offsets_bytes < (uint64_t{experts} + 1) * 4)
    return mb::fail(MB_ERR_INVALID, "%s: offsets are NULL or too small for %u experts", entry, experts);
  if (entries && (chosen == nullptr || order == nullptr || slots == nullptr || chosen_bytes < entries * 4 ||
                  order_bytes < entries * 4 || slots_bytes < entries * 4))
    return mb::fail(MB_ERR_INVALID, "%s: experts, order or slots are NULL or too small for %llu entries", entry,
                    (unsigned long long)entries);
  if (!mb::aligned(chosen, 4) || !mb::aligned(offsets, 4) || !mb::aligned(order, 4) || !mb::aligned(slots, 4) ||
      !mb::aligned(workspace, 4))
    return mb::fail(MB_ERR_ALIGNMENT, "%s: every buffer must lie on 4 bytes", entry);
  const uint64_t needed = mb_dispatch_workspace(entries, experts);
  if (needed && (workspace == nullptr || workspace_bytes < needed))
    return mb::fail(MB_ERR_INVALID, "%s: the workspace is NULL or too small: %llu bytes needed", entry,
                    (unsigned long long)needed);
  const uint32_t blocks = static_cast<uint32_t>(entries ? mb::dispatch_blocks(entries) : 1);
  uint32_t bits = 1;
  while ((1u << bits) < experts) ++bits;
  const uint32_t lds = mb::kDispatchWaves * experts * 4;
  const hipStream_t on = static_cast<hipStream_t>(stream);
  uint32_t* counts = blocks > 1 ? static_cast<uint32_t*>(workspace) : nullptr;
  if (counts) {
    mb::dispatch_count_kernel<<<dim3(blocks), dim3(1024), lds, on>>>(chosen, static_cast<uint32_t>(entries), experts,
                                                                    bits, counts);
    if (int rc = mb::launch_status("dispatch_count")) return rc;
  }
  mb::dispatch_place_kernel<<<dim3(blocks), dim3(1024), lds, on>>>(chosen, static_cast<uint32_t>(entries), experts,
                                                                  bits, counts, offsets, order, slots);
  return mb::launch_status("dispatch_place");
}

static int check_combine(const char* entry, int dtype, const void* y, uint64_t y_bytes, uint64_t y_rows,
                         const int32_t* slots, uint64_t slots_bytes, const float* weights, uint64_t weights_bytes,
                         uint64_t tokens, uint32_t top, uint64_t n) {
  const uint32_t item = mb::elem_bytes(dtype);
  if (!item) return mb::fail(MB_ERR_INVALID, "%s: unknown element type %d", entry, dtype);
  if (top == 0 || top > mb::kMostTop)
    return mb::fail(MB_ERR_INVALID, "%s: %u slots a token outside 1..%u", entry, top, mb::kMostTop);
  if (tokens > (1u << 24) || y_rows > (1u << 24) || n > (1u << 20) || tokens * ((n + 511) / 512) > (1u << 25))
    return mb::fail(MB_ERR_UNSUPPORTED, "%s: %llu tokens of %llu columns exceed one launch", entry,
                    (unsigned long long)tokens, (unsigned long long)n);
  if (tokens == 0) return MB_OK;
  if (y_bytes < y_rows * n * item || (y == nullptr && y_rows * n))
    return mb::fail(MB_ERR_INVALID, "%s: y is NULL or too small for %llu x %llu", entry, (unsigned long long)y_rows,
                    (unsigned long long)n);
  if (!mb::aligned(y, item)) return mb::fail(MB_ERR_ALIGNMENT, "%s: y must lie on its elements' %u bytes", entry, item);
  if (slots == nullptr || weights == nullptr || slots_bytes < tokens * top * 4 || weights_bytes < tokens * top * 4)
    return mb::fail(MB_ERR_INVALID, "%s: slots or weights are NULL or too small for %llu x %u", entry,
                    (unsigned long long)tokens, top);
  if (!mb::aligned(slots, 4) || !mb::aligned(weights, 4))
    return mb::fail(MB_ERR_ALIGNMENT, "%s: slots and weights must lie on 4 bytes", entry);
  return MB_OK;
}

static int check_rows_out(const char* entry, const char* what, const void* p, uint64_t bytes, uint64_t rows,
                          uint64_t n, uint32_t item) {
  if (rows * n && (p == nullptr || bytes < rows * n * item))
    return mb::fail(MB_ERR_INVALID, "%s: %s is NULL or too small for %llu x %llu", entry, what,
                    (unsigned long long)rows, (unsigned long long)n);
  if (!mb::aligned(p, item))
    return mb::fail(MB_ERR_ALIGNMENT, "%s: %s must lie on its elements' %u bytes", entry, what, item);
  return MB_OK;
}

int mb_combine(int dtype, const void* y, uint64_t y_bytes, uint32_t y_rows, const int32_t* slots,
               uint64_t slots_bytes, const float* weights, uint64_t weights_bytes, void* out, uint64_t out_bytes,
               uint32_t tokens, uint32_t top, uint32_t n, void* stream) {
  const char* entry = "mb_combine";
  if (int rc = check_combine(entry, dtype, y, y_bytes, y_rows, slots, slots_bytes, weights, weights_bytes, tokens, top,
                             n))
    return rc;
  if (tokens == 0 || n == 0) return MB_OK;
  if (int rc = check_rows_out(entry, "out", out, out_bytes, tokens, n, mb::elem_bytes(dtype))) return rc;
  const uint64_t tasks = uint64_t{tokens} * ((n + 511) / 512);
  auto launch = [&](auto kernel, auto t) {
    using T = decltype(t);
    kernel<<<dim3(static_cast<uint32_t>((tasks + 3) / 4)), dim3(256), 0, static_cast<hipStream_t>(stream)>>>(
        static_cast<const T*>(y), y_rows, slots, weights, static_cast<T*>(out), tokens, top, n);
  };
  const bool streamed = mb::streams(uint64_t{tokens} * n * mb::elem_bytes(dtype));
  MB_FOR_DTYPE(dtype, {
    if (streamed)
      launch(mb::combine_kernel<T, true>, T());
    else
      launch(mb::combine_kernel<T, false>, T());
  });
  return mb::launch_status("combine");
}

int mb_combine_backward(int dtype, const void* d_out, uint64_t d_out_bytes, const void* y, uint64_t y_bytes,
                        uint32_t y_rows, const int32_t* slots, uint64_t slots_bytes, const float* weights,
                        uint64_t weights_bytes, void* d_y, uint64_t d_y_bytes, float* d_weights,
                        uint64_t d_weights_bytes, uint32_t tokens, uint32_t top, uint32_t n, void* stream) {
  const char* entry = "mb_combine_backward";
  if (int rc = check_combine(entry, dtype, y, y_bytes, y_rows, slots, slots_bytes, weights, weights_bytes, tokens, top,
                             n))
    return rc;
  // A workgroup of 256 a token, and a launch holds at most 2^32 - 1 work items.
  if (tokens > 0xffffffu) return mb::fail(MB_ERR_UNSUPPORTED, "%s: at most %u tokens", entry, 0xffffffu);
  const uint32_t item = mb::elem_bytes(dtype);
  if (tokens == 0) return MB_OK;
  if (int rc = check_rows_out(entry, "d_out", d_out, d_out_bytes, tokens, n, item)) return rc;
  if (int rc = check_rows_out(entry, "d_y", d_y, d_y_bytes, y_rows, n, item)) return rc;
  if (int rc = check_rows_out(entry, "d_weights", d_weights, d_weights_bytes, tokens, top, 4)) return rc;
  auto launch = [&](auto kernel, auto t) {
    using T = decltype(t);
    kernel<<<dim3(tokens), dim3(256), 0, static_cast<hipStream_t>(stream)>>>(
        static_cast<const T*>(d_out), static_cast<const T*>(y), y_rows, slots, weights, static_cast<T*>(d_y),
        d_weights, top, n);
  };
  const bool streamed = mb::streams(uint64_t{y_rows} * n * item);
  MB_FOR_DTYPE(dtype, {
    if (streamed)
      launch(mb::combine_backward_kernel<T, true>, T());
    else
      launch(mb::combine_backward_kernel<T, false>, T());
  });
  return mb::launch_status("combine_backward");
}

}  // extern "C"
