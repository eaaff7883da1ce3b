// From a router's logits to experts (vm_select_experts).
//
//   score  = softmax over the row's open experts (logit above -inf), or 1 / (1 + e^-logit)
//   choice = score + bias; without a bias the logit itself, which orders the experts as their scores do
//   kept   = the top_groups groups whose group_top best choices have the largest sum
//   chosen = the top_k largest choices of the kept groups, the lowest index of several equal ones first
//   weight = score (over the chosen scores' sum if renormalised) * factor
//
// Choices are compared as they are in 64 bits: biases and scores lie so close that in 32 bits every tenth window of 8192
// tokens would hold a token whose experts, or their order, differ from the formula's.
//
// One wave per row.  The groups are dealt to the lanes, a power of two of lanes to each and V neighbouring experts to a
// lane, so that the order (lane, value) is the experts' order and a group's sums stay within its lanes.

#include <hip/hip_ext.h>
#include <hip/hip_runtime.h>

#include "vm_common.h"
#include "vm_internal.h"

namespace vm {

namespace {

constexpr uint32_t kRouteWaves = 4;

// Keys of 64 bits in the order of the numbers: 0 for what cannot be chosen, above all others for NaN.  Both zeros are one.
__device__ __forceinline__ uint64_t choice_key(double v) {
  if (v != v) return ~0ull;
  const uint64_t b = __builtin_bit_cast(uint64_t, v + 0.0);
  const uint64_t key = (b >> 63) != 0 ? ~b : b | (1ull << 63);
  return v == -__builtin_huge_val() ? 0 : key;
}
__device__ __forceinline__ double key_value(uint64_t key) {
  return __builtin_bit_cast(double, (key >> 63) != 0 ? key & ~(1ull << 63) : ~key);
}

__device__ __forceinline__ uint64_t shfl_xor_u64(uint64_t v, int d) {
  const uint32_t lo = static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), d));
  const uint32_t hi = static_cast<uint32_t>(__shfl_xor(static_cast<int>(v >> 32), d));
  return (static_cast<uint64_t>(hi) << 32) | lo;
}
__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v += __builtin_bit_cast(double, shfl_xor_u64(__builtin_bit_cast(uint64_t, v), d));
  return v;
}

// Largest key of the wave and the first lane that holds it.
__device__ __forceinline__ uint64_t wave_first_max(uint64_t key, uint32_t* lane) {
  const uint32_t hi = wave_max_u32(static_cast<uint32_t>(key >> 32));
  uint64_t who = __ballot(static_cast<uint32_t>(key >> 32) == hi);
  uint32_t lo = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(key), __builtin_ctzll(who)));
  if ((who & (who - 1)) != 0) {
    lo = wave_max_u32(static_cast<uint32_t>(key >> 32) == hi ? static_cast<uint32_t>(key) : 0u);
    who = __ballot(key == ((static_cast<uint64_t>(hi) << 32) | lo));
  }
  *lane = static_cast<uint32_t>(__builtin_ctzll(who));
  return (static_cast<uint64_t>(hi) << 32) | lo;
}

// What a lane holds: experts first .. first + count - 1 of group `group`.
struct Share {
  uint32_t group, first, count;
};

__device__ __forceinline__ Share lane_share(const RouteLaunch& p, uint32_t lane, uint32_t values) {
  const uint32_t group = lane >> p.lane_bits, sub = lane & ((1u << p.lane_bits) - 1u);
  const uint32_t at = sub * values;
  const uint32_t count = group < p.groups && at < p.group_size ? min(p.group_size - at, values) : 0u;
  return {group, group * p.group_size + at, count};
}

__device__ __forceinline__ double sigmoid64(double v) { return 1.0 / (1.0 + exp(-v)); }

// Whether the lane's group is among the kept ones; `rank` is its key, the same in all its lanes.
__device__ __forceinline__ bool group_kept(const RouteLaunch& p, uint32_t group, uint64_t rank) {
  uint32_t better = 0;
  for (uint32_t g = 0; g < p.groups; ++g) {
    const uint64_t other = readlane_u64(rank, g << p.lane_bits);
    better += other > rank || (other == rank && g < group) ? 1u : 0u;
  }
  return better < p.top_groups;
}

// Writes slot `slot` of a row; expert ~0: none.
__device__ __forceinline__ void write_slot(const RouteLaunch& p, uint32_t row, uint32_t slot, uint32_t expert, double weight) {
  const uint64_t at = static_cast<uint64_t>(row) * p.top_k + slot;
  p.inds[at] = static_cast<int32_t>(expert);
  const float w = static_cast<float>(weight);
  if (p.weights_dtype == 0) static_cast<uint16_t*>(p.weights)[at] = static_cast<uint16_t>(f32_to_bf16(w));
  else static_cast<float*>(p.weights)[at] = w;
}

// score * factor / total of the chosen; scores that are all too small for 64 bits weigh nothing.
__device__ __forceinline__ double chosen_weight(const RouteLaunch& p, double score, double total) {
  if (!p.renormalize) return score * p.factor;
  return total == 0.0 ? 0.0 : score / total * p.factor;
}

// Everything in 64 bits.
template <int V>
__device__ void route_wide(const RouteLaunch& p, uint32_t row, uint32_t lane, const Share& mine, const float l[V]) {
  double score[V];
  uint64_t key[V];
  if (p.sigmoid) {
#pragma unroll
    for (int j = 0; j < V; ++j) score[j] = sigmoid64(l[j]);
  } else {
    float top = -__builtin_huge_valf();
#pragma unroll
    for (int j = 0; j < V; ++j) top = fmaxf(top, l[j]);
    top = wave_max_f32(top);
    if (top == -__builtin_huge_valf()) top = 0.0f;
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      score[j] = l[j] == -__builtin_huge_valf() ? 0.0 : exp(static_cast<double>(l[j]) - static_cast<double>(top));
      sum += score[j];
    }
    sum = wave_sum_f64(sum);
#pragma unroll
    for (int j = 0; j < V; ++j) score[j] = sum == 0.0 ? 0.0 : score[j] / sum;
  }
#pragma unroll
  for (int j = 0; j < V; ++j) {
    double c = l[j];
    if (p.bias != nullptr && static_cast<uint32_t>(j) < mine.count)
      c = score[j] + static_cast<double>(load_any(p.bias, mine.first + j, p.bias_dtype));
    key[j] = l[j] == -__builtin_huge_valf() ? 0 : choice_key(c);   // closed, or behind the lane's last expert
  }
  if (p.groups > 1) {
    const bool by_score = p.bias == nullptr && p.group_top > 1;    // sums of scores, not of logits
    uint64_t first = 0, second = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const uint64_t k = by_score && key[j] != 0 ? choice_key(score[j]) : key[j];
      second = max(second, min(first, k));
      first = max(first, k);
    }
    for (uint32_t d = 1; d < (1u << p.lane_bits); d <<= 1) {
      const uint64_t f = shfl_xor_u64(first, static_cast<int>(d)), s = shfl_xor_u64(second, static_cast<int>(d));
      second = max(max(second, s), min(first, f));
      first = max(first, f);
    }
    uint64_t rank = first;
    if (p.group_top > 1 && second != 0) rank = choice_key(key_value(first) + key_value(second));
    if (!group_kept(p, mine.group, rank)) {
#pragma unroll
      for (int j = 0; j < V; ++j) key[j] = 0;
    }
  }
  uint32_t expert = ~0u;
  double kept = 0.0;
  for (uint32_t slot = 0; slot < p.top_k; ++slot) {
    uint64_t best = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) best = max(best, key[j]);
    uint32_t who;
    if (wave_first_max(best, &who) == 0) break;
    uint32_t at = 0;
    double s = 0.0;
    bool found = false;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const bool here = !found && key[j] == best;
      at = here ? mine.first + j : at;
      s = here ? score[j] : s;
      if (here && lane == who) key[j] = 0;
      found = found || here;
    }
    const uint32_t e = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(at), who));
    const double es = __builtin_bit_cast(double, readlane_u64(__builtin_bit_cast(uint64_t, s), who));
    if (lane == slot) {
      expert = e;
      kept = es;
    }
  }
  const double total = p.renormalize ? wave_sum_f64(kept) : 1.0;
  if (lane < p.top_k) write_slot(p, row, lane, expert, expert == ~0u ? 0.0 : chosen_weight(p, kept, total));
}

template <int V>
__global__ __launch_bounds__(64 * kRouteWaves) void k_route(RouteLaunch p) {
  const uint32_t lane = threadIdx.x & 63u;
  const uint32_t row = blockIdx.x * kRouteWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (row >= p.rows) return;
  const Share mine = lane_share(p, lane, V);
  float l[V];
  const uint64_t base = static_cast<uint64_t>(row) * p.stride;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const bool in = static_cast<uint32_t>(j) < mine.count;
    const float v = load_any(p.logits, base + (in ? mine.first + j : 0u), p.logits_dtype);
    l[j] = in ? v : -__builtin_huge_valf();
  }
  route_wide<V>(p, row, lane, mine, l);
}

template <int V>
hipError_t route_go(const RouteLaunch& p, hipStream_t stream) {
  const dim3 grid((p.rows + kRouteWaves - 1) / kRouteWaves), block(64 * kRouteWaves);
  hipEvent_t start = nullptr, stop = nullptr;
  if (timing_events("route", &start, &stop))
    hipExtLaunchKernelGGL(k_route<V>, grid, block, 0, stream, start, stop, 0, p);
  else
    hipLaunchKernelGGL(k_route<V>, grid, block, 0, stream, p);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_route(RouteLaunch p, hipStream_t stream) {
  if (p.rows == 0 || p.groups == 0 || p.groups > 64 || p.top_k > 64) return hipErrorInvalidValue;
  p.lane_bits = 0;
  while ((p.groups << (p.lane_bits + 1)) <= 64) ++p.lane_bits;   // 64 lanes hold the groups, 2^lane_bits each
  const uint32_t values = (p.group_size + (1u << p.lane_bits) - 1) >> p.lane_bits;
  if (values <= 1) return route_go<1>(p, stream);
  if (values <= 2) return route_go<2>(p, stream);
  if (values <= 4) return route_go<4>(p, stream);
  if (values <= 8) return route_go<8>(p, stream);
  if (values <= 16) return route_go<16>(p, stream);
  if (values <= 32) return route_go<32>(p, stream);
  return hipErrorInvalidValue;
}

}  // namespace vm
