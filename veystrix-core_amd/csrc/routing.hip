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
// One wave per row.  The groups are dealt to the lanes, a power of two of lanes to each and up to 32 neighbouring experts to
// a lane, so that the order (lane, value) is the experts' order and a group's sums stay within its lanes.
//
// 64 bits for all experts would be most of the work (8192 rows of 512 with a sigmoid and a bias, top-10, 31 us).  So choices in
// 32 bits find the candidates: the top_k-th largest of the lanes' largest choices, less what 32 bits may be off, is a bound
// that every chosen expert passes and few others do; those, one to a lane, are compared in 64 bits (12.1 us in a graph, traced
// 12.4; the logits alone are 17 MB, 3.4 at a copy's rate; bound by a wave's instructions, 495 vector and 311 scalar ones by
// counter, a good part of them over a dozen candidates in 64 lanes).  Groups are decided in 32 bits where kept and lost ones
// lie further apart than 32 bits may be off (four of eight groups 16.1 us).  Softmax scores with a bias, or not
// renormalised, take the row's sum in 64 bits, an exponential for every expert (16.6 and 14.2 us; without either 10.9).
// Rows that are not decided so (masses of equal choices, groups that nearly tie) take the whole way in 64 bits.

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

// This wave's stores to LDS before its loads from there.
__device__ __forceinline__ void wait_found() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
  __builtin_amdgcn_s_waitcnt(15 | (3 << 14) | (7 << 4));   // the LDS count at zero
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
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

// v to bf16 in one rounding: where fp32 holds the middle of two bf16 values (the last 16 bits 0x8000) and v lies beside it,
// one step towards v.
__device__ __forceinline__ uint32_t f64_to_bf16(double v) {
  float f = static_cast<float>(v);
  const uint32_t bits = __float_as_uint(f);
  const double rest = v - static_cast<double>(f);
  if ((bits & 0xffffu) == 0x8000u && rest != 0.0) f = __uint_as_float((rest > 0.0) == (f > 0.0f) ? bits + 1 : bits - 1);
  return f32_to_bf16(f);
}

// Writes slot `slot` of a row; expert ~0: none.
__device__ __forceinline__ void write_slot(const RouteLaunch& p, uint32_t row, uint32_t slot, uint32_t expert, double weight) {
  const uint64_t at = static_cast<uint64_t>(row) * p.top_k + slot;
  p.inds[at] = static_cast<int32_t>(expert);
  if (p.weights_dtype == 0) static_cast<uint16_t*>(p.weights)[at] = static_cast<uint16_t>(f64_to_bf16(weight));
  else static_cast<float*>(p.weights)[at] = static_cast<float>(weight);
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

// A lane's experts' values; those it does not have are `none`.  WIDE: whole aligned runs of V values.
template <int V>
__device__ __forceinline__ void load_share(const void* base, uint32_t dtype, uint64_t at, uint32_t count, bool wide, float none,
                                           float v[V]) {
  if (wide && V >= 4) {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = none;
    if (count == 0) return;
    if (dtype == 0) {
      const uint16_t* src = static_cast<const uint16_t*>(base) + at;
      if constexpr (V >= 8) {
#pragma unroll
        for (int j = 0; j < V; j += 8) {
          const uint4 a = ldg16(src + j);
          const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
          for (int i = 0; i < 8; ++i) v[j + i] = bf16_to_f32((w[i / 2] >> (16 * (i % 2))) & 0xffffu);
        }
      } else if constexpr (V == 4) {
        const uint32_t w[2] = {ldg_u32(src), ldg_u32(src + 2)};
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = bf16_to_f32((w[i / 2] >> (16 * (i % 2))) & 0xffffu);
      }
    } else {
      const float* src = static_cast<const float*>(base) + at;
      if constexpr (V >= 4) {
#pragma unroll
        for (int j = 0; j < V; j += 4) {
          const uint4 a = ldg16(src + j);
          v[j] = __uint_as_float(a.x); v[j + 1] = __uint_as_float(a.y);
          v[j + 2] = __uint_as_float(a.z); v[j + 3] = __uint_as_float(a.w);
        }
      }
    }
  } else if (dtype == 0) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const bool in = static_cast<uint32_t>(j) < count;
      const float x = ActBF16::from_bits(ActBF16::load_bits(base, in ? at + j : at - at));
      v[j] = in ? x : none;
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const bool in = static_cast<uint32_t>(j) < count;
      const float x = ActF32::from_bits(ActF32::load_bits(base, in ? at + j : at - at));
      v[j] = in ? x : none;
    }
  }
}

// Keys of 32 bits in the order of floats, as choice_key.
__device__ __forceinline__ uint32_t float_key(float v) {
  if (v != v) return ~0u;
  const uint32_t b = __float_as_uint(v + 0.0f);
  return v == -__builtin_huge_valf() ? 0u : (b >> 31) != 0 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_float(uint32_t key) {
  return __uint_as_float((key >> 31) != 0 ? key & 0x7fffffffu : ~key);
}

// Lanes below this one among `lanes`.
__device__ __forceinline__ uint32_t lanes_below(uint64_t lanes) {
  return __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(lanes >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(lanes), 0));
}

// How far a score in fp32 may be off: exp2 and reciprocal of a step each, a sum and a product round a sigmoid by less than
// 2^-21; the argument of a softmax's exponential loses |l - top| 2^-24 of it, at most 0.37 * 2^-23, and its sum of up to
// 1024 terms in trees of up to 38 levels 38 * 2^-24, each times a score of at most one.
constexpr float kSigmoidOff = 0x1p-20f, kSoftmaxOff = 0x1p-17f;

// The chosen experts from choices in 32 bits, where these decide: groups by a margin, then every expert that may be among
// the top_k, one to a lane, whose choices in 64 bits give the order.  False where they do not: groups too close, or more
// than 64 candidates.
template <int V>
__device__ bool route_narrow(const RouteLaunch& p, uint32_t row, uint32_t lane, const Share& mine, const float l[V],
                             const float bias[V], uint2* found) {
  const bool biased = p.bias != nullptr;
  float score[V];
  float top = 0.0f;
  const bool scores = biased || (p.groups > 1 && p.group_top > 1);
  if (!p.sigmoid) {
    top = -__builtin_huge_valf();
#pragma unroll
    for (int j = 0; j < V; ++j) top = fmaxf(top, l[j]);
    top = wave_max_f32(top);
    if (top == -__builtin_huge_valf()) top = 0.0f;
  }
  if (scores) {
    if (p.sigmoid) {
#pragma unroll
      for (int j = 0; j < V; ++j)
        score[j] = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(l[j] * -0x1.715476p+0f));
    } else {
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        score[j] = __builtin_amdgcn_exp2f((l[j] - top) * 0x1.715476p+0f);
        sum += score[j];
      }
      sum = __builtin_amdgcn_rcpf(wave_sum_all(sum));
#pragma unroll
      for (int j = 0; j < V; ++j) score[j] *= sum;
    }
  }
  uint32_t key[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const float c = biased ? score[j] + bias[j] : l[j];
    key[j] = l[j] == -__builtin_huge_valf() ? 0u : float_key(c);
  }
  const float off = p.sigmoid ? kSigmoidOff : kSoftmaxOff;
  if (p.groups > 1) {
    const bool by_score = !biased && p.group_top > 1;
    uint32_t first = 0, second = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const uint32_t k = by_score && key[j] != 0 ? float_key(score[j]) : key[j];
      second = max(second, min(first, k));
      first = max(first, k);
    }
    for (uint32_t d = 1; d < (1u << p.lane_bits); d <<= 1) {
      const uint32_t f = static_cast<uint32_t>(__shfl_xor(static_cast<int>(first), d));
      const uint32_t s = static_cast<uint32_t>(__shfl_xor(static_cast<int>(second), d));
      second = max(max(second, s), min(first, f));
      first = max(first, f);
    }
    uint32_t rank = first;
    float size = first != 0 ? fabsf(key_float(first)) : 0.0f;
    if (p.group_top > 1 && second != 0) {
      rank = float_key(key_float(first) + key_float(second));
      size += fabsf(key_float(second));
    }
    uint32_t better = 0;
    for (uint32_t g = 0; g < p.groups; ++g) {
      const uint32_t other = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(rank), g << p.lane_bits));
      better += other > rank || (other == rank && g < mine.group) ? 1u : 0u;
    }
    const bool kept = better < p.top_groups;
    if (scores) {   // ranks in 32 bits: kept and lost ones must lie apart
      const uint32_t worst_kept = ~wave_max_u32(mine.group < p.groups && kept ? ~rank : 0u);
      const uint32_t best_lost = wave_max_u32(mine.group < p.groups && !kept ? rank : 0u);
      // of each rank two scores' errors and three roundings of its terms' size
      const float margin = 4.0f * off + 0x1p-21f * wave_max_f32(size);
      if (best_lost != 0 && !(key_float(worst_kept) - key_float(best_lost) > margin)) return false;
    }
    if (!kept) {
#pragma unroll
      for (int j = 0; j < V; ++j) key[j] = 0;
    }
  }
  // The top_k-th largest of the lanes' largest choices is no more than the row's top_k-th largest.
  uint32_t best = 0;
#pragma unroll
  for (int j = 0; j < V; ++j) best = max(best, key[j]);
  // Its first 18 bits are enough: a bound that is 2^-9 low lets few more pass, and takes a comparison a bit.
  uint32_t least = 0;
#pragma unroll
  for (int bit = 31; bit >= 14; --bit) {
    const uint32_t more = least | (1u << bit);
    if (static_cast<uint32_t>(__builtin_popcountll(__ballot(best >= more))) >= p.top_k) least = more;
  }
  // Where fewer lanes hold open experts, the bound of all choices (8192 rows of 512 in 8 groups, one kept, top-16, 21.5 us; the
  // top_k-th largest itself, a wave's maximum at a time, takes a tenth more); still 0: every open expert.
  if (least == 0) {
#pragma unroll
    for (int bit = 31; bit >= 14; --bit) {
      const uint32_t more = least | (1u << bit);
      uint32_t count = 0;
#pragma unroll
      for (int j = 0; j < V; ++j) count += static_cast<uint32_t>(__builtin_popcountll(__ballot(key[j] >= more)));
      if (count >= p.top_k) least = more;
    }
  }
  if (biased && least != 0) {
    const float t = key_float(least);
    // a NaN or an infinity there leaves the bound as it is
    const float low = t - (2.0f * off + 0x1p-21f * fabsf(t));
    if (low - low == 0.0f) least = float_key(low);
  }
  least = max(least, 1u);
  uint32_t before = 0, count = 0;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const uint64_t who = __ballot(key[j] >= least);
    before += lanes_below(who);
    count += static_cast<uint32_t>(__builtin_popcountll(who));
  }
  if (count > 64) return false;
#pragma unroll
  for (int j = 0; j < V; ++j)
    if (key[j] >= least) found[before++] = make_uint2(mine.first + j, __float_as_uint(l[j]));
  __builtin_amdgcn_wave_barrier();
  wait_found();
  // One candidate per lane, in the experts' order.
  const bool live = lane < count;
  const uint2 own = found[live ? lane : 0u];
  const double logit = live ? static_cast<double>(__uint_as_float(own.y)) : 0.0;
  double all = 1.0;
  if (!p.sigmoid && (biased || !p.renormalize)) {
    all = 0.0;
#pragma unroll
    for (int j = 0; j < V; ++j)
      all += l[j] == -__builtin_huge_valf() ? 0.0 : exp(static_cast<double>(l[j]) - static_cast<double>(top));
    all = wave_sum_f64(all);
  }
  // renormalised without a bias the sum over all experts cancels
  const double mass = p.sigmoid ? sigmoid64(logit) : exp(logit - static_cast<double>(top)) / all;
  uint64_t order = 0;
  if (live) order = choice_key(biased ? mass + static_cast<double>(load_any(p.bias, own.x, p.bias_dtype)) : logit);
  uint32_t place = 0;
  for (uint32_t c = 0; c < count; ++c) {   // candidate c's place: those before it, and of its own choice the earlier ones
    const uint64_t its = readlane_u64(order, c);
    const uint64_t before_it = __ballot(order > its) | (__ballot(order == its) & ((1ull << c) - 1ull));
    place = lane == c ? static_cast<uint32_t>(__builtin_popcountll(before_it)) : place;
  }
  const bool chosen = live && place < p.top_k;
  const double total = p.renormalize ? wave_sum_f64(chosen ? mass : 0.0) : 1.0;
  if (chosen) write_slot(p, row, place, own.x, chosen_weight(p, mass, total));
  if (lane >= count && lane < p.top_k) write_slot(p, row, lane, ~0u, 0.0);
  return true;
}

template <int V>
__global__ __launch_bounds__(64 * kRouteWaves) void k_route(RouteLaunch p) {
  __shared__ uint2 s_found[kRouteWaves][64];
  const uint32_t lane = threadIdx.x & 63u;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t row = blockIdx.x * kRouteWaves + wave;
  if (row >= p.rows) return;
  const Share mine = lane_share(p, lane, V);
  float l[V], bias[V];
  const uint64_t base = static_cast<uint64_t>(row) * p.stride;
  load_share<V>(p.logits, p.logits_dtype, base + mine.first, mine.count, p.wide_logits, -__builtin_huge_valf(), l);
  if (p.bias != nullptr) load_share<V>(p.bias, p.bias_dtype, mine.first, mine.count, p.wide_bias, 0.0f, bias);
  if (!route_narrow<V>(p, row, lane, mine, l, bias, s_found[wave])) route_wide<V>(p, row, lane, mine, l);
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

// Whether every lane of a call holds `values` neighbours or none, in whole units of its loads.
bool route_wide_loads(const RouteLaunch& p, const void* base, uint64_t stride, uint32_t dtype, uint32_t values) {
  const uint64_t size = dtype == 0 ? 2 : 4;
  const uint64_t unit = dtype == 0 && values == 4 ? 4 : 16;
  return values >= 4 && p.group_size % values == 0 &&
         (reinterpret_cast<uintptr_t>(base) | (p.rows > 1 ? stride * size : 0)) % unit == 0 &&
         p.group_size * size % unit == 0;
}

hipError_t launch_route(RouteLaunch p, hipStream_t stream) {
  if (p.rows == 0 || p.groups == 0 || p.groups > 64 || p.top_k > 64) return hipErrorInvalidValue;
  p.lane_bits = 0;
  while ((p.groups << (p.lane_bits + 1)) <= 64) ++p.lane_bits;   // 64 lanes hold the groups, 2^lane_bits each
  const uint32_t values = (p.group_size + (1u << p.lane_bits) - 1) >> p.lane_bits;
  uint32_t held = 1;
  while (held < values) held *= 2;
  p.wide_logits = route_wide_loads(p, p.logits, p.stride, p.logits_dtype, held);
  p.wide_bias = route_wide_loads(p, p.bias, 0, p.bias_dtype, held);
  if (values <= 1) return route_go<1>(p, stream);
  if (values <= 2) return route_go<2>(p, stream);
  if (values <= 4) return route_go<4>(p, stream);
  if (values <= 8) return route_go<8>(p, stream);
  if (values <= 16) return route_go<16>(p, stream);
  if (values <= 32) return route_go<32>(p, stream);
  return hipErrorInvalidValue;
}

}  // namespace vm
