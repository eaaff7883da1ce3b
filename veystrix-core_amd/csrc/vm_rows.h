// Tiles of rows of one group, for kernels whose blocks each work on one: from the lists of a sort (row_sort.hip), or
// found by the block itself among the ids of a small call.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "vm_internal.h"

namespace vm {

// Adds one to a group's count for every lane with a group; with RANK returns the count before the lane's own.  Lanes of
// one group, as in runs of rows of one request, take one addition together: 64 to one address come one after the other.
template <bool RANK>
__device__ __forceinline__ uint32_t count_one(uint32_t* counts, uint32_t g, uint32_t groups) {
  const uint64_t live = __ballot(g < groups);
  if (live == 0) return 0;
  const uint32_t leader = static_cast<uint32_t>(__builtin_ctzll(live));
  const uint32_t one = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(g), leader));
  const uint32_t lane = threadIdx.x & 63u;
  if (__ballot(g < groups && g != one) == 0) {
    uint32_t first = 0;
    if (lane == leader) first = atomicAdd(&counts[one], static_cast<uint32_t>(__popcll(live)));
    if constexpr (!RANK) return 0;
    first = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(first), leader));
    return first + static_cast<uint32_t>(__popcll(live & ((1ull << lane) - 1)));
  }
  uint32_t rank = 0;
  if (g < groups) rank = atomicAdd(&counts[g], 1u);
  return RANK ? rank : 0;
}

// Inclusive sum over the lanes up to one's own: within rows of 16 lanes, then the last lane of a row to the next, then
// that of the first half to the second.
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
  constexpr int kShr = 0x110, kBcast15 = 0x142, kBcast31 = 0x143;
  const auto moved = [&](auto ctrl, auto rows) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), decltype(ctrl)::value,
                                                             decltype(rows)::value, 0xf, true));
  };
  using All = std::integral_constant<int, 0xf>;
  v += moved(std::integral_constant<int, kShr + 1>{}, All{});
  v += moved(std::integral_constant<int, kShr + 2>{}, All{});
  v += moved(std::integral_constant<int, kShr + 4>{}, All{});
  v += moved(std::integral_constant<int, kShr + 8>{}, All{});
  v += moved(std::integral_constant<int, kBcast15>{}, std::integral_constant<int, 0xa>{});
  v += moved(std::integral_constant<int, kBcast31>{}, std::integral_constant<int, 0xc>{});
  return v;
}

// A block's tile, and in every lane the row of the tile's row `lane` (its last one's behind that).
struct BlockTile {
  uint32_t group, rows, group_rows, row;
};

constexpr uint32_t kFindWords = kMaxGroups + 64 + 64 + 4;   // LDS that find_tile takes

// Tile `local` of the eighth `xcd` of the tiles (each XCD a contiguous run): false, in all threads, if there is none.  A
// block of THREADS counts the groups' rows, lays their tiles out as the sort does, and lists the rows of its own in the
// order of the ids, so that all blocks of a launch agree.  At
// most kFindRounds ids per thread.
template <uint32_t THREADS, uint32_t TILE>
__device__ __forceinline__ bool find_tile(const int32_t* ids, uint32_t rows, uint32_t groups, uint32_t xcd, uint32_t local,
                                          uint32_t* lds, BlockTile* out) {
  constexpr uint32_t kRounds = kFindRounds, kWaves = THREADS / 64;
  static_assert(kRounds * kWaves <= 64 && TILE <= 64, "one lane per round and wave, and per row");
  uint32_t *counts = lds, *list = lds + kMaxGroups, *waves = list + 64, *info = waves + 64;
  const uint32_t tid = threadIdx.x, lane = tid & 63u;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  uint32_t g[kRounds];
#pragma unroll
  for (uint32_t j = 0; j < kRounds; ++j) {
    const uint32_t i = j * THREADS + tid;
    g[j] = i < rows ? static_cast<uint32_t>(ids[i]) : groups;
  }
  for (uint32_t i = tid; i < groups; i += THREADS) counts[i] = 0;
  lds_barrier();
#pragma unroll
  for (uint32_t j = 0; j < kRounds; ++j)
    if (j * THREADS < rows) count_one<false>(counts, g[j], groups);
  lds_barrier();
  // a thread's run of groups, their tiles, and the tiles before them
  const uint32_t per = (groups + THREADS - 1) / THREADS, first = min(tid * per, groups), last = min(first + per, groups);
  uint32_t own = 0;
  for (uint32_t i = first; i < last; ++i) own += (counts[i] + TILE - 1) / TILE;
  const uint32_t upto = wave_scan(own);
  if (lane == 63) waves[wave] = upto;
  lds_barrier();
  uint32_t before = upto - own, count = 0;
#pragma unroll
  for (uint32_t w = 0; w < kWaves; ++w) {
    const uint32_t n = waves[w];
    before += w < wave ? n : 0u;
    count += n;
  }
  const uint32_t run = (count + 7) / 8, tile = xcd * run + local;
  if (local >= run || tile >= count) return false;
  if (tile >= before && tile < before + own) {
    uint32_t i = first, k = tile - before;
    for (uint32_t t; k >= (t = (counts[i] + TILE - 1) / TILE); ++i) k -= t;
    info[0] = i;
    info[1] = k * TILE;
    info[2] = counts[i];
  }
  lds_barrier();
  const uint32_t group = info[0], skip = info[1], group_rows = info[2];
#pragma unroll
  for (uint32_t j = 0; j < kRounds; ++j) {
    if (j * THREADS >= rows) break;
    const uint64_t mine = __ballot(g[j] == group);
    if (lane == 0) waves[j * kWaves + wave] = static_cast<uint32_t>(__popcll(mine));
  }
  lds_barrier();
  // of waves of rounds behind the ids nothing is used
  const uint32_t in = waves[lane], ranks = wave_scan(in) - in;
#pragma unroll
  for (uint32_t j = 0; j < kRounds; ++j) {
    if (j * THREADS >= rows) break;
    const uint64_t mine = __ballot(g[j] == group);
    const uint32_t at = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(ranks), j * kWaves + wave)) +
                        static_cast<uint32_t>(__popcll(mine & ((1ull << lane) - 1))) - skip;
    if (g[j] == group && at < TILE) list[at] = j * THREADS + tid;
  }
  lds_barrier();
  out->group = group;
  out->group_rows = group_rows;
  out->rows = min(group_rows - skip, TILE);
  out->row = list[min(lane, out->rows - 1)];
  lds_barrier();   // the list has been read before the LDS is used again
  return true;
}

// The same from a sort's lists.
__device__ __forceinline__ bool listed_tile(const RowTile* tiles, const uint32_t* tile_count, const uint32_t* row_pair,
                                            uint32_t xcd, uint32_t local, BlockTile* out) {
  const uint32_t count = *tile_count, run = (count + 7) / 8, tile = xcd * run + local;
  if (local >= run || tile >= count) return false;
  const RowTile td = tiles[tile];
  out->group = td.group;
  out->rows = td.rows;
  out->group_rows = td.group_rows;
  out->row = row_pair[td.row + min(threadIdx.x & 63u, td.rows - 1)];
  return true;
}

}  // namespace vm
