// Rows sorted by group on the device, for the grouped products and the adapters: the rows of every group side by side
// and a list of tiles of up to tile_rows of them.  Rows whose id names no group are left out.  Blocks of small calls find
// their tiles without it (vm_rows.h).
//
// The order of a group's rows is the order in which a block's threads counted them, which changes no result: every row
// is its own set of sums.
//
// Calls of up to kOneLaunchRows rows take one launch: every block counts all ids (its own rows, those before and those
// behind) in LDS, lays the groups out by one scan, and places its own rows; nothing has to be zeroed or waited for
// between blocks.  Larger calls count by blocks first (a launch), and every block adds those counts up instead.
// 320 rows of 512 groups 4.8 us, 8192 in runs of one of 32 8.1 (22 in the four launches of the layer's sort); 81920 of
// 512 in two launches 4.9 + 9.4.  It is bound by latency: LDS additions, a scan and the tile list one after the other.

#include <hip/hip_ext.h>
#include <hip/hip_runtime.h>

#include "vm_internal.h"
#include "vm_rows.h"

namespace vm {

namespace {

constexpr uint32_t kThreads = 1024;
constexpr uint32_t kPerThread = 4;
constexpr uint32_t kBlockRows = kThreads * kPerThread;

// Exclusive scan of one value per thread over the block.
__device__ __forceinline__ uint32_t scan_1024(uint32_t v, uint32_t* s_wave) {
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const uint32_t sum = wave_scan(v);
  if (lane == 63) s_wave[wave] = sum;
  __syncthreads();
  uint32_t before = 0;
  for (uint32_t i = 0; i < wave; ++i) before += s_wave[i];
  __syncthreads();
  return before + sum - v;
}

__global__ __launch_bounds__(kThreads) void k_row_count(RowSortLaunch p) {
  __shared__ uint32_t s_count[kThreads];
  const uint32_t t = threadIdx.x, base = blockIdx.x * kBlockRows;
  s_count[t] = 0;
  __syncthreads();
#pragma unroll
  for (uint32_t j = 0; j < kPerThread; ++j) {
    const uint32_t i = base + j * kThreads + t;
    const uint32_t g = i < p.rows ? static_cast<uint32_t>(p.ids[i]) : p.groups;
    count_one<false>(s_count, g, p.groups);
  }
  __syncthreads();
  if (t < p.groups) p.block_counts[static_cast<size_t>(blockIdx.x) * p.groups + t] = s_count[t];
}

// COUNTED: k_row_count has written every block's counts.
template <bool COUNTED>
__global__ __launch_bounds__(kThreads) void k_row_place(RowSortLaunch p) {
  __shared__ uint32_t s_before[kThreads], s_own[kThreads], s_after[kThreads];
  __shared__ uint32_t s_wave[kThreads / 64];
  const uint32_t t = threadIdx.x, first = blockIdx.x * kBlockRows, last = min(first + kBlockRows, p.rows);
  s_before[t] = s_own[t] = s_after[t] = 0;
  __syncthreads();
  uint32_t g[kPerThread], rank[kPerThread];
#pragma unroll
  for (uint32_t j = 0; j < kPerThread; ++j) {
    const uint32_t i = first + j * kThreads + t;
    g[j] = i < last ? static_cast<uint32_t>(p.ids[i]) : p.groups;
    rank[j] = count_one<true>(s_own, g[j], p.groups);
  }
  uint32_t before = 0, total = 0;
  if constexpr (COUNTED) {
    if (t < p.groups) {
#pragma unroll 8
      for (uint32_t b = 0; b < gridDim.x; ++b) {
        const uint32_t n = p.block_counts[static_cast<size_t>(b) * p.groups + t];
        before += b < blockIdx.x ? n : 0u;
        total += n;
      }
    }
  } else {
#pragma unroll 4
    for (uint32_t i = t; i < first; i += kThreads) count_one<false>(s_before, static_cast<uint32_t>(p.ids[i]), p.groups);
#pragma unroll 4
    for (uint32_t i = first + kBlockRows + t; i < p.rows; i += kThreads)
      count_one<false>(s_after, static_cast<uint32_t>(p.ids[i]), p.groups);
  }
  __syncthreads();
  if constexpr (!COUNTED) {
    before = s_before[t];
    total = before + s_own[t] + s_after[t];
  }
  const uint32_t row = scan_1024(total, s_wave);
  __syncthreads();
  s_before[t] = row + before;   // this block's first place in group t
  const uint32_t tiles = (total + p.tile_rows - 1) / p.tile_rows;
  if (blockIdx.x == 0) {
    // the tile list: thread k writes tiles k, k + 1024, .. of the group whose tiles hold k
    const uint32_t tile = scan_1024(tiles, s_wave);
    s_own[t] = tile;            // the ranks have been taken
    s_after[t] = row;
    __syncthreads();
    __shared__ uint32_t s_total[2];
    if (t == kThreads - 1) {
      s_total[0] = tile + tiles;
      s_total[1] = row + total;
    }
    __syncthreads();
    const uint32_t count = s_total[0];
    if (t == 0) *p.tile_count = count;
    for (uint32_t k = t; k < count; k += kThreads) {
      uint32_t lo = 0, hi = kThreads;   // the last group whose first tile is at most k
      while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (s_own[mid] <= k) lo = mid;
        else hi = mid;
      }
      const uint32_t begin = s_after[lo], end = lo + 1 < kThreads ? s_after[lo + 1] : s_total[1];
      const uint32_t start = begin + (k - s_own[lo]) * p.tile_rows;
      p.tiles[k] = RowTile{lo, start, min(end - start, p.tile_rows), end - begin};
    }
  }
  __syncthreads();
#pragma unroll
  for (uint32_t j = 0; j < kPerThread; ++j)
    if (g[j] < p.groups) p.row_pair[s_before[g[j]] + rank[j]] = first + j * kThreads + t;
}

template <class Kernel>
hipError_t go(Kernel kernel, uint32_t blocks, const RowSortLaunch& p, hipStream_t stream) {
  hipEvent_t start = nullptr, stop = nullptr;
  if (timing_events("sort", &start, &stop))
    hipExtLaunchKernelGGL(kernel, dim3(blocks), dim3(kThreads), 0, stream, start, stop, 0, p);
  else
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(kThreads), 0, stream, p);
  return hipGetLastError();
}

}  // namespace

uint32_t row_sort_blocks(uint32_t rows) { return (rows + kBlockRows - 1) / kBlockRows; }

hipError_t launch_row_sort(const RowSortLaunch& p, hipStream_t stream) {
  if (p.rows == 0 || p.groups == 0 || p.groups > kThreads || p.tile_rows == 0) return hipErrorInvalidValue;
  const uint32_t blocks = row_sort_blocks(p.rows);
  if (p.rows <= kOneLaunchRows) return go(&k_row_place<false>, blocks, p, stream);
  const hipError_t e = go(&k_row_count, blocks, p, stream);
  return e == hipSuccess ? go(&k_row_place<true>, blocks, p, stream) : e;
}

}  // namespace vm
