// Low-rank adapters of many requests beside the projection they share:
//   out[t] = base[t] + s_i * B_i (A_i x[t]),  i = ids[t]        (base[t] where ids[t] names no adapter)
// bf16, A_i [rank, k], B_i [n, rank]; the rank sums stay in fp32 between the two products.
//
// Two forms:
//   k_adapter_rows   a block per row and column split: decode, where every row has an adapter of its own.  Each block
//                    computes the row's rank sums itself (A_i comes from the L2 for all but the first) rather than
//                    wait for another launch.
//   k_adapter_tiles  tiles of 16 rows sorted by adapter: the rank sums by MFMA with k split over the block's four
//                    waves, joined in LDS, then B_i's product strip by strip, added to base.  The rank sums are split
//                    into a bf16 value and the bf16 rest, two MFMAs, so they lose no more than 2^-16 of themselves;
//                    the second product is bound by base and out, so this is free.

#include <hip/hip_ext.h>
#include <hip/hip_runtime.h>

#include "vm_internal.h"

namespace vm {

namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

constexpr uint32_t kThreads = 256;
constexpr uint32_t kWaves = kThreads / 64;

__device__ uint4 g_adapter_zeros[8];   // units at and behind the end of a row load from here

// Eight values of a bf16 row from element `at`, those at `width` and behind it zero.
template <bool VEC>
__device__ __forceinline__ uint4 unit_of(const uint16_t* row, uint32_t at, uint32_t width) {
  if constexpr (VEC) return ldg16(at < width ? row + at : reinterpret_cast<const uint16_t*>(g_adapter_zeros));
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t lo = at + 2 * j < width ? ldg_u16(row + at + 2 * j) : 0u;
    const uint32_t hi = at + 2 * j + 1 < width ? ldg_u16(row + at + 2 * j + 1) : 0u;
    w[j] = lo | (hi << 16);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ float dot8(uint4 a, uint4 b, float acc) {
  const uint32_t u[4] = {a.x, a.y, a.z, a.w}, v[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
  for (int j = 0; j < 4; ++j)
    acc = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, u[j]), __builtin_bit_cast(bf16x2, v[j]), acc, false);
  return acc;
}

// Columns [lo, hi) of a row without an adapter.
__device__ __forceinline__ void copy_row(const AdapterLaunch& p, uint32_t row, uint32_t lo, uint32_t hi, uint32_t t,
                                         uint32_t threads) {
  const uint16_t* b = p.base + static_cast<uint64_t>(row) * p.base_stride;
  uint16_t* o = p.out + static_cast<uint64_t>(row) * p.out_stride;
  if (b == o) return;
  for (uint32_t n = lo + t; n < hi; n += threads) o[n] = b[n];
}

// ------------------------------------------------------------------ rows ---

template <bool VEC_K, bool VEC_R>
__global__ __launch_bounds__(kThreads) void k_adapter_rows(AdapterLaunch p) {
  constexpr int kRanks = 4;  // rank rows a wave sums at once
  __shared__ float s_v[kAdapterMaxRank];
  const uint32_t tid = threadIdx.x, lane = tid & 63u;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t row = blockIdx.x / p.splits, split = blockIdx.x % p.splits;
  const uint32_t lo = split * p.split_cols, hi = min(lo + p.split_cols, p.n);
  const uint32_t id = static_cast<uint32_t>(p.ids[row]);
  if (id >= p.adapters) {
    copy_row(p, row, lo, hi, tid, kThreads);
    return;
  }
  const uint16_t* x = p.x + static_cast<uint64_t>(row) * p.x_stride;
  const uint16_t* a = p.a + static_cast<uint64_t>(id) * p.rank * p.k;
  const uint16_t* b = p.b + static_cast<uint64_t>(id) * p.n * p.rank;
  const float scale = p.scales != nullptr ? p.scales[id] : 1.0f;
  for (uint32_t j0 = wave * kRanks; j0 < p.rank; j0 += kWaves * kRanks) {
    float acc[kRanks] = {};
    const uint16_t* a_row[kRanks];
#pragma unroll
    for (int q = 0; q < kRanks; ++q) a_row[q] = a + static_cast<uint64_t>(min(j0 + q, p.rank - 1)) * p.k;
#pragma unroll 4
    for (uint32_t at = lane * 8u; at < p.k; at += 512u) {
      const uint4 v = unit_of<VEC_K>(x, at, p.k);
#pragma unroll
      for (int q = 0; q < kRanks; ++q) acc[q] = dot8(v, unit_of<VEC_K>(a_row[q], at, p.k), acc[q]);
    }
#pragma unroll
    for (int q = 0; q < kRanks; ++q) {
      const float s = wave_sum_all(acc[q]);
      if (lane == 0 && j0 + q < p.rank) s_v[j0 + q] = s * scale;
    }
  }
  __syncthreads();
  for (uint32_t n = lo + tid; n < hi; n += kThreads) {
    const uint16_t* b_row = b + static_cast<uint64_t>(n) * p.rank;
    float y = bf16_to_f32(p.base[static_cast<uint64_t>(row) * p.base_stride + n]), acc = 0.0f;
    for (uint32_t r = 0; r < p.rank; r += 8) {
      const uint4 v = unit_of<VEC_R>(b_row, r, p.rank);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j) {
        const float bv = __uint_as_float(j & 1u ? w[j / 2] & 0xffff0000u : w[j / 2] << 16);
        if (VEC_R || r + j < p.rank) acc = fmaf(bv, s_v[r + j], acc);
      }
    }
    p.out[static_cast<uint64_t>(row) * p.out_stride + n] = static_cast<uint16_t>(f32_to_bf16(y + acc));
  }
}

// ----------------------------------------------------------------- tiles ---

__device__ __forceinline__ f32x4_t mfma(uint4 a, uint4 b, f32x4_t acc) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), acc,
                                                 0, 0, 0);
}

// RF 16-row fragments of A (rank up to 16 RF).
template <int RF, bool VEC_K, bool VEC_R>
__global__ __launch_bounds__(kThreads) void k_adapter_tiles(AdapterLaunch p) {
  constexpr uint32_t kRankPad = (RF + 1) / 2 * 32;          // rank in whole MFMA steps
  constexpr uint32_t kPitch = kRankPad * 2 + 16;            // bytes of a row of rank sums in LDS
  constexpr int kDepth = 2;
  __shared__ f32x4_t s_part[kWaves][RF][64];
  __shared__ uint4 s_v[2][kAdapterTile * kPitch / 16];      // the rank sums' bf16 values and rests
  const uint32_t tid = threadIdx.x, lane = tid & 63u, lm = lane & 15u, kb = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t lin = blockIdx.x;
  if (lin >= p.tile_blocks) {  // rows without an adapter
    const uint32_t first = ((lin - p.tile_blocks) * kWaves + wave) * 64u;
    const uint32_t i = first + lane;
    uint64_t left = __ballot(i < p.rows && static_cast<uint32_t>(p.ids[i]) >= p.adapters);
    while (left != 0) {
      const uint32_t j = static_cast<uint32_t>(__builtin_ctzll(left));
      left &= left - 1;
      copy_row(p, first + j, 0, p.n, lane, 64);
    }
    return;
  }
  // each XCD takes a contiguous run of the tiles with all their splits
  const uint32_t local = (lin >> 3) / p.splits, split = (lin >> 3) % p.splits;
  const uint32_t count = *p.tile_count, run = (count + 7) / 8;
  const uint32_t tile = (lin & 7u) * run + local;
  if (local >= run || tile >= count) return;
  const uint2 td = p.tiles[tile];
  const uint32_t id = td.x, row0 = p.row_off[id] + td.y;
  const uint32_t rows = min(p.row_off[id + 1] - row0, kAdapterTile);
  const uint32_t row = p.row_pair[row0 + min(lm, rows - 1)];
  const uint16_t* x = p.x + static_cast<uint64_t>(row) * p.x_stride;
  const uint16_t* a_row[RF];
#pragma unroll
  for (int f = 0; f < RF; ++f)
    a_row[f] = p.a + (static_cast<uint64_t>(id) * p.rank + min(f * 16u + lm, p.rank - 1)) * p.k;

  // rank sums: wave w takes the chunks w, w + 4, .. of 64 inputs; those behind the last one load zeros
  const uint32_t chunks = (p.k + 63) / 64;
  const uint32_t mine = chunks > wave ? (chunks - wave + kWaves - 1) / kWaves : 0u;
  struct Chunk {
    uint4 a[RF][2], x[2];
  } buf[kDepth];
  auto load = [&](Chunk& c, uint32_t i) {
    const uint32_t at = (wave + i * kWaves) * 64u + kb * 8u;
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) {
      c.x[h] = unit_of<VEC_K>(x, at + 32u * h, p.k);
#pragma unroll
      for (int f = 0; f < RF; ++f) c.a[f][h] = unit_of<VEC_K>(a_row[f], at + 32u * h, p.k);
    }
  };
  f32x4_t acc[RF];
#pragma unroll
  for (int f = 0; f < RF; ++f) acc[f] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int j = 0; j < kDepth; ++j) load(buf[j], j);
  for (uint32_t i = 0; i < mine; i += kDepth) {
#pragma unroll
    for (int j = 0; j < kDepth; ++j) {
#pragma unroll
      for (int f = 0; f < RF; ++f) {
        acc[f] = mfma(buf[j].a[f][0], buf[j].x[0], acc[f]);
        acc[f] = mfma(buf[j].a[f][1], buf[j].x[1], acc[f]);
      }
      load(buf[j], i + j + kDepth);
    }
  }
#pragma unroll
  for (int f = 0; f < RF; ++f) s_part[wave][f][lane] = acc[f];
  __syncthreads();
  // lane holds rank sums 16 f + 4 kb .. +3 of its row; ranks at and behind `rank` are zero
  const float scale = p.scales != nullptr ? p.scales[id] : 1.0f;
  uint8_t* v_hi = reinterpret_cast<uint8_t*>(s_v[0]);
  uint8_t* v_lo = reinterpret_cast<uint8_t*>(s_v[1]);
  for (uint32_t f = wave; f < kRankPad / 16; f += kWaves) {
    uint32_t hi[4], lo[4];
    f32x4_t v = {0.0f, 0.0f, 0.0f, 0.0f};
    if (f < RF) v = s_part[0][f][lane] + s_part[1][f][lane] + s_part[2][f][lane] + s_part[3][f][lane];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float r = f * 16u + kb * 4u + i < p.rank ? v[i] * scale : 0.0f;
      hi[i] = f32_to_bf16(r);
      const float rest = r - bf16_to_f32(hi[i]);
      lo[i] = __builtin_isfinite(rest) ? f32_to_bf16(rest) : 0u;  // a sum that rounds to infinity leaves no rest
    }
    const uint32_t at = lm * kPitch + (f * 16u + kb * 4u) * 2u;
    *reinterpret_cast<uint2*>(v_hi + at) = make_uint2(hi[0] | (hi[1] << 16), hi[2] | (hi[3] << 16));
    *reinterpret_cast<uint2*>(v_lo + at) = make_uint2(lo[0] | (lo[1] << 16), lo[2] | (lo[3] << 16));
  }
  __syncthreads();
  constexpr int kSteps = kRankPad / 32;
  uint4 hi[kSteps], lo[kSteps];
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    hi[s] = *reinterpret_cast<const uint4*>(v_hi + lm * kPitch + s * 64 + kb * 16);
    lo[s] = *reinterpret_cast<const uint4*>(v_lo + lm * kPitch + s * 64 + kb * 16);
  }

  const uint32_t first = split * p.split_cols, end = min(first + p.split_cols, p.n);
  const uint16_t* b = p.b + static_cast<uint64_t>(id) * p.n * p.rank;
  const uint16_t* base = p.base + static_cast<uint64_t>(row) * p.base_stride;
  uint16_t* out = p.out + static_cast<uint64_t>(row) * p.out_stride;
  for (uint32_t col = first + wave * 64u; col < end; col += kWaves * 64u) {
    f32x4_t y[4];
#pragma unroll
    for (int f = 0; f < 4; ++f) {
      y[f] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
      const uint16_t* b_row = b + static_cast<uint64_t>(min(col + f * 16u + lm, p.n - 1)) * p.rank;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const uint4 w = unit_of<VEC_R>(b_row, s * 32u + kb * 8u, p.rank);
        y[f] = mfma(w, hi[s], y[f]);
        y[f] = mfma(w, lo[s], y[f]);
      }
    }
    if (lm >= rows) continue;
#pragma unroll
    for (int f = 0; f < 4; ++f) {
      const uint32_t at = col + f * 16u + kb * 4u;
      if (p.quads) {
        if (at >= p.n) continue;
        const uint2 v = *reinterpret_cast<const uint2*>(base + at);
        const float o[4] = {__uint_as_float(v.x << 16) + y[f][0], __uint_as_float(v.x & 0xffff0000u) + y[f][1],
                            __uint_as_float(v.y << 16) + y[f][2], __uint_as_float(v.y & 0xffff0000u) + y[f][3]};
        *reinterpret_cast<uint2*>(out + at) =
            make_uint2(f32_to_bf16(o[0]) | (f32_to_bf16(o[1]) << 16), f32_to_bf16(o[2]) | (f32_to_bf16(o[3]) << 16));
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (at + i < p.n) out[at + i] = static_cast<uint16_t>(f32_to_bf16(bf16_to_f32(base[at + i]) + y[f][i]));
      }
    }
  }
}

template <class Kernel>
hipError_t go(Kernel kernel, uint32_t blocks, const AdapterLaunch& p, hipStream_t stream) {
  hipEvent_t start = nullptr, stop = nullptr;
  if (timing_events("adapters", &start, &stop))
    hipExtLaunchKernelGGL(kernel, dim3(blocks), dim3(kThreads), 0, stream, start, stop, 0, p);
  else
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(kThreads), 0, stream, p);
  return hipGetLastError();
}

template <int RF>
hipError_t tiles_go(const AdapterLaunch& p, uint32_t blocks, hipStream_t stream) {
  if (p.vector_k && p.vector_rank) return go(&k_adapter_tiles<RF, true, true>, blocks, p, stream);
  if (p.vector_k) return go(&k_adapter_tiles<RF, true, false>, blocks, p, stream);
  return go(&k_adapter_tiles<RF, false, false>, blocks, p, stream);
}

}  // namespace

uint64_t adapter_blocks(uint32_t rows, uint32_t adapters, uint32_t n, bool tiled) {
  const uint64_t passes = (uint64_t(n) + kThreads - 1) / kThreads;
  const uint64_t units = tiled ? (uint64_t(rows) + kAdapterTile - 1) / kAdapterTile + adapters + 7 : rows;
  return (units >= 512 ? units : units * passes) + rows / (64 * kWaves) + 1;
}

hipError_t launch_adapters(AdapterLaunch p, bool tiled, hipStream_t stream) {
  if (p.rows == 0 || p.rank == 0 || p.rank > kAdapterMaxRank) return hipErrorInvalidValue;
  if (!p.vector_k) p.vector_rank = false;
  const uint32_t units = tiled ? grouped_max_tiles(p.rows, p.adapters, kAdapterTile) : p.rows;
  // columns per block: all of them once the rows fill the chip twice, at least one pass of the block
  const uint32_t passes = (p.n + kThreads - 1) / kThreads;
  const uint32_t want = units >= 512 ? 1u : min(passes, (512 + units - 1) / units);
  p.split_cols = (passes + want - 1) / want * kThreads;
  p.splits = (p.n + p.split_cols - 1) / p.split_cols;
  if (!tiled) {
    const uint32_t blocks = p.rows * p.splits;
    if (p.vector_k && p.vector_rank) return go(&k_adapter_rows<true, true>, blocks, p, stream);
    if (p.vector_k) return go(&k_adapter_rows<true, false>, blocks, p, stream);
    return go(&k_adapter_rows<false, false>, blocks, p, stream);
  }
  p.tile_blocks = (units + 7) / 8 * 8 * p.splits;
  const uint32_t blocks = p.tile_blocks + (p.rows + 64 * kWaves - 1) / (64 * kWaves);
  if (p.rank <= 16) return tiles_go<1>(p, blocks, stream);
  if (p.rank <= 32) return tiles_go<2>(p, blocks, stream);
  if (p.rank <= 64) return tiles_go<4>(p, blocks, stream);
  return tiles_go<8>(p, blocks, stream);
}

}  // namespace vm
