// Low-rank adapters of many requests beside the projection they share:
//   out[t] = base[t] + s_i * B_i (A_i x[t]),  i = ids[t]        (base[t] where ids[t] names no adapter)
// bf16, A_i [rank, k], B_i [n, rank]; the rank sums stay in fp32 between the two products.
//
// Two forms:
//   k_adapter_rows   a block per row and column split: decode, where every row has an adapter of its own.  Each block
//                    computes the row's rank sums itself (A_i comes from the L2 for all but the first) rather than
//                    wait for another launch.  64 rows of rank 16, 2560 -> 2560: 6.3 us.
//   k_adapter_tiles  tiles of 16 rows sorted by adapter: the rank sums by MFMA with k split over the block's four
//                    waves, joined in LDS, then B_i's product strip by strip, added to base.  The rank sums enter it as
//                    three bf16 parts of eight bits each, three MFMAs, so they lose none of fp32's 24; the second product
//                    is bound by base and out.
//
// Operands come by DMA in whole 128-byte runs of their rows: loads straight in the matrix units' pattern reach 16 bytes a
// clock and CU, these 55.  1777 rows of rank 64, 2560 -> 1280, take 16.7 us, of which finding the rows 2; 8192 of rank 32,
// 2560 -> 2560, 46 behind a sort of 8, where x, base and out (126 MB) alone take 26.5 at the rate of a copy: with about two
// tiles per CU, each block's waves wait for x, then for base and B.  Rank sums in a launch of their own (53 to 58 with the
// sort, for 54) and a third stage (60) were no faster.  Rows off the vector units move by elements: 600 of rank 33, 2560
// wide, 18.1 us (of rank 40 14.1), 600 of rank 32, 2555 wide, 91 (2560 wide 13.2).

#include <hip/hip_ext.h>
#include <hip/hip_runtime.h>

#include "vm_dma.h"
#include "vm_internal.h"
#include "vm_rows.h"

namespace vm {

namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

constexpr uint32_t kThreads = 256;  // of the rows' kernel
constexpr uint32_t kWaves = kThreads / 64;

constexpr uint32_t kCopyRows = 4;  // rows checked per wave of the blocks for rows without an adapter

__device__ uint4 g_adapter_zeros[kChunk / 16];  // units at and behind the end of a row load from here

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
  if (p.vector_n) {  // the columns of a split are whole units of eight
    for (uint32_t n = lo + 8 * t; n < hi; n += 8 * threads) *reinterpret_cast<uint4*>(o + n) = ldg16(b + n);
  } else {
    for (uint32_t n = lo + t; n < hi; n += threads) o[n] = b[n];
  }
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

constexpr uint32_t kTileWaves = 4;
constexpr uint32_t kTileThreads = kTileWaves * 64;
constexpr uint32_t kTileCols = 64;   // columns of a wave's strip

__device__ __forceinline__ f32x4_t mfma(uint4 a, uint4 b, f32x4_t acc) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), acc,
                                                 0, 0, 0);
}

// A rank sum as three bf16 values of its sign, cut off rather than rounded, so that none is infinite unless the sum is.
// Where nothing is left for the second or third it takes 2^-40 of the first, not zero, whose product with an infinity of
// B would be NaN.
__device__ __forceinline__ void split_sum(float r, uint32_t& hi, uint32_t& mid, uint32_t& lo) {
  hi = __float_as_uint(r) >> 16;
  const float first = bf16_to_f32(hi), rest = r - first;
  mid = __float_as_uint(rest) >> 16;
  const float last = rest - bf16_to_f32(mid);
  lo = __float_as_uint(last) >> 16;
  const uint32_t least = __float_as_uint(first * 0x1p-40f) >> 16;
  if (!(fabsf(rest) > 0.0f)) mid = least;   // zero, or none where the sum is infinite
  if (!(fabsf(last) > 0.0f)) lo = least;
}

// LDS of the waves, each its own part.  For the rank sums stage J is A's 16 RF rows of a chunk (main J) and the tile's 16
// rows of x (side J).  After them main J holds a strip of B (64 rows of at most 16 RF ranks: as many bytes), and the two
// sides the strip's products.  Four objects, and whole offsets in one step: past a few of those the compiler no longer
// tells the objects apart and waits for every load in flight before it reads any.
template <int RF>
constexpr uint32_t main_bytes() {
  return 16 * RF * kChunk;
}
constexpr uint32_t kSideBytes = kAdapterTile * kChunk;
template <int J, int RF>
__device__ __forceinline__ uint8_t* lds_main(uint32_t at) {
  __shared__ uint4 buf[kTileWaves * main_bytes<RF>() / 16];
  return reinterpret_cast<uint8_t*>(buf) + at;
}
template <int J>
__device__ __forceinline__ uint8_t* lds_side(uint32_t at) {
  __shared__ uint4 buf[kTileWaves * kSideBytes / 16];
  return reinterpret_cast<uint8_t*>(buf) + at;
}

// Rank sums of the tile, this wave's chunks w, w + 4, .. of 64 inputs.  Operands by DMA, a chunk ahead.
template <int RF>
__device__ __forceinline__ void rank_sums_dma(const AdapterLaunch& p, uint32_t id, uint32_t tile_row,
                                              uint32_t wave, uint32_t lane, f32x4_t acc[RF]) {
  constexpr int kLoads = (kAdapterTile + 16 * RF) / 8;
  const uint32_t lm = lane & 15u, kb = lane >> 4, sub = lane / 8u;
  const uint8_t* src[kLoads];
  const uint32_t unit = ((lane % 8u) ^ tile_swz(sub)) * 16u;   // byte of the lane's unit in a chunk of rows sub, 8 + sub, ..
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const uint32_t r = i * 8u + sub;
    if (i < 2) {
      const uint32_t row = static_cast<uint32_t>(__shfl(static_cast<int>(tile_row), r));
      src[i] = reinterpret_cast<const uint8_t*>(p.x + static_cast<uint64_t>(row) * p.x_stride) + unit;
    } else {
      const uint32_t j = min(r - kAdapterTile, p.rank - 1);
      src[i] = reinterpret_cast<const uint8_t*>(p.a + (static_cast<uint64_t>(id) * p.rank + j) * p.k) + unit;
    }
  }
  const uint32_t k_bytes = p.k * 2, chunks = (k_bytes + kChunk - 1) / kChunk;
  const uint8_t* zeros = reinterpret_cast<const uint8_t*>(g_adapter_zeros);
  VM_KEEP(zeros);
  auto issue = [&](auto J, uint32_t c) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      load_to_lds(c * kChunk + unit < k_bytes ? src[i] + c * kChunk : zeros,
                  i < 2 ? lds_side<decltype(J)::value>(wave * kSideBytes + i * 1024u)
                        : lds_main<decltype(J)::value, RF>(wave * main_bytes<RF>() + (i - 2) * 1024u));
    __builtin_amdgcn_sched_barrier(0);
  };
  const uint32_t s = tile_swz(lm);
  const uint32_t u[2] = {lm * kChunk + (kb ^ s) * 16u, lm * kChunk + ((4u | kb) ^ s) * 16u};
  // a wave without a chunk, and the steps behind a wave's last one, load zeros: every step issues the same loads
  using J0 = std::integral_constant<int, 0>;
  issue(J0{}, wave);
  for (uint32_t c = wave; c < chunks; c += 2 * kTileWaves) {
    unroll<0, 2>([&](auto J) {
      constexpr int j = decltype(J)::value;
      issue(std::integral_constant<int, 1 - j>{}, c + (j + 1) * kTileWaves);
      wait_vm<kLoads>();   // this step's loads have landed; the next one's are in flight
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint4 x = *reinterpret_cast<const uint4*>(lds_side<j>(wave * kSideBytes + u[h]));
#pragma unroll
        for (uint32_t f = 0; f < RF; ++f)
          acc[f] = mfma(*reinterpret_cast<const uint4*>(lds_main<j, RF>(wave * main_bytes<RF>() + u[h] + f * 16 * kChunk)), x,
                        acc[f]);
      }
      wait_lgkm0();        // the stage has been read before it is filled again
      __builtin_amdgcn_sched_barrier(0);
    });
  }
  wait_vm<0>();
}

// The same with every lane fetching its own operands: rows off the 16-byte units.
template <int RF>
__device__ __forceinline__ void rank_sums_direct(const AdapterLaunch& p, uint32_t id, uint32_t tile_row,
                                                 uint32_t wave, uint32_t lane, f32x4_t acc[RF]) {
  const uint32_t lm = lane & 15u, kb = lane >> 4;
  const uint16_t* x = p.x + static_cast<uint64_t>(static_cast<uint32_t>(__shfl(static_cast<int>(tile_row), lm))) * p.x_stride;
  for (uint32_t c = wave * 64u; c < p.k; c += kTileWaves * 64u) {
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) {
      const uint32_t at = c + 32u * h + kb * 8u;
      const uint4 xv = unit_of<false>(x, at, p.k);
#pragma unroll
      for (int f = 0; f < RF; ++f) {
        const uint32_t j = min(f * 16u + lm, p.rank - 1);
        acc[f] = mfma(unit_of<false>(p.a + (static_cast<uint64_t>(id) * p.rank + j) * p.k, at, p.k), xv, acc[f]);
      }
    }
  }
}

// RF 16-row fragments of A (rank up to 16 RF).  VEC_K: x and A, and VEC_R: B move as 16-byte units; VEC_N: base and out.
template <int RF, bool VEC_K, bool VEC_R, bool VEC_N>
__global__ __launch_bounds__(kTileThreads) void k_adapter_tiles(AdapterLaunch p) {
  constexpr int kSteps = (RF + 1) / 2;                      // MFMA steps over the rank
  constexpr uint32_t kPitch = kSteps * 64 + 16;             // bytes of a row of rank sums in LDS
  static_assert(3 * kAdapterTile * kPitch <= kTileWaves * main_bytes<RF>(), "the rank sums fit");
  const uint32_t tid = threadIdx.x, lane = tid & 63u, lm = lane & 15u, kb = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t lin = blockIdx.x;
  if (lin >= p.tile_blocks) {  // rows without an adapter
    const uint32_t first = ((lin - p.tile_blocks) * kTileWaves + wave) * kCopyRows;
    const uint32_t i = first + lane;
    uint64_t left = __ballot(lane < kCopyRows && i < p.rows && static_cast<uint32_t>(p.ids[i]) >= p.adapters);
    while (left != 0) {
      const uint32_t j = static_cast<uint32_t>(__builtin_ctzll(left));
      left &= left - 1;
      copy_row(p, first + j, 0, p.n, lane, 64);
    }
    return;
  }
  // each XCD takes a contiguous run of the tiles with all their splits
  const uint32_t local = (lin >> 3) / p.splits, split = (lin >> 3) % p.splits;
  BlockTile td;
  if (p.tiles != nullptr) {
    if (!listed_tile(p.tiles, p.tile_count, p.row_pair, lin & 7u, local, &td)) return;
  } else {
    uint32_t* words = reinterpret_cast<uint32_t*>(lds_main<0, RF>(0));
    static_assert(kFindWords * 4 <= kTileWaves * main_bytes<RF>(), "a stage holds find_tile's words");
    if (!find_tile<kTileThreads, kAdapterTile>(p.ids, p.rows, p.adapters, lin & 7u, local, words, &td)) return;
  }
  const uint32_t id = td.group, rows = td.rows;
  const auto row_of = [&](uint32_t r) { return static_cast<uint32_t>(__shfl(static_cast<int>(td.row), r)); };
  const float scale = p.scales != nullptr ? p.scales[id] : 1.0f;

  f32x4_t acc[RF];
#pragma unroll
  for (int f = 0; f < RF; ++f) acc[f] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  if constexpr (VEC_K) rank_sums_dma<RF>(p, id, td.row, wave, lane, acc);
  else rank_sums_direct<RF>(p, id, td.row, wave, lane, acc);

  // Strips of 64 columns.  B's rows of a strip lie side by side: one copy of 64 rank values to LDS, whose units are
  // swizzled within their rows where a row is a power of two of them; base goes to registers.  Both are fetched a strip
  // ahead.
  const uint32_t first = split * p.split_cols, end = min(first + p.split_cols, p.n);
  const uint8_t* b = reinterpret_cast<const uint8_t*>(p.b + static_cast<uint64_t>(id) * p.n * p.rank);
  const uint32_t units = p.rank / 8, b_units = p.n * units;   // of a row, of the matrix (VEC_R)
  const uint32_t mask = (units & (units - 1)) == 0 ? units - 1 : 0u, shift = mask == 0 ? 0u : 4u - __builtin_ctz(units);
  constexpr int kB = 2 * RF;
  uint32_t b_unit[kB];   // unit of the strip that the lane copies with load i
  if constexpr (VEC_R) {
#pragma unroll
    for (uint32_t i = 0; i < kB; ++i) {
      const uint32_t v = i * 64u + lane, r = v / units;
      b_unit[i] = r * units + ((v - r * units) ^ ((r >> shift) & mask));
    }
  }
  auto copy_b = [&](auto J, uint32_t col) {
    if constexpr (VEC_R) {
#pragma unroll
      for (uint32_t i = 0; i < kB; ++i)
        load_to_lds(b + static_cast<uint64_t>(min(col * units + b_unit[i], b_units - 1)) * 16u,
                    lds_main<decltype(J)::value, RF>(wave * main_bytes<RF>() + i * 1024u));
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // lane j serves eight columns of row j / 4: 32 h + 8 (j % 4) of each half h of a strip
  const uint32_t my_row = lane >> 2, sub = 8u * (lane & 3u);
  const uint32_t out_row = row_of(my_row);
  const uint16_t* base_row = p.base + static_cast<uint64_t>(out_row) * p.base_stride;
  uint16_t* const out = p.out + static_cast<uint64_t>(out_row) * p.out_stride;
  uint4 base[2][2];
  auto load_base = [&](int j, uint32_t col) {
    if constexpr (VEC_N) {
      // units behind the row's end load its last one, which is not stored
#pragma unroll
      for (uint32_t h = 0; h < 2; ++h) base[j][h] = ldg16(base_row + min(col + 32u * h + sub, p.n - 8u));
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  // the waves' rank sums join: in main 0, and in main 1 their bf16 parts
  f32x4_t* part = reinterpret_cast<f32x4_t*>(lds_main<0, RF>(0));
  constexpr uint32_t kWavePart = main_bytes<RF>() / 16;
#pragma unroll
  for (int f = 0; f < RF; ++f) part[wave * kWavePart + f * 64 + lane] = acc[f];
  uint32_t col = first + wave * kTileCols;
  load_base(0, col);
  lds_barrier();
  // lane holds rank sums 16 f + 4 kb .. +3 of its row; ranks at and behind `rank` are zero
  uint8_t* v_part = lds_main<1, RF>(0);
  for (uint32_t f = wave; f < kSteps * 2; f += kTileWaves) {
    uint32_t bits[3][4];
    f32x4_t v = {0.0f, 0.0f, 0.0f, 0.0f};
    if (f < RF) {
#pragma unroll
      for (uint32_t w = 0; w < kTileWaves; ++w) v += part[w * kWavePart + f * 64 + lane];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) split_sum(f * 16u + kb * 4u + i < p.rank ? v[i] * scale : 0.0f, bits[0][i], bits[1][i], bits[2][i]);
    const uint32_t at = lm * kPitch + (f * 16u + kb * 4u) * 2u;
#pragma unroll
    for (int q = 0; q < 3; ++q)
      *reinterpret_cast<uint2*>(v_part + q * kAdapterTile * kPitch + at) =
          make_uint2(bits[q][0] | (bits[q][1] << 16), bits[q][2] | (bits[q][3] << 16));
  }
  lds_barrier();
  copy_b(std::integral_constant<int, 0>{}, col);
  uint4 sums[3][kSteps];
#pragma unroll
  for (int q = 0; q < 3; ++q)
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
      sums[q][s] = *reinterpret_cast<const uint4*>(v_part + q * kAdapterTile * kPitch + lm * kPitch + s * 64 + kb * 16);
  lds_barrier();  // the rank sums have been read before a strip of B takes their place

  auto strip = [&](auto J) {
    constexpr int j = decltype(J)::value;
    const uint32_t next = col + kTileWaves * kTileCols;
    copy_b(std::integral_constant<int, 1 - j>{}, min(next, p.n - 1));
    load_base(1 - j, next);
    f32x4_t y[4];
#pragma unroll
    for (int f = 0; f < 4; ++f) y[f] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    // this strip's copies have landed: behind them only the next strip's and the stores of the one before
    if constexpr (VEC_R) wait_vm<kB + (VEC_N ? 2 : 0)>();
#pragma unroll
    for (uint32_t f = 0; f < 4; ++f) {
      const uint32_t r = 16u * f + lm;
      uint4 w[kSteps];
#pragma unroll
      for (uint32_t s = 0; s < kSteps; ++s) {
        const uint32_t unit = s * 4u + kb;
        w[s] = make_uint4(0, 0, 0, 0);
        if constexpr (VEC_R) {
          if (unit < units) w[s] = *reinterpret_cast<const uint4*>(
                lds_main<j, RF>(wave * main_bytes<RF>() + (r * units + (unit ^ ((r >> shift) & mask))) * 16u));
        } else {
          const uint16_t* row = p.b + (static_cast<uint64_t>(id) * p.n + min(col + r, p.n - 1)) * p.rank;
          w[s] = unit_of<false>(row, unit * 8u, p.rank);
        }
      }
      // the first parts of all ranks, then the others: small parts next to sums that the first ones have left
#pragma unroll
      for (int q = 0; q < 3; ++q)
#pragma unroll
        for (uint32_t s = 0; s < kSteps; ++s) y[f] = mfma(w[s], sums[q][s], y[f]);
    }
    // lane holds columns 16 f + 4 kb .. +3 of row lm, unit 4 (f % 2) + kb of half f / 2, stored at that ^ (lm % 8)
#pragma unroll
    for (uint32_t f = 0; f < 4; ++f) {
      const uint32_t at = wave * kSideBytes + lm * 128u + ((4u * (f & 1u) + kb) ^ (lm & 7u)) * 16u;
      *reinterpret_cast<f32x4_t*>(f < 2 ? lds_side<0>(at) : lds_side<1>(at)) = y[f];
    }
    wait_lgkm0();  // the wave's own stores, in order
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) {
      float o[8];
#pragma unroll
      for (uint32_t q = 0; q < 2; ++q) {
        const uint32_t from = wave * kSideBytes + my_row * 128u + ((2u * (lane & 3u) + q) ^ (my_row & 7u)) * 16u;
        const f32x4_t v = *reinterpret_cast<const f32x4_t*>(h == 0 ? lds_side<0>(from) : lds_side<1>(from));
#pragma unroll
        for (int i = 0; i < 4; ++i) o[4 * q + i] = v[i];
      }
      if (my_row >= rows) continue;
      const uint32_t at = col + 32u * h + sub;
      if constexpr (VEC_N) {
        const uint32_t v[4] = {base[j][h].x, base[j][h].y, base[j][h].z, base[j][h].w};
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          w[i] = f32_to_bf16(__uint_as_float(v[i] << 16) + o[2 * i]) |
                 (f32_to_bf16(__uint_as_float(v[i] & 0xffff0000u) + o[2 * i + 1]) << 16);
        if (at < p.n) *reinterpret_cast<uint4*>(out + at) = make_uint4(w[0], w[1], w[2], w[3]);
      } else {
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i)
          if (at + i < p.n) out[at + i] = static_cast<uint16_t>(f32_to_bf16(bf16_to_f32(base_row[at + i]) + o[i]));
      }
    }
    wait_lgkm0();  // stage and products have been read before they are written again
    __builtin_amdgcn_sched_barrier(0);
    col = next;
  };
  while (col < end) {
    strip(std::integral_constant<int, 0>{});
    if (col >= end) break;
    strip(std::integral_constant<int, 1>{});
  }
  wait_vm<0>();  // no load into LDS outlives the block
}

template <class Kernel>
hipError_t go(Kernel kernel, uint32_t blocks, uint32_t threads, const AdapterLaunch& p, hipStream_t stream) {
  hipEvent_t start = nullptr, stop = nullptr;
  if (timing_events("adapters", &start, &stop))
    hipExtLaunchKernelGGL(kernel, dim3(blocks), dim3(threads), 0, stream, start, stop, 0, p);
  else
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(threads), 0, stream, p);
  return hipGetLastError();
}

// Operands off the vector units share one instance per rank.
template <int RF>
hipError_t tiles_go(const AdapterLaunch& p, uint32_t blocks, hipStream_t stream) {
  if (p.vector_k && p.vector_rank)
    return p.vector_n ? go(&k_adapter_tiles<RF, true, true, true>, blocks, kTileThreads, p, stream)
                      : go(&k_adapter_tiles<RF, true, true, false>, blocks, kTileThreads, p, stream);
  if (p.vector_k)
    return p.vector_n ? go(&k_adapter_tiles<RF, true, false, true>, blocks, kTileThreads, p, stream)
                      : go(&k_adapter_tiles<RF, true, false, false>, blocks, kTileThreads, p, stream);
  return go(&k_adapter_tiles<RF, false, false, false>, blocks, kTileThreads, p, stream);
}

// Columns per block, a multiple of `least`: as many splits of the columns as keep the blocks of `units` rows or tiles
// within `slots`, since every split of a unit computes its rank sums again.
uint32_t split_columns(uint32_t n, uint32_t units, uint32_t least, uint32_t slots) {
  const uint32_t parts = (n + least - 1) / least;
  const uint32_t want = min(parts, max(1u, slots / units));
  return (parts + want - 1) / want * least;
}

}  // namespace

// Calls whose rank sums are few run one block per row and column split, each of which computes its row's rank sums
// itself; in tiles sixteen rows share them, but a block has to find its rows.  2560 wide, 16 adapters, kernel time of rows
// and tiles: rank 16, 64 / 128 / 200 rows 6.3 / 7.3 / 9.5 us and 7.8 / 7.8 / 8.0; rank 32, 32 / 64 / 100 rows 8.1 / 9.0 / 10.0
// and 8.7 / 8.6 / 9.0; rank 64, 2 / 8 / 32 rows 8.3 / 11.5 / 13.3 and 10.0 / 10.7 / 12.1; rank 128, 2 / 4 rows 19.0 / 19.6 and
// 15.9 / 16.6.
bool adapter_tiled(uint32_t rows, uint32_t rank) {
  return rows > 512 || uint64_t(rows) * rank > (rank <= 32 ? 2048u : 480u);
}

// Every block of a tiled call of few rows finds its own tile: 300 rows of rank 32, 2560 wide, 9.8 us, behind a sort 4.2 +
// 8.9; 1777 of rank 64, 2560 -> 1280, 16.6 and 5.1 + 14.4; 2560 of rank 32 20.6 and 5.5 + 16.5; 4000 26.3 and 6.1 + 20.6, to
// 10240 columns 87.6 and 6.8 + 81.0.
bool adapter_sorted(uint32_t rows) { return rows > 2048; }

uint64_t adapter_blocks(uint32_t rows, uint32_t adapters, uint32_t n, bool tiled) {
  const uint64_t parts = (uint64_t(n) + kThreads - 1) / kThreads;
  const uint64_t units = tiled ? uint64_t(rows) / kAdapterTile + adapters + 7 : rows;
  return (units >= 1024 ? units : units * parts) + rows / (kCopyRows * kTileWaves) + 1;
}

hipError_t launch_adapters(AdapterLaunch p, bool tiled, hipStream_t stream) {
  if (p.rows == 0 || p.rank == 0 || p.rank > kAdapterMaxRank) return hipErrorInvalidValue;
  if (!p.vector_k) p.vector_rank = false;
  if (!tiled) {
    p.split_cols = split_columns(p.n, p.rows, kThreads, 256);
    p.splits = (p.n + p.split_cols - 1) / p.split_cols;
    const uint32_t blocks = p.rows * p.splits;
    if (p.vector_k && p.vector_rank) return go(&k_adapter_rows<true, true>, blocks, kThreads, p, stream);
    if (p.vector_k) return go(&k_adapter_rows<true, false>, blocks, kThreads, p, stream);
    return go(&k_adapter_rows<false, false>, blocks, kThreads, p, stream);
  }
  if (p.tiles == nullptr && p.rows > kFindRounds * kTileThreads) return hipErrorInvalidValue;
  const uint32_t units = row_max_tiles(p.rows, p.adapters, kAdapterTile);
  // By their LDS four, three, two or one block run per CU; five eighths of those, or the one, since each more repeats the
  // rank sums (all: 1777 rows of rank 64, 2560 -> 1280, 21.2 us, so 17.0; 600 of rank 64 19.2 and 15.6; 1500 of rank 32,
  // 5120 -> 2560, 24.9 and 21.1; 300 of rank 128 16.4 and 17.5; half: 600 rows 16.4, three quarters: 1777 rows 21.2).
  const uint32_t slots = p.rank <= 16 ? 640u : p.rank <= 32 ? 480u : p.rank <= 64 ? 320u : 256u;
  p.split_cols = split_columns(p.n, units, kTileWaves * kTileCols, slots);
  p.splits = (p.n + p.split_cols - 1) / p.split_cols;
  p.tile_blocks = (units + 7) / 8 * 8 * p.splits;
  const uint32_t blocks = p.tile_blocks + (p.rows + kCopyRows * kTileWaves - 1) / (kCopyRows * kTileWaves);
  if (p.rank <= 16) return tiles_go<1>(p, blocks, stream);
  if (p.rank <= 32) return tiles_go<2>(p, blocks, stream);
  if (p.rank <= 64) return tiles_go<4>(p, blocks, stream);
  return tiles_go<8>(p, blocks, stream);
}

}  // namespace vm
