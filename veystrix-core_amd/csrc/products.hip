// Products of routed rows with the matrix of their expert: out[i] = x[i / x_div] . W[ids[i]]^T, fp32 sums, bf16 or MX
// operands (vm_mx.h), optionally y = silu(gate) * up over a matrix of gate rows then up rows, and the output in bf16
// or MX.
//
// Both formats move through the kernels as 128-byte chunks of a row (64 bf16 or 128 e4m3 inputs) made of eight
// 16-byte units; a lane's operands of one chunk are units kb and 4 + kb of row lane % 16, kb = lane / 16, the same k
// for the matrix and the rows.  A bf16 unit is one v_mfma_f32_16x16x32_bf16 operand.  An MX unit is converted to two
// of them: an e4m3 value times its group's power of two is a bf16 value, so both formats have the bf16 unit's sums (its
// cancelled terms survive to 2^-24 of the largest).  The scaled 8-bit MFMA, at twice the rate, lost those below 2^-16
// of its group's largest product and put 2e-5 of the terms' magnitude on a sum (measured), which an MX output shows as
// flipped values; these products read hundreds of matrices for a few rows each and wait for HBM, not for the MFMA.
// The matrix is the first operand, the rows the second, so a lane receives outputs 4 kb .. +3 of row lane % 16: four
// neighbouring outputs to store.
//
// With hundreds of experts the weights are most of the bytes, each read for a few to a few hundred rows.  Three forms:
//   k_stream, rows one by one   calls of few routed rows: no sort, one launch; a block per routed row and 64 matrix
//                               rows, the matrix streamed from HBM into the operand registers.
//   k_stream, tiles of 16       few rows per expert: the same over rows sorted by expert, so each matrix is read once
//                               per 16 rows.
//   k_tiles                     tiles of 64 or 128 sorted rows by 128 matrix rows, both staged through LDS by DMA.
// Rows whose id names no expert are written as zeros by blocks behind the tiles'.

#include <hip/hip_ext.h>
#include <hip/hip_runtime.h>

#include <type_traits>

#include "vm_internal.h"
#include "vm_mx.h"

namespace vm {

namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

constexpr uint32_t kChunk = 128;          // bytes of a row per step
constexpr int kStrip = 4;                 // 16-row fragments of the matrix per wave
constexpr uint32_t kZeroRows = 64;        // routed rows checked per wave of the zeroing blocks

enum : int { kOutBf16 = 0, kOutMx = 1 };

__device__ uint4 g_product_zeros[kChunk / 16];  // units at and behind the end of a row load from here

// One lane's MFMA operands of a 16-byte unit: itself, or two of bf16 values, e4m3 times 2^scale.  `scale` is the float
// 2^(s - 127) of the scale byte s; bf16's subnormals and groups of scale 2^-127 come out as zero.
template <bool MX>
struct Operand {
  uint4 part[MX ? 2 : 1];
  __device__ __forceinline__ Operand(const uint4& unit, float scale) {
    if constexpr (MX) {
      const uint32_t w[4] = {unit.x, unit.y, unit.z, unit.w};
      uint32_t o[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        o[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i], scale, false));
        o[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i], scale, true));
      }
      part[0] = make_uint4(o[0], o[1], o[2], o[3]);
      part[1] = make_uint4(o[4], o[5], o[6], o[7]);
    } else {
      part[0] = unit;
    }
  }
};

// acc += matrix unit x row unit
template <bool MX>
__device__ __forceinline__ f32x4_t unit_mfma(const Operand<MX>& w, const Operand<MX>& x, f32x4_t acc) {
#pragma unroll
  for (int i = 0; i < (MX ? 2 : 1); ++i)
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, w.part[i]),
                                                  __builtin_bit_cast(bf16x8_t, x.part[i]), acc, 0, 0, 0);
  return acc;
}

// The scale of a lane's unit h (inputs 16 kb .. +15 of half h of the chunk) from the chunk's four scale bytes.
__device__ __forceinline__ float unit_scale(uint32_t bytes, uint32_t kb, int h) {
  return __uint_as_float(((bytes >> (16 * h + 8u * (kb >> 1))) & 0xffu) << 23);
}

// The four scale bytes of chunk c of one row, those behind its end zero.  WHOLE: whole chunks, aligned rows.
template <bool WHOLE>
__device__ __forceinline__ uint32_t chunk_scales(const uint8_t* row, uint32_t c, uint32_t groups) {
  if constexpr (WHOLE) return ldg_u32(row + c * 4u);
  uint32_t v = 0;
#pragma unroll
  for (uint32_t j = 0; j < 4; ++j)
    if (c * 4u + j < groups) v |= static_cast<uint32_t>(row[c * 4u + j]) << (8u * j);
  return v;
}

// Matrix row behind row `r` (0..63) of a wave's strip that starts at output column `col`: with SwiGLU fragments
// alternate between 16 gate rows and the 16 up rows of the same outputs.
template <bool SWIGLU>
__device__ __forceinline__ uint32_t matrix_row(uint32_t col, uint32_t r, uint32_t n) {
  if constexpr (SWIGLU) return min(col + (r >> 5) * 16u + (r & 15u), n - 1u) + ((r >> 4) & 1u) * n;
  else return min(col + r, n - 1u);
}

// Outputs per strip.
template <bool SWIGLU>
constexpr uint32_t strip_cols() {
  return SWIGLU ? 32u : 64u;
}

// silu(g) * u with the hardware exp2 and reciprocal, two or three units of fp32's last place each and one rounding to
// the output's type behind them.
__device__ __forceinline__ float swiglu(float g, float u) {
  return g * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(g * -1.44269504088896f)) * u;
}

// Stores one strip of one 16-row fragment: lane holds outputs 4 kb .. +3 of each fragment for its routed row.
template <bool SWIGLU, int OUT>
__device__ __forceinline__ void store_strip(const ProductLaunch& p, const f32x4_t acc[kStrip], uint32_t col,
                                            uint32_t pair, bool live, uint32_t kb) {
  constexpr int kFrags = SWIGLU ? kStrip / 2 : kStrip;
  float y[kFrags][4];
#pragma unroll
  for (int f = 0; f < kFrags; ++f)
#pragma unroll
    for (int i = 0; i < 4; ++i) y[f][i] = SWIGLU ? swiglu(acc[2 * f][i], acc[2 * f + 1][i]) : acc[f][i];
  if constexpr (OUT == kOutMx) {
    static_assert(SWIGLU || OUT == kOutBf16, "a strip of SwiGLU outputs is one group");
    uint32_t m = 0;
#pragma unroll
    for (int f = 0; f < kFrags; ++f)
#pragma unroll
      for (int i = 0; i < 4; ++i) m = max(m, mx_magnitude(y[f][i]));
    m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), 16)));
    m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), 32)));
    const uint32_t e = mx_scale(m);
    if (!live) return;
    const uint64_t first = static_cast<uint64_t>(pair) * p.n + col;
#pragma unroll
    for (int f = 0; f < kFrags; ++f)
      *reinterpret_cast<uint32_t*>(p.values + first + f * 16 + kb * 4) = mx_pack4(y[f][0], y[f][1], y[f][2], y[f][3], e);
    if (kb == 0) p.scales[first / kMxGroup] = static_cast<uint8_t>(e);
  } else {
    if (!live) return;
    uint16_t* row = p.out + static_cast<uint64_t>(pair) * p.n;
#pragma unroll
    for (int f = 0; f < kFrags; ++f) {
      const uint32_t at = col + f * 16 + kb * 4;
      if (p.n % 4 == 0) {
        if (at < p.n)
          *reinterpret_cast<uint2*>(row + at) = make_uint2(f32_to_bf16(y[f][0]) | (f32_to_bf16(y[f][1]) << 16),
                                                           f32_to_bf16(y[f][2]) | (f32_to_bf16(y[f][3]) << 16));
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (at + i < p.n) row[at + i] = static_cast<uint16_t>(f32_to_bf16(y[f][i]));
      }
    }
  }
}

// One wave zeroes output row `pair`.
template <int OUT>
__device__ __forceinline__ void zero_row(const ProductLaunch& p, uint32_t pair, uint32_t lane) {
  if constexpr (OUT == kOutMx) {
    uint32_t* v = reinterpret_cast<uint32_t*>(p.values + static_cast<uint64_t>(pair) * p.n);
    for (uint32_t i = lane; i < p.n / 4; i += 64) v[i] = 0;
    for (uint32_t i = lane; i < p.n / kMxGroup; i += 64) p.scales[static_cast<uint64_t>(pair) * (p.n / kMxGroup) + i] = 0;
  } else {
    for (uint32_t i = lane; i < p.n; i += 64) p.out[static_cast<uint64_t>(pair) * p.n + i] = 0;
  }
}

// One wave zeroes the output rows among routed rows first .. +kZeroRows whose id names no expert.
template <int OUT>
__device__ void zero_rows(const ProductLaunch& p, uint32_t first, uint32_t lane) {
  const uint32_t i = first + lane;
  const bool none = i < p.rows && static_cast<uint32_t>(p.ids[i]) >= p.experts;
  uint64_t left = __ballot(none);
  while (left != 0) {
    const uint32_t j = static_cast<uint32_t>(__builtin_ctzll(left));
    left &= left - 1;
    zero_row<OUT>(p, first + j, lane);
  }
}

// ---------------------------------------------------------------- stream ---

// One row of 16 lanes' addresses: unit `u` of chunk `c`, or zeros at and behind the row's end.
__device__ __forceinline__ const uint8_t* unit_at(const uint8_t* row, uint32_t c, uint32_t u, uint32_t k_bytes) {
  const uint32_t at = c * kChunk + u * 16u;
  return at < k_bytes ? row + at : reinterpret_cast<const uint8_t*>(g_product_zeros);
}

// The operands of one chunk and strip.
template <bool MX, bool WHOLE>
struct StreamChunk {
  uint4 w[kStrip][2], x[2];
  uint32_t ws[kStrip], xs;

  __device__ __forceinline__ void load(const uint8_t* const w_row[kStrip], const uint8_t* const ws_row[kStrip],
                                       const uint8_t* x_row, const uint8_t* xs_row, uint32_t c, uint32_t kb,
                                       uint32_t k_bytes) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      x[h] = ldg16(unit_at(x_row, c, 4 * h + kb, k_bytes));
#pragma unroll
      for (int f = 0; f < kStrip; ++f) w[f][h] = ldg16(unit_at(w_row[f], c, 4 * h + kb, k_bytes));
    }
    if constexpr (MX) {
      // chunks behind the last one have zero values under any scale
      const uint32_t groups = k_bytes / kMxGroup, at = WHOLE ? min(c, groups / 4u - 1u) : c;
      xs = chunk_scales<WHOLE>(xs_row, at, groups);
#pragma unroll
      for (int f = 0; f < kStrip; ++f) ws[f] = chunk_scales<WHOLE>(ws_row[f], at, groups);
    }
  }
  __device__ __forceinline__ void mfma(f32x4_t acc[kStrip], uint32_t kb) const {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const Operand<MX> xo(x[h], MX ? unit_scale(xs, kb, h) : 1.0f);
#pragma unroll
      for (int f = 0; f < kStrip; ++f)
        acc[f] = unit_mfma(Operand<MX>(w[f][h], MX ? unit_scale(ws[f], kb, h) : 1.0f), xo, acc[f]);
    }
  }
};

// KS waves of a block split a strip's chunks between them and add up in LDS (4), or each wave has a strip of its own
// (1).  SORTED: tiles of up to 16 sorted rows; else one routed row per block.  WHOLE: K is whole chunks and scales are
// aligned to their four bytes.
template <bool MX, bool SWIGLU, int OUT, int KS, bool SORTED, bool WHOLE>
__global__ __launch_bounds__(256) void k_stream(ProductLaunch p) {
  constexpr int kWaves = 4, kDepth = 2;
  const uint32_t tid = threadIdx.x, lane = tid & 63u, lm = lane & 15u, kb = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  constexpr uint32_t kCols = strip_cols<SWIGLU>() * (kWaves / KS);
  const uint32_t slices = (p.n + kCols - 1) / kCols;
  uint32_t expert, pair, rows = 1, slice;
  if constexpr (SORTED) {
    // each XCD takes a contiguous run of the tiles with all their slices: its L2 serves a tile's rows to every slice
    const uint32_t lin = blockIdx.x, local = (lin >> 3) / slices;
    slice = (lin >> 3) % slices;
    const uint32_t count = *p.tile_count, chunk = (count + 7) / 8;
    const uint32_t tile = (lin & 7u) * chunk + local;
    if (lin >= p.tile_blocks) {
      zero_rows<OUT>(p, ((lin - p.tile_blocks) * kWaves + wave) * kZeroRows, lane);
      return;
    }
    if (local >= chunk || tile >= count) return;
    const uint2 td = p.tiles[tile];
    expert = td.x;
    const uint32_t row0 = p.row_off[expert] + td.y;
    rows = min(p.row_off[expert + 1] - row0, kStreamRows);
    pair = p.row_pair[row0 + min(lm, rows - 1)];
  } else {
    pair = blockIdx.x / slices;
    slice = blockIdx.x % slices;
    expert = static_cast<uint32_t>(p.ids[pair]);
    if (expert >= p.experts) {
      if (slice == 0 && wave == 0) zero_row<OUT>(p, pair, lane);
      return;
    }
  }
  const uint32_t col = slice * kCols + (KS == 1 ? wave * strip_cols<SWIGLU>() : 0u);
  const uint32_t x_row_id = pair / p.x_div;
  const uint8_t* x_row = p.x + static_cast<uint64_t>(x_row_id) * p.x_stride;
  const uint8_t* xs_row = MX ? p.x_scales + static_cast<uint64_t>(x_row_id) * p.x_scale_stride : nullptr;
  const uint8_t* w_row[kStrip];
  const uint8_t* ws_row[kStrip];
#pragma unroll
  for (int f = 0; f < kStrip; ++f) {
    const uint64_t r = matrix_row<SWIGLU>(col, f * 16u + lm, p.n);
    w_row[f] = p.w + expert * p.w_expert + r * p.w_stride;
    ws_row[f] = MX ? p.w_scales + expert * p.w_scale_expert + r * p.w_scale_stride : nullptr;
  }
  const uint32_t chunks = (p.k_bytes + kChunk - 1) / kChunk;
  const uint32_t first = KS == 1 ? 0u : wave;
  const uint32_t count = chunks > first ? (chunks - first + KS - 1) / KS : 0u;
  f32x4_t acc[kStrip];
#pragma unroll
  for (int f = 0; f < kStrip; ++f) acc[f] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  // chunks behind the last one load zeros, so no load of the pipeline is conditional
  StreamChunk<MX, WHOLE> buf[kDepth];
#pragma unroll
  for (int j = 0; j < kDepth; ++j) buf[j].load(w_row, ws_row, x_row, xs_row, first + j * KS, kb, p.k_bytes);
  for (uint32_t i = 0; i < count; i += kDepth) {
#pragma unroll
    for (int j = 0; j < kDepth; ++j) {
      buf[j].mfma(acc, kb);
      buf[j].load(w_row, ws_row, x_row, xs_row, first + (i + j + kDepth) * KS, kb, p.k_bytes);
    }
  }
  if constexpr (KS > 1) {
    __shared__ f32x4_t s_acc[KS - 1][kStrip][64];
    if (wave != 0) {
#pragma unroll
      for (int f = 0; f < kStrip; ++f) s_acc[wave - 1][f][lane] = acc[f];
    }
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int w = 0; w < KS - 1; ++w)
#pragma unroll
      for (int f = 0; f < kStrip; ++f) acc[f] += s_acc[w][f][lane];
  }
  if (col >= p.n) return;
  store_strip<SWIGLU, OUT>(p, acc, col, pair, lm < rows, kb);
}

// ----------------------------------------------------------------- tiles ---

constexpr uint32_t kTileCols = 128;       // matrix rows per block

// Unit u of row r lies at unit u ^ swz(r) of its 128 bytes: an operand read (lane: row lane % 16, unit lane / 16 or
// 4 + lane / 16) then spreads over all 64 banks in every lane grouping of the read.
__device__ __forceinline__ uint32_t tile_swz(uint32_t r) { return ((r >> 1) & 2u) | ((r << 1) & 4u); }

// Stage J: the tile's rows, then the matrix rows, 128 bytes each; and the four scale bytes of each.  One LDS object
// per stage, so that the compiler can tell the stage being read from the one being filled.
template <int J, int BM>
__device__ __forceinline__ uint8_t* tile_stage() {
  __shared__ uint4 buf[(BM + kTileCols) * kChunk / 16];
  return reinterpret_cast<uint8_t*>(buf);
}
template <int J, int BM>
__device__ __forceinline__ uint32_t* tile_scales() {
  __shared__ uint32_t buf[BM + kTileCols];
  return buf;
}

// s_waitcnt for the vector memory count or the LDS count at zero, the others left alone
__device__ __forceinline__ void wait_vm0() { __builtin_amdgcn_s_waitcnt((7 << 4) | (15 << 8)); }
__device__ __forceinline__ void wait_lgkm0() { __builtin_amdgcn_s_waitcnt(15 | (3 << 14) | (7 << 4)); }

// A block barrier that no memory access is moved across and that waits for none by itself.
__device__ __forceinline__ void bare_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// BM rows by 128 matrix rows; four waves of BM / 2 rows by 64 matrix rows each.  WHOLE: K is whole chunks.
template <bool MX, bool SWIGLU, int OUT, int BM, bool WHOLE>
__global__ __launch_bounds__(256) void k_tiles(ProductLaunch p) {
  constexpr int kWaves = 4;
  constexpr int kRowFrags = BM / 32;               // 16-row fragments per wave
  constexpr int kDmaX = BM / 8 / kWaves;           // 1 KB loads (eight rows) per wave and chunk
  constexpr int kDmaW = kTileCols / 8 / kWaves;
  constexpr uint32_t kCols = strip_cols<SWIGLU>() * (kTileCols / 64);
  const uint32_t tid = threadIdx.x, lane = tid & 63u, lm = lane & 15u, kb = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t slices = (p.n + kCols - 1) / kCols;
  const uint32_t lin = blockIdx.x, local = (lin >> 3) / slices, slice = (lin >> 3) % slices;
  const uint32_t count = *p.tile_count, run = (count + 7) / 8;
  const uint32_t tile = (lin & 7u) * run + local;
  if (lin >= p.tile_blocks) {
    zero_rows<OUT>(p, ((lin - p.tile_blocks) * kWaves + wave) * kZeroRows, lane);
    return;
  }
  if (local >= run || tile >= count) return;
  const uint2 td = p.tiles[tile];
  const uint32_t expert = td.x;
  const uint32_t row0 = p.row_off[expert] + td.y;
  const uint32_t rows = min(p.row_off[expert + 1] - row0, static_cast<uint32_t>(BM));
  const uint32_t col0 = slice * kCols;
  const uint8_t* w = p.w + expert * p.w_expert;

  // DMA: load i of a wave fills eight rows; lane j loads unit (j % 8) ^ swz(row) of row j / 8 into bytes 16 j, so the
  // swizzle costs nothing.  Rows behind the tile's last one load it again.
  const uint32_t sub = lane / 8u, unit = (lane % 8u);
  const uint8_t* src[kDmaX + kDmaW];
  uint32_t at[kDmaX + kDmaW];   // byte of the lane's unit in a chunk
#pragma unroll
  for (int i = 0; i < kDmaX; ++i) {
    const uint32_t r = (wave * kDmaX + i) * 8u + sub;
    const uint32_t pair = p.row_pair[row0 + min(r, rows - 1)];
    at[i] = (unit ^ tile_swz(r)) * 16u;
    src[i] = p.x + static_cast<uint64_t>(pair / p.x_div) * p.x_stride + at[i];
  }
#pragma unroll
  for (int i = 0; i < kDmaW; ++i) {
    const uint32_t r = (wave * kDmaW + i) * 8u + sub;
    const uint32_t n = matrix_row<SWIGLU>(col0 + (r >> 6) * strip_cols<SWIGLU>(), r & 63u, p.n);
    at[kDmaX + i] = (unit ^ tile_swz(r)) * 16u;
    src[kDmaX + i] = w + n * p.w_stride + at[kDmaX + i];
  }
  // scales: thread t serves row t of the stage
  const uint8_t* scale_row = nullptr;
  if constexpr (MX) {
    if (tid < BM) {
      const uint32_t pair = p.row_pair[row0 + min(tid, rows - 1)];
      scale_row = p.x_scales + static_cast<uint64_t>(pair / p.x_div) * p.x_scale_stride;
    } else if (tid < BM + kTileCols) {
      const uint32_t r = tid - BM;
      const uint32_t n = matrix_row<SWIGLU>(col0 + (r >> 6) * strip_cols<SWIGLU>(), r & 63u, p.n);
      scale_row = p.w_scales + expert * p.w_scale_expert + n * p.w_scale_stride;
    }
  }
  const uint32_t chunks = (p.k_bytes + kChunk - 1) / kChunk, groups = p.k_bytes / kMxGroup;
  auto issue = [&](auto J, uint32_t c) {
    uint8_t* st = tile_stage<decltype(J)::value, BM>();
#pragma unroll
    for (int i = 0; i < kDmaX + kDmaW; ++i) {
      const uint32_t g = i < kDmaX ? wave * kDmaX + i : BM / 8 + wave * kDmaW + (i - kDmaX);
      const uint8_t* s = src[i] + c * kChunk;
      if constexpr (!WHOLE)
        if (c * kChunk + at[i] >= p.k_bytes) s = reinterpret_cast<const uint8_t*>(g_product_zeros);
      __builtin_amdgcn_global_load_lds(s, (__attribute__((address_space(3))) void*)(st + g * 1024u), 16, 0, 0);
    }
  };
  auto scales_of = [&](uint32_t c) -> uint32_t {
    return scale_row != nullptr ? chunk_scales<WHOLE>(scale_row, c, groups) : 0u;
  };
  auto keep_scales = [&](auto J, uint32_t v) {
    if (tid < BM + kTileCols) tile_scales<decltype(J)::value, BM>()[tid] = v;
  };

  const uint32_t wm = wave & 1u, wn = wave >> 1;
  const uint32_t s = tile_swz(lm);
  const uint32_t u0 = (kb ^ s) * 16u, u1 = ((4u | kb) ^ s) * 16u;
  const uint32_t x_base = (wm * (BM / 2) + lm) * kChunk, w_base = (BM + wn * 64u + lm) * kChunk;
  f32x4_t acc[kRowFrags][kStrip];
#pragma unroll
  for (int i = 0; i < kRowFrags; ++i)
#pragma unroll
    for (int f = 0; f < kStrip; ++f) acc[i][f] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  auto compute = [&](auto J) {
    const uint8_t* st = tile_stage<decltype(J)::value, BM>();
    uint32_t xs[kRowFrags], ws[kStrip];
    if constexpr (MX) {
      const uint32_t* sc = tile_scales<decltype(J)::value, BM>();
#pragma unroll
      for (int f = 0; f < kStrip; ++f) ws[f] = sc[BM + wn * 64 + f * 16 + lm];
#pragma unroll
      for (int i = 0; i < kRowFrags; ++i) xs[i] = sc[wm * (BM / 2) + i * 16 + lm];
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t u = h ? u1 : u0;
      uint4 xv[kRowFrags], wv[kStrip];
#pragma unroll
      for (int f = 0; f < kStrip; ++f) wv[f] = *reinterpret_cast<const uint4*>(st + w_base + f * 16 * kChunk + u);
#pragma unroll
      for (int i = 0; i < kRowFrags; ++i) xv[i] = *reinterpret_cast<const uint4*>(st + x_base + i * 16 * kChunk + u);
#pragma unroll
      for (int f = 0; f < kStrip; ++f) {
        const Operand<MX> wo(wv[f], MX ? unit_scale(ws[f], kb, h) : 1.0f);
#pragma unroll
        for (int i = 0; i < kRowFrags; ++i)
          acc[i][f] = unit_mfma(wo, Operand<MX>(xv[i], MX ? unit_scale(xs[i], kb, h) : 1.0f), acc[i][f]);
      }
    }
  };

  using J0 = std::integral_constant<int, 0>;
  using J1 = std::integral_constant<int, 1>;
  auto step = [&](auto J, auto JN, uint32_t c) {
    uint32_t v = 0;
    if (c + 1 < chunks) {
      issue(JN, c + 1);
      if constexpr (MX) v = scales_of(c + 1);
    }
    compute(J);
    wait_vm0();    // the next stage has landed; it was loaded for as long as this one was multiplied
    if constexpr (MX) keep_scales(JN, v);
    wait_lgkm0();  // this wave's reads and writes are done before the barrier
    bare_barrier();
  };
  issue(J0{}, 0);
  if constexpr (MX) keep_scales(J0{}, scales_of(0));
  wait_vm0();
  wait_lgkm0();
  bare_barrier();
  for (uint32_t c = 0; c < chunks; c += 2) {
    step(J0{}, J1{}, c);
    if (c + 1 < chunks) step(J1{}, J0{}, c + 1);
  }

  const uint32_t col = col0 + wn * strip_cols<SWIGLU>();
  if (col >= p.n) return;
#pragma unroll
  for (int i = 0; i < kRowFrags; ++i) {
    const uint32_t r = wm * (BM / 2) + i * 16u + lm;
    const uint32_t pair = p.row_pair[row0 + min(r, rows - 1)];
    store_strip<SWIGLU, OUT>(p, acc[i], col, pair, r < rows, kb);
  }
}

// -------------------------------------------------------------- dispatch ---

template <class Kernel>
hipError_t go(Kernel kernel, uint32_t blocks, const ProductLaunch& p, hipStream_t stream) {
  hipEvent_t start = nullptr, stop = nullptr;
  if (timing_events("products", &start, &stop))
    hipExtLaunchKernelGGL(kernel, dim3(blocks), dim3(256), 0, stream, start, stop, 0, p);
  else
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(256), 0, stream, p);
  return hipGetLastError();
}

// Every row of scales starts at a multiple of four bytes, the scales of one chunk.
bool scales_aligned(const ProductLaunch& p) {
  return (reinterpret_cast<uintptr_t>(p.x_scales) | reinterpret_cast<uintptr_t>(p.w_scales) | p.x_scale_stride |
          p.w_scale_stride | p.w_scale_expert) % 4 == 0;
}

template <bool MX, bool SWIGLU, int OUT>
hipError_t products_go(ProductLaunch p, uint32_t tile_rows, hipStream_t stream) {
  const uint32_t chunks = (p.k_bytes + kChunk - 1) / kChunk;
  const bool split = chunks >= 16;  // a wave of a split strip then has at least four chunks
  const bool whole = p.k_bytes % kChunk == 0 && (!MX || scales_aligned(p));
  const auto stream_go = [&](auto sorted, uint32_t units, uint32_t more) {
    constexpr bool kSorted = decltype(sorted)::value;
    const uint32_t cols = strip_cols<SWIGLU>() * (split ? 1u : 4u);
    p.tile_blocks = (p.n + cols - 1) / cols * units;
    const uint32_t blocks = p.tile_blocks + more;
    // bf16 loads check the row's end in either case
    if (MX && whole)
      return split ? go(&k_stream<MX, SWIGLU, OUT, 4, kSorted, MX>, blocks, p, stream)
                   : go(&k_stream<MX, SWIGLU, OUT, 1, kSorted, MX>, blocks, p, stream);
    return split ? go(&k_stream<MX, SWIGLU, OUT, 4, kSorted, false>, blocks, p, stream)
                 : go(&k_stream<MX, SWIGLU, OUT, 1, kSorted, false>, blocks, p, stream);
  };
  if (tile_rows == 0) return stream_go(std::false_type{}, p.rows, 0);
  const uint32_t tiles = (grouped_max_tiles(p.rows, p.experts, tile_rows) + 7) / 8 * 8;
  const uint32_t zero = (p.rows + 4 * kZeroRows - 1) / (4 * kZeroRows);
  if (tile_rows == kStreamRows) return stream_go(std::true_type{}, tiles, zero);
  const uint32_t cols = strip_cols<SWIGLU>() * 2u;
  p.tile_blocks = (p.n + cols - 1) / cols * tiles;
  if (tile_rows == 64)
    return whole ? go(&k_tiles<MX, SWIGLU, OUT, 64, true>, p.tile_blocks + zero, p, stream)
                 : go(&k_tiles<MX, SWIGLU, OUT, 64, false>, p.tile_blocks + zero, p, stream);
  return whole ? go(&k_tiles<MX, SWIGLU, OUT, 128, true>, p.tile_blocks + zero, p, stream)
               : go(&k_tiles<MX, SWIGLU, OUT, 128, false>, p.tile_blocks + zero, p, stream);
}

}  // namespace

uint32_t product_tile_rows(uint32_t rows, uint32_t experts) {
  if (rows <= 32) return 0;
  const uint32_t mean = rows / experts;
  return mean < 12 ? kStreamRows : mean < 96 ? 64u : 128u;
}

uint64_t product_blocks(uint32_t rows, uint32_t experts, uint32_t n, uint32_t tile_rows, bool swiglu) {
  const uint64_t strips = (uint64_t(n) + (swiglu ? 31 : 63)) / (swiglu ? 32 : 64);
  const uint64_t units = tile_rows == 0 ? rows : (uint64_t(rows) + tile_rows - 1) / tile_rows + experts + 7;
  return units * strips + rows / (4 * kZeroRows) + 1;
}

hipError_t launch_products(const ProductLaunch& p, uint32_t tile_rows, hipStream_t stream) {
  if (p.values != nullptr && !p.swiglu) return hipErrorInvalidValue;
  if (p.mx) {
    if (!p.swiglu) return products_go<true, false, kOutBf16>(p, tile_rows, stream);
    return p.values != nullptr ? products_go<true, true, kOutMx>(p, tile_rows, stream)
                               : products_go<true, true, kOutBf16>(p, tile_rows, stream);
  }
  if (!p.swiglu) return products_go<false, false, kOutBf16>(p, tile_rows, stream);
  return p.values != nullptr ? products_go<false, true, kOutMx>(p, tile_rows, stream)
                             : products_go<false, true, kOutBf16>(p, tile_rows, stream);
}

}  // namespace vm
