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
// The matrix is the first operand, the rows the second, so a lane receives outputs of row lane % 16.
//
// With hundreds of experts the weights are most of the bytes, each read for a few to a few hundred rows.  Two forms:
//   k_rows    calls of few routed rows: no sort, one launch; a block per routed row and a few dozen matrix rows, each
//             read a kilobyte at a time by one wave and multiplied by v_dot2.
//   k_tiles   tiles of up to 32 or 64 rows sorted by expert by 128 or 256 matrix rows, both staged in LDS by DMA.
// MFMA operands loaded straight from memory (16 rows of 64 bytes per load) are limited to 16 bytes per clock and CU,
// the L1's rate for lanes of different rows; the DMA's eight rows of 128 bytes reach 55 (measured).
// Rows whose id names no expert are written as zeros by blocks behind the tiles'.
//
// Bound by the matrices' bytes: one token, ten of 512 experts, bf16 2048 -> 2 x 512, 10.8 us (42 MB); 2048 tokens MX 2560
// -> 2 x 640 347 us behind a sort of 13 (1.7 GB, 5.0 TB/s; a copy reaches 4.7); 8192 tokens bf16 605 behind 14: 2.1 GB of
// matrices, 3.1 GB past the L2 since an expert's two or three tiles do not all meet its matrix there, 5.2 TB/s.

#include <hip/hip_ext.h>
#include <hip/hip_runtime.h>

#include <type_traits>

#include "vm_dma.h"
#include "vm_internal.h"
#include "vm_mx.h"
#include "vm_rows.h"

namespace vm {

namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

constexpr int kStrip = 4;                 // 16-row fragments of the matrix per wave
constexpr uint32_t kZeroRows = 8;         // routed rows checked per wave of the zeroing blocks

enum : int { kOutBf16 = 0, kOutMx = 1 };

__device__ uint4 g_product_zeros[kChunk / 16];  // units at and behind the end of a row load from here

// One lane's MFMA operands of a 16-byte unit: itself, or two of bf16 values, e4m3 ones times the power of two whose
// exponent bits `scale` holds (0: 2^-127, 255: NaN).
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

// Matrix row behind row `r` (0..63) of a wave's strip that starts at output column `col`.  Row 4 q + i of fragment f
// becomes output i of lane group q, so the fragments are dealt to give a lane neighbouring outputs over all of them:
// 16 of the strip's 64, or with SwiGLU 8 of its 32, where fragments alternate between gate rows and up rows.
template <bool SWIGLU>
__device__ __forceinline__ uint32_t matrix_row(uint32_t col, uint32_t r, uint32_t n) {
  const uint32_t f = r >> 4, q = (r >> 2) & 3u, i = r & 3u;
  if constexpr (SWIGLU) return min(col + 8u * q + 4u * (f >> 1) + i, n - 1u) + (f & 1u) * n;
  else return min(col + 16u * q + 4u * f + i, n - 1u);
}

// Outputs per strip.
template <bool SWIGLU>
constexpr uint32_t strip_cols() {
  return SWIGLU ? 32u : 64u;
}

// silu(g) * u with the hardware exp2 and reciprocal, off by 16 + 2 |g| half steps of fp32 at most (|g| of them from the
// rounding of exp2's argument).  A negative gate's exponential comes as its root on either factor, h g and h u, so that
// neither it nor the reciprocal, of 1 to 2, is subnormal, which the hardware flushes: from the product's own range on
// down to gates of -174, where |silu| is 2^-244, the result keeps its bits however large u is.
__device__ __forceinline__ float swiglu(float g, float u) {
  const float h = __builtin_amdgcn_exp2f(fabsf(g) * -0x1.715476p-1f);   // e^(-|g| / 2)
  const float r = __builtin_amdgcn_rcpf(fmaf(h, h, 1.0f));
  const float w = g < 0.0f ? h : 1.0f;
  return g * w * r * (w * u);
}

// Stores one strip of one 16-row fragment: a lane holds 16 (SwiGLU: 8) neighbouring outputs of its routed row.
template <bool SWIGLU, int OUT>
__device__ __forceinline__ void store_strip(const ProductLaunch& p, const f32x4_t acc[kStrip], uint32_t col,
                                            uint32_t pair, bool live, uint32_t kb) {
  constexpr uint32_t kOut = SWIGLU ? 8 : 16;
  float y[kOut];
#pragma unroll
  for (uint32_t j = 0; j < kOut; ++j)
    y[j] = SWIGLU ? swiglu(acc[2 * (j / 4)][j % 4], acc[2 * (j / 4) + 1][j % 4]) : acc[j / 4][j % 4];
  const uint32_t at = col + kOut * kb;
  const uint64_t row = static_cast<uint64_t>(pair) * p.n;
  if constexpr (OUT == kOutMx) {
    static_assert(SWIGLU, "a strip of SwiGLU outputs is one group");
    uint32_t m = 0;
#pragma unroll
    for (uint32_t j = 0; j < kOut; ++j) m = max(m, mx_magnitude(y[j]));
    m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), 16)));
    m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), 32)));
    const uint32_t e = mx_scale(m);
    if (!live) return;
    *reinterpret_cast<uint2*>(p.values + row + at) =
        make_uint2(mx_pack4(y[0], y[1], y[2], y[3], e), mx_pack4(y[4], y[5], y[6], y[7], e));
    if (kb == 0) p.scales[(row + col) / kMxGroup] = static_cast<uint8_t>(e);
  } else {
    if (!live) return;
    if (p.n % 8 == 0 && p.out_aligned) {
#pragma unroll
      for (uint32_t j = 0; j < kOut; j += 8) {
        uint32_t w[4];
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) w[i] = f32_to_bf16(y[j + 2 * i]) | (f32_to_bf16(y[j + 2 * i + 1]) << 16);
        if (at + j < p.n) *reinterpret_cast<uint4*>(p.out + row + at + j) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    } else {
#pragma unroll
      for (uint32_t j = 0; j < kOut; ++j)
        if (at + j < p.n) p.out[row + at + j] = static_cast<uint16_t>(f32_to_bf16(y[j]));
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
  const bool none = lane < kZeroRows && i < p.rows && static_cast<uint32_t>(p.ids[i]) >= p.experts;
  uint64_t left = __ballot(none);
  while (left != 0) {
    const uint32_t j = static_cast<uint32_t>(__builtin_ctzll(left));
    left &= left - 1;
    zero_row<OUT>(p, first + j, lane);
  }
}

// ------------------------------------------------------------------ rows ---

constexpr int kRowBatch = 8;              // matrix rows a wave sums at once
constexpr uint32_t kRowStep = 64 * 16;    // bytes of a row per step of a wave

// Eight (bf16) or sixteen (MX) products of a lane's unit, fp32 sums.
template <bool MX>
__device__ __forceinline__ float unit_dot(const Operand<MX>& w, const Operand<MX>& x, float acc) {
#pragma unroll
  for (int i = 0; i < (MX ? 2 : 1); ++i) {
    const uint32_t a[4] = {w.part[i].x, w.part[i].y, w.part[i].z, w.part[i].w};
    const uint32_t b[4] = {x.part[i].x, x.part[i].y, x.part[i].z, x.part[i].w};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      acc = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, a[j]), __builtin_bit_cast(bf16x2, b[j]), acc, false);
  }
  return acc;
}

__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }

// One routed row per block and 8 WAVES matrix rows, eight per wave: a wave reads a kilobyte of one matrix row at a
// time, the row's unit of the lane stays in registers for all eight.
template <bool MX, bool SWIGLU, int OUT, int WAVES, bool ONCE>
__global__ __launch_bounds__(64 * WAVES) void k_rows(ProductLaunch p) {
  constexpr uint32_t kMatrix = kRowBatch * WAVES, kCols = SWIGLU ? kMatrix / 2 : kMatrix;
  static_assert(OUT == kOutBf16 || kCols == kMxGroup, "a block's outputs are one group");
  __shared__ float s_y[kMatrix];
  const uint32_t tid = threadIdx.x, lane = tid & 63u;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t slices = (p.n + kCols - 1) / kCols;
  const uint32_t pair = blockIdx.x / slices, col0 = blockIdx.x % slices * kCols;
  const uint32_t expert = static_cast<uint32_t>(p.ids[pair]);
  if (expert >= p.experts) {
    if (col0 == 0 && wave == 0) zero_row<OUT>(p, pair, lane);
    return;
  }
  const uint8_t* x_row = p.x + static_cast<uint64_t>(pair / p.x_div) * p.x_stride;
  const uint8_t* xs_row = MX ? p.x_scales + static_cast<uint64_t>(pair / p.x_div) * p.x_scale_stride : nullptr;
  const uint8_t *w_row[kRowBatch], *ws_row[kRowBatch];
#pragma unroll
  for (int j = 0; j < kRowBatch; ++j) {
    // with SwiGLU rows 2 j and 2 j + 1 of the block are gate and up of its output j
    const uint32_t r = wave * kRowBatch + j;
    const uint64_t m = SWIGLU ? min(col0 + r / 2, p.n - 1) + (r & 1u) * p.n : min(col0 + r, p.n - 1);
    w_row[j] = p.w + expert * p.w_expert + m * p.w_stride;
    ws_row[j] = MX ? p.w_scales + expert * p.w_scale_expert + m * p.w_scale_stride : nullptr;
  }
  float acc[kRowBatch] = {};
  uint4 xv, wv[kRowBatch];
  uint32_t xs = 0, ws[kRowBatch] = {};
  const uint8_t* zeros = reinterpret_cast<const uint8_t*>(g_product_zeros);
  VM_KEEP(zeros);
  auto load = [&](uint32_t at) {
    const bool in = at < p.k_bytes;
    xv = ldg16(in ? x_row + at : zeros);
#pragma unroll
    for (int j = 0; j < kRowBatch; ++j) {
      const uint8_t* from = in ? w_row[j] + at : zeros;
      wv[j] = ONCE ? ldg16_nt(from) : ldg16(from);
    }
    if constexpr (MX) {
      const uint32_t g = min(at, p.k_bytes - 1) / kMxGroup;
      xs = xs_row[g];
#pragma unroll
      for (int j = 0; j < kRowBatch; ++j) ws[j] = ws_row[j][g];
    }
  };
  load(lane * 16u);
  for (uint32_t at = lane * 16u; at - lane * 16u < p.k_bytes; at += kRowStep) {
    const Operand<MX> x(xv, scale_of(xs));
    uint4 now[kRowBatch];
    uint32_t scale[kRowBatch];
#pragma unroll
    for (int j = 0; j < kRowBatch; ++j) {
      now[j] = wv[j];
      scale[j] = ws[j];
    }
    load(at + kRowStep);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < kRowBatch; ++j) acc[j] = unit_dot(Operand<MX>(now[j], scale_of(scale[j])), x, acc[j]);
  }
#pragma unroll
  for (int j = 0; j < kRowBatch; ++j) {
    const float y = group_sum<64>(acc[j]);
    if (lane == 63) s_y[wave * kRowBatch + j] = y;
  }
  __syncthreads();
  if (tid >= kCols) return;
  const float y = SWIGLU ? swiglu(s_y[2 * tid], s_y[2 * tid + 1]) : s_y[tid];
  const uint64_t at = static_cast<uint64_t>(pair) * p.n + col0 + tid;
  if constexpr (OUT == kOutMx) {
    uint32_t m = mx_magnitude(y);
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), d)));
    const uint32_t e = mx_scale(m);
    p.values[at] = static_cast<uint8_t>(mx_pack4(y, y, y, y, e));
    if (tid == 0) p.scales[at / kMxGroup] = static_cast<uint8_t>(e);
  } else if (col0 + tid < p.n) {
    p.out[at] = static_cast<uint16_t>(f32_to_bf16(y));
  }
}

// ----------------------------------------------------------------- tiles ---

// Stage J: the tile's rows, then the matrix rows, 128 bytes each.  One LDS object per stage, so that the compiler can
// tell the stage being read from the one being filled.
template <int J, int ROWS>
__device__ __forceinline__ uint8_t* tile_stage() {
  __shared__ uint4 buf[ROWS * kChunk / 16];
  return reinterpret_cast<uint8_t*>(buf);
}

// WM x WN waves of 16 RF rows by 64 matrix rows each.  WHOLE: K is whole chunks and scales are aligned.
template <bool MX, bool SWIGLU, int OUT, int RF, int WM, int WN, bool WHOLE>
__global__ __launch_bounds__(64 * WM * WN, 2) void k_tiles(ProductLaunch p) {
  constexpr int kWaves = WM * WN;
  constexpr uint32_t kRows = 16 * RF * WM, kMatrix = 64 * WN;
  constexpr int kDmaX = kRows / 8 / kWaves;           // 1 KB loads (eight rows) per wave and chunk
  constexpr int kDmaW = kMatrix / 8 / kWaves;
  static_assert(kDmaX * 8 * kWaves == kRows && kDmaW * 8 * kWaves == kMatrix, "whole loads per wave");
  constexpr uint32_t kCols = strip_cols<SWIGLU>() * WN;
  const uint32_t tid = threadIdx.x, lane = tid & 63u, lm = lane & 15u, kb = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t slices = (p.n + kCols - 1) / kCols;
  const uint32_t lin = blockIdx.x, local = (lin >> 3) / slices, slice = (lin >> 3) % slices;
  if (lin >= p.tile_blocks) {
    zero_rows<OUT>(p, ((lin - p.tile_blocks) * kWaves + wave) * kZeroRows, lane);
    return;
  }
  BlockTile td;
  if (p.tiles != nullptr) {
    if (!listed_tile(p.tiles, p.tile_count, p.row_pair, lin & 7u, local, &td)) return;
  } else {
    uint32_t* words = reinterpret_cast<uint32_t*>(tile_stage<0, kRows + kMatrix>());
    static_assert(kFindWords * 4 <= (kRows + kMatrix) * kChunk, "a stage holds find_tile's words");
    if (!find_tile<64 * kWaves, kRows>(p.ids, p.rows, p.experts, lin & 7u, local, words, &td)) return;
  }
  const uint32_t expert = td.group, rows = td.rows;
  const auto row_of = [&](uint32_t r) { return static_cast<uint32_t>(__shfl(static_cast<int>(td.row), r)); };
  const uint32_t col0 = slice * kCols;
  const uint8_t* w = p.w + expert * p.w_expert;
  const auto matrix_at = [&](uint32_t r) {   // matrix row of the block's row r
    return matrix_row<SWIGLU>(col0 + (r >> 6) * strip_cols<SWIGLU>(), r & 63u, p.n);
  };

  // DMA: load i of a wave fills eight rows; lane j loads unit (j % 8) ^ swz(row) of row j / 8 into bytes 16 j, so the
  // swizzle costs nothing.  Rows behind the tile's last one load it again.
  const uint32_t sub = lane / 8u, unit = (lane % 8u);
  const uint8_t* src[kDmaX + kDmaW];
  const uint32_t at = (unit ^ tile_swz(sub)) * 16u;   // byte of the lane's unit in a chunk, of rows sub, 8 + sub, ..
#pragma unroll
  for (int i = 0; i < kDmaX; ++i) {
    const uint32_t r = (wave * kDmaX + i) * 8u + sub;
    const uint32_t pair = row_of(r);
    src[i] = p.x + static_cast<uint64_t>(pair / p.x_div) * p.x_stride + at;
  }
#pragma unroll
  for (int i = 0; i < kDmaW; ++i) {
    const uint32_t r = (wave * kDmaW + i) * 8u + sub;
    src[kDmaX + i] = w + matrix_at(r) * p.w_stride + at;
  }
  const uint32_t wm = wave % WM, wn = wave / WM;
  // Scales: lane j holds the chunk's four bytes of the wave's row j and of its matrix row j; the lanes of a fragment
  // fetch theirs from there, so that the scales take no LDS (with a few KB of it one block less fits a CU).
  const uint8_t *xs_row = nullptr, *ws_row = nullptr;
  if constexpr (MX) {
    const uint32_t pair = row_of(min(wm * (16 * RF) + lane, 63u));
    xs_row = p.x_scales + static_cast<uint64_t>(pair / p.x_div) * p.x_scale_stride;
    ws_row = p.w_scales + expert * p.w_scale_expert + matrix_at(wn * 64u + lane) * p.w_scale_stride;
  }
  const uint32_t chunks = (p.k_bytes + kChunk - 1) / kChunk, groups = p.k_bytes / kMxGroup;
  const uint8_t* zeros = reinterpret_cast<const uint8_t*>(g_product_zeros);
  if constexpr (!WHOLE) VM_KEEP(zeros);
  const auto from = [&](int i, uint32_t c) {
    const uint8_t* s = src[i] + c * kChunk;
    if constexpr (!WHOLE)
      if (c * kChunk + at >= p.k_bytes) s = zeros;
    return s;
  };
  const bool once = p.once && td.group_rows <= kRows;
  auto issue = [&](auto J, uint32_t c) {
    uint8_t* st = tile_stage<decltype(J)::value, kRows + kMatrix>();
    uint8_t* st_w = st + kRows / 8 * 1024u + wave * kDmaW * 1024u;
#pragma unroll
    for (int i = 0; i < kDmaX; ++i) load_to_lds(from(i, c), st + (wave * kDmaX + i) * 1024u);
    if (once) {
#pragma unroll
      for (int i = 0; i < kDmaW; ++i) load_to_lds<true>(from(kDmaX + i, c), st_w + i * 1024u);
    } else {
#pragma unroll
      for (int i = 0; i < kDmaW; ++i) load_to_lds(from(kDmaX + i, c), st_w + i * 1024u);
    }
  };

  const uint32_t s = tile_swz(lm);
  const uint32_t u0 = (kb ^ s) * 16u, u1 = ((4u | kb) ^ s) * 16u;
  const uint32_t x_base = (wm * (16 * RF) + lm) * kChunk, w_base = (kRows + wn * 64u + lm) * kChunk;
  // 16-row fragments of this wave that hold rows of the tile
  const uint32_t live = rows > wm * (16 * RF) ? min((rows - wm * (16 * RF) + 15u) / 16u, static_cast<uint32_t>(RF)) : 0u;
  f32x4_t acc[RF][kStrip];
#pragma unroll
  for (int i = 0; i < RF; ++i)
#pragma unroll
    for (int f = 0; f < kStrip; ++f) acc[i][f] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  uint32_t held_x[2], held_w[2];   // the scale bytes of the stages
  // F fragments of stage J: all reads first, so that the second half's are under way while the first is multiplied
  auto compute = [&](auto J, auto frags) {
    constexpr int F = decltype(frags)::value;
    const uint8_t* st = tile_stage<decltype(J)::value, kRows + kMatrix>();
    uint32_t xs[F], ws[kStrip];
    uint4 xv[2][F], wv[2][kStrip];
    if constexpr (MX) {
      const auto from = [&](uint32_t j, uint32_t v) {
        return static_cast<uint32_t>(__builtin_amdgcn_ds_bpermute(static_cast<int>((j * 16u + lm) * 4u), static_cast<int>(v)));
      };
#pragma unroll
      for (uint32_t f = 0; f < kStrip; ++f) ws[f] = from(f, held_w[decltype(J)::value]);
#pragma unroll
      for (uint32_t i = 0; i < F; ++i) xs[i] = from(i, held_x[decltype(J)::value]);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t u = h ? u1 : u0;
#pragma unroll
      for (int f = 0; f < kStrip; ++f) wv[h][f] = *reinterpret_cast<const uint4*>(st + w_base + f * 16 * kChunk + u);
#pragma unroll
      for (int i = 0; i < F; ++i) xv[h][i] = *reinterpret_cast<const uint4*>(st + x_base + i * 16 * kChunk + u);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int f = 0; f < kStrip; ++f) {
        const Operand<MX> wo(wv[h][f], MX ? unit_scale(ws[f], kb, h) : 1.0f);
#pragma unroll
        for (int i = 0; i < F; ++i)
          acc[i][f] = unit_mfma(wo, Operand<MX>(xv[h][i], MX ? unit_scale(xs[i], kb, h) : 1.0f), acc[i][f]);
      }
  };

  // Two stages: one is multiplied while the next chunk is on its way to the other (behind the last chunk that one again,
  // which is not read).  More stages were slower than the second block per CU that their LDS costs.
  auto begin = [&](auto J, uint32_t c) {
    if constexpr (MX) {
      held_x[decltype(J)::value] = chunk_scales<WHOLE>(xs_row, c, groups);
      held_w[decltype(J)::value] = chunk_scales<WHOLE>(ws_row, c, groups);
    }
    __builtin_amdgcn_sched_barrier(0);
    issue(J, c);
    __builtin_amdgcn_sched_barrier(0);
  };
  begin(std::integral_constant<int, 0>{}, 0);
  for (uint32_t c = 0; c < chunks; c += 2) {
    unroll<0, 2>([&](auto J) {
      constexpr int j = decltype(J)::value;
      if (c + j >= chunks) return;
      wait_vm<0>();    // this wave's loads of the stage have landed
      wait_lgkm0();    // its reads of the other stage are done
      bare_barrier();
      begin(std::integral_constant<int, 1 - j>{}, min(c + j + 1, chunks - 1));
      if (live == RF) compute(J, std::integral_constant<int, RF>{});
      else if (RF > 3 && live == 3) compute(J, std::integral_constant<int, RF < 3 ? RF : 3>{});
      else if (RF > 2 && live == 2) compute(J, std::integral_constant<int, RF < 2 ? RF : 2>{});
      else if (live > 0) compute(J, std::integral_constant<int, 1>{});
      __builtin_amdgcn_sched_barrier(0);
    });
  }
  wait_vm<0>();  // no load into LDS outlives the block

  const uint32_t col = col0 + wn * strip_cols<SWIGLU>();
  if (col >= p.n) return;
#pragma unroll
  for (int i = 0; i < RF; ++i) {
    const uint32_t r = wm * (16 * RF) + i * 16u + lm;
    const uint32_t pair = row_of(r);
    store_strip<SWIGLU, OUT>(p, acc[i], col, pair, r < rows, kb);
  }
}

// -------------------------------------------------------------- dispatch ---

template <class Kernel>
hipError_t go(Kernel kernel, uint32_t blocks, uint32_t threads, const ProductLaunch& p, hipStream_t stream) {
  hipEvent_t start = nullptr, stop = nullptr;
  if (timing_events("products", &start, &stop))
    hipExtLaunchKernelGGL(kernel, dim3(blocks), dim3(threads), 0, stream, start, stop, 0, p);
  else
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(threads), 0, stream, p);
  return hipGetLastError();
}

// Every row of scales starts at a multiple of four bytes, the scales of one chunk.
bool scales_aligned(const ProductLaunch& p) {
  return (reinterpret_cast<uintptr_t>(p.x_scales) | reinterpret_cast<uintptr_t>(p.w_scales) | p.x_scale_stride |
          p.w_scale_stride | p.w_scale_expert) % 4 == 0;
}

template <bool MX, bool SWIGLU, int OUT>
hipError_t products_go(ProductLaunch p, uint32_t tile_rows, hipStream_t stream) {
  if (tile_rows == 0) {
    constexpr int kWaves = OUT == kOutMx ? 8 : 4;
    constexpr uint32_t cols = kRowBatch * kWaves / (SWIGLU ? 2 : 1);
    const uint32_t blocks = (p.n + cols - 1) / cols * p.rows;
    return p.once ? go(&k_rows<MX, SWIGLU, OUT, kWaves, true>, blocks, 64 * kWaves, p, stream)
                  : go(&k_rows<MX, SWIGLU, OUT, kWaves, false>, blocks, 64 * kWaves, p, stream);
  }
  const uint32_t tiles = (row_max_tiles(p.rows, p.experts, tile_rows) + 7) / 8 * 8;
  const bool whole = p.k_bytes % kChunk == 0 && (!MX || scales_aligned(p));
  const auto tiles_go = [&](auto rf, auto wm, auto wn) {
    constexpr int RF = decltype(rf)::value, WM = decltype(wm)::value, WN = decltype(wn)::value;
    constexpr uint32_t kWaves = WM * WN, cols = strip_cols<SWIGLU>() * WN;
    p.tile_blocks = (p.n + cols - 1) / cols * tiles;
    if (p.tiles == nullptr && p.rows > kFindRounds * 64 * kWaves) return hipErrorInvalidValue;
    const uint32_t blocks = p.tile_blocks + (p.rows + kWaves * kZeroRows - 1) / (kWaves * kZeroRows);
    return whole ? go(&k_tiles<MX, SWIGLU, OUT, RF, WM, WN, true>, blocks, 64 * kWaves, p, stream)
                 : go(&k_tiles<MX, SWIGLU, OUT, RF, WM, WN, false>, blocks, 64 * kWaves, p, stream);
  };
  using I1 = std::integral_constant<int, 1>;
  using I2 = std::integral_constant<int, 2>;
  using I4 = std::integral_constant<int, 4>;
  // 256 matrix rows per block read a tile's rows half as often as 128 and twice as many tile rows per wave reuse each
  // matrix operand, but fewer blocks run: once they fill the chip four times over, if the product of a few rows is not
  // a short one, too.  64-row tiles, 256 and 128: 2048 tokens MX 2560 -> 2 x 640, ten of 512 experts, 364 and 409 us,
  // 8192 tokens bf16 2048 -> 2 x 512 616 and 666; four of 64 experts, 8192 tokens, 1024 -> 2 x 256 62 and 60, four of
  // 20, 2048 tokens, 1024 -> 2 x 512 42 and 36.
  const uint32_t slices = (p.n + 4 * strip_cols<SWIGLU>() - 1) / (4 * strip_cols<SWIGLU>());
  const uint32_t chunks = (p.k_bytes + kChunk - 1) / kChunk;
  const bool wide = uint64_t(tiles) * slices >= 2048 && chunks * tile_rows >= 256;
  if (tile_rows == 32) return wide ? tiles_go(I2{}, I1{}, I4{}) : tiles_go(I2{}, I1{}, I2{});
  return wide ? tiles_go(I4{}, I1{}, I4{}) : tiles_go(I2{}, I2{}, I2{});
}

}  // namespace

// Every block of a call of few rows and experts finds its own tile: 333 tokens of four of 64 experts, 1024 -> 2 x 256,
// 15.5 us, behind a sort 19.3; 1000 tokens 19.9 and 22.5; of 20 experts, 2 x 512, 23.4 and 25.1.  Hundreds of experts mean
// thousands of blocks, which would all count: 32 tokens of ten of 512 experts MX 2560 -> 2 x 640 50.4 and 49.4, 200 of
// eight of 256 176 and 174.  Tiles of 32 rows mean less than 2048 rows then, which blocks of two waves can list.
bool product_sorted(uint32_t rows, uint32_t experts) { return rows > 4096 || experts > 128; }

// Rows up to which a call runs them one by one, if its tiles need a sort and if not.  An expert met twice is then read
// twice, which sixteen tokens of ten experts seldom do: 80 rows of 512 experts 58 us and 63 in sorted tiles, but 320 with
// skewed popularity 177 and 116.  1024 -> 2 x 512, one by one and in tiles: 64 / 96 rows of 20 experts 12.7 / 15.9 and 13.7 /
// 13.8, of 64 experts 18.0 / 25.0 and 19.4 / 21.6, 64 / 128 rows of 128 experts 20.5 / 37.1 and 22.0 / 33.1.
constexpr uint32_t kOneByOneSorted = 160, kOneByOneFound = 80;
// Mean rows per expert from which tiles hold 64 rows rather than 32: ten of 512 experts, 2048 -> 2 x 512, 512 / 1024 /
// 2048 tokens (10 / 20 / 40 rows) 363 / 373 / 390 us with 64 and 363 / 395 / 433 with 32.
constexpr uint32_t kTallMean = 16;

uint32_t product_tile_rows(uint32_t rows, uint32_t experts) {
  if (rows <= (product_sorted(rows, experts) ? kOneByOneSorted : kOneByOneFound)) return 0;
  return rows / experts < kTallMean ? 32u : 64u;
}

// Matrices that together outgrow the 256 MB Infinity Cache stream past the caches where one tile reads them (k_tiles
// looks at each group): 2048 -> 2 x 512, ten of 512 experts, 512 tokens 364 to 336 us, eight tokens 58 to 55, 2048 tokens
// with skewed popularity 448 to 419; MX 2560 -> 2 x 640, 2048 tokens, 363 to 356.  Read by several tiles or held by that
// cache they must not: 8192 tokens 613 to 941, 333 tokens of four of 64 experts, 1024 -> 2 x 256, 20 to 23.
bool product_once(const ProductLaunch& p) {
  return uint64_t(p.experts) * p.n * (p.swiglu ? 2 : 1) * p.k_bytes > (256ull << 20);
}

uint64_t product_blocks(uint32_t rows, uint32_t experts, uint32_t n, uint32_t tile_rows, bool swiglu) {
  const uint64_t strips = (uint64_t(n) + (swiglu ? 15 : 31)) / (swiglu ? 16 : 32);  // the narrowest blocks
  const uint64_t units = tile_rows == 0 ? rows : uint64_t(rows) / tile_rows + experts + 7;
  return units * strips + rows / (2 * kZeroRows) + 1;
}

hipError_t launch_products(ProductLaunch p, uint32_t tile_rows, hipStream_t stream) {
  p.once = product_once(p);
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
