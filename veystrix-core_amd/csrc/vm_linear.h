// The kernels of linear.hip (bf16) and linear_mx.hip, which are two files because their instances compile for minutes.
//
// Matrix products with bias, activation and residual in their epilogue (vm_linear):
//   out = activation(x . W^T + bias) + residual, fp32 sums, bf16 or MX operands (vm_mx.h), out in bf16 or fp32.
//
// Both formats move as runs of a row (64 or 128 bytes: 16-byte units of 8 bf16 or 16 e4m3 inputs), staged in LDS by DMA
// (vm_dma.h); an MX unit is converted to two bf16 operands in registers (vm_operand.h), so both formats have the bf16
// unit's sums.  The matrix is the first operand, the rows the second, so a lane receives four neighbouring outputs of row
// lane % 16.  Three kinds of calls, chosen by choose_form (vm_linear_form.h):
//   k_few     up to four rows: the matrix read once by plain loads, no MFMA; bound by its bytes (one row 2560 -> 2560, 13 MB,
//             4.6 us, of which a launch is two; of MX 3.7; four rows 5.6).
//   k_linear  small tiles, whose waves share the inputs where there are few tiles, so that a call of few rows is done in
//             a few steps: bound by the loads' way from L2 and HBM (32 rows MX 2560 -> 2 x 640 6.4 us, 64 rows 2560 -> 2560
//             7.9, 333 rows 1000 -> 1333 7.8, 2048 rows 2048 -> 512 12.1: 134 MB past the L2s at 11 TB/s).
//   k_large   large tiles: bound by the products (1240 TFLOP/s of 2560 inputs, 1330 of 8192, a library's 8192^3 product
//             1610) and, all tiles of a round ending together, by the outputs' way to HBM.
// Times are a kernel trace's medians.

#pragma once

#include <hip/hip_ext.h>
#include <hip/hip_runtime.h>

#include <type_traits>

#include "vm_any.h"
#include "vm_dma.h"
#include "vm_internal.h"
#include "vm_linear_form.h"
#include "vm_mx.h"
#include "vm_operand.h"

namespace vm {

namespace {

__device__ uint4 g_linear_zeros[kChunk / 16];  // units at and behind the end of a row load from here

// The lanes' 16 (4) bytes at `src` to LDS at `dst` (the same in all lanes) and on, lane by lane.  As assembly, because
// the compiler waits for all such loads of its own before any LDS read that it cannot tell from their targets, which with
// four stages is every one; it holds no registers, and its users wait for it by wait_vm.
__device__ __forceinline__ void dma16(const void* src, uint32_t dst) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(dst) : "memory", "m0");
}
__device__ __forceinline__ void dma16(const void* base, uint32_t offset, uint32_t dst) {   // base the same in all lanes
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %0" ::"s"(base), "v"(offset), "s"(dst) : "memory", "m0");
}
__device__ __forceinline__ void dma4(const void* src, uint32_t dst) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(src), "s"(dst) : "memory", "m0");
}
__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) void*)p));
}

// ------------------------------------------------------------- epilogue ---

// What an instance's epilogue computes, so that unrolled code holds one activation.
enum : int { kEpiPlain = 0, kEpiSigmoid = 1, kEpiGelu = 2, kEpiSwiglu = 3 };

// v Phi(v).  For z = |v| / sqrt 2, Phi(-|v|) = erfc(z) / 2 is t e^(-z^2) 2^P(t) with t = 1 / (1 + 0.55 z) and P a
// polynomial of the ninth degree, fitted for the least largest error over z up to 9.6 (2^-23 in log2; with fp32's roundings
// 8 + 2 v^2 half steps over eight million values, on to z of 10.1, behind which fp32 holds nothing).  The power of two comes
// as its root on either factor, since the hardware flushes subnormal ones, from |v| of 13 on.  erfcf took 22 us of the
// 8192 x 2560 outputs of a call of 119, this 9.
__device__ __forceinline__ float gelu32(float v) {
  const float t = __builtin_amdgcn_rcpf(fmaf(fabsf(v), 0x1.8e3e18p-2f, 1.0f));
  constexpr float kP[10] = {-0x1.581160p+0f, 0x1.6ffd0ap-1f,  0x1.1d3eb2p-2f,  -0x1.0b859cp-3f, 0x1.a717ccp-2f,   // P / 2
                            -0x1.3176e0p+0f, 0x1.304d2cp+0f, -0x1.f55f98p-2f, 0x1.5652f8p-5f,  0x1.0f3ca0p-6f};
  float e = kP[9];
#pragma unroll
  for (int i = 8; i >= 0; --i) e = fmaf(e, t, kP[i]);
  const float root = __builtin_amdgcn_exp2f(fmaf(v * v, -0x1.715476p-2f, e)), q = t * root;
  return v < 0.0f ? v * q * root : v * fmaf(-q, root, 1.0f);
}

// v or 1 times 1 / (1 + e^-u): silu, sigmoid (u = v) and, since (1 + tanh t) / 2 is the sigmoid of 2 t, gelu_tanh, whose
// u = v (a + b v^2) alone takes the square, which overflows from 2^64 on: times a b of zero it would be no number.  A
// negative u's exponential comes as its root on either factor, as swiglu's, so that results keep their bits down to fp32's
// least: off by 16 + 2 |u| half steps at most, gelu_tanh by up to 20 + 7 |u| with u's own roundings.
struct SigmoidForm {
  bool cubic, times;
  __device__ __forceinline__ explicit SigmoidForm(uint32_t activation)
      : cubic(activation == kActGeluTanh), times(activation != kActSigmoid) {}
  __device__ __forceinline__ float operator()(float v) const {
    const float u = cubic ? v * fmaf(v * v, 0x1.2444f2p-4f, 0x1.988454p+0f) : v;
    const float root = __builtin_amdgcn_exp2f(fabsf(u) * -0x1.715476p-1f);   // e^(-|u| / 2)
    const float r = __builtin_amdgcn_rcpf(fmaf(root, root, 1.0f));
    const float w = u < 0.0f ? root : 1.0f;
    return (times ? v * w : w) * r * w;
  }
};

__device__ __forceinline__ void add_bias(const LinearLaunch& p, uint32_t at, uint32_t left, float v[8]) {
#pragma unroll
  for (uint32_t j = 0; j < 8; ++j) v[j] += load_any(p.bias, at + min(j, left - 1), p.bias_dtype);
}

// Activation, residual and store of eight sums of row `row` from column `col`; `up`: SwiGLU's other half.
__device__ __forceinline__ void finish8(const LinearLaunch& p, uint32_t row, uint32_t col, float v[8], float up[8]) {
  if (p.bias != nullptr) {
    add_bias(p, col, p.n - col, v);
    if (p.activation == kActSwiglu) add_bias(p, p.n + col, p.n - col, up);
  }
  switch (p.activation) {
    case kActRelu:
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = v[j] < 0.0f ? 0.0f : v[j];   // NaN stays
      break;
    case kActGelu:
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = gelu32(v[j]);
      break;
    case kActSilu:
    case kActGeluTanh:
    case kActSigmoid: {
      const SigmoidForm sigmoid(p.activation);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = sigmoid(v[j]);
      break;
    }
    case kActSwiglu:
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = swiglu(v[j], up[j]);
      break;
    default: break;
  }
  if (p.residual != nullptr) {
    float r[8];
    load_run<8>(p.residual + row * p.residual_stride, p.residual_dtype, col, p.n, r);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] += r[j];
  }
  store_run<8>(p.out + row * p.out_stride, p.out_dtype, col, p.n, v);
}

// ------------------------------------------------------------- few rows ---

// The sum of one output through the epilogue.
__device__ __forceinline__ void finish1(const LinearLaunch& p, uint32_t row, uint32_t col, float v, float up) {
  if (p.bias != nullptr) {
    v += load_any(p.bias, col, p.bias_dtype);
    if (p.activation == kActSwiglu) up += load_any(p.bias, p.n + col, p.bias_dtype);
  }
  switch (p.activation) {
    case kActNone: break;
    case kActRelu: v = v < 0.0f ? 0.0f : v; break;
    case kActGelu: v = gelu32(v); break;
    case kActSwiglu: v = swiglu(v, up); break;
    default: v = SigmoidForm(p.activation)(v);
  }
  if (p.residual != nullptr) v += load_any(p.residual + row * p.residual_stride, col, p.residual_dtype);
  if (p.out_dtype == 0) ActBF16::store(p.out + row * p.out_stride, col, v);
  else ActF32::store(p.out + row * p.out_stride, col, v);
}

template <bool MX>
__device__ __forceinline__ float few_dot(const Operand<MX>& w, const Operand<MX>& x, float acc) {
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

// Up to R rows by four matrix rows (with SwiGLU two gates and their ups) per block, no MFMA: a wave reads a kilobyte of
// each matrix row at a time, and the block's waves share the rows' length, so that all of a call's matrix is asked for
// at once.
template <bool MX, int R>
__global__ __launch_bounds__(64 * kFewWaves) void k_few(LinearLaunch p) {
  __shared__ float s_sum[kFewWaves][kFewMatrix * R];
  const uint32_t tid = threadIdx.x, lane = tid & 63u;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6), waves = blockDim.x / 64u;
  const bool pairs = p.activation == kActSwiglu;
  const uint32_t cols = pairs ? kFewMatrix / 2 : kFewMatrix, col0 = blockIdx.x * cols;
  const uint8_t *w_row[kFewMatrix], *ws_row[kFewMatrix], *x_row[R], *xs_row[R];
#pragma unroll
  for (uint32_t j = 0; j < kFewMatrix; ++j) {
    const bool up = pairs && j >= kFewMatrix / 2;
    const uint64_t m = min(col0 + (up ? j - kFewMatrix / 2 : j), p.n - 1) + (up ? p.n : 0u);
    w_row[j] = p.w + m * p.w_stride;
    ws_row[j] = MX ? p.w_scales + m * p.w_scale_stride : nullptr;
  }
#pragma unroll
  for (uint32_t i = 0; i < R; ++i) {
    const uint64_t r = min(i, p.rows - 1);
    x_row[i] = p.x + r * p.x_stride;
    xs_row[i] = MX ? p.x_scales + r * p.x_scale_stride : nullptr;
  }
  float acc[kFewMatrix][R] = {};
  for (uint32_t at = wave * 1024u + lane * 16u; at < p.k_bytes; at += waves * 1024u) {
    uint4 w[kFewMatrix], x[R];
    uint32_t ws[kFewMatrix] = {}, xs[R] = {};
#pragma unroll
    for (int j = 0; j < kFewMatrix; ++j) w[j] = ldg16(w_row[j] + at);
#pragma unroll
    for (int i = 0; i < R; ++i) x[i] = ldg16(x_row[i] + at);
    if constexpr (MX) {
#pragma unroll
      for (int j = 0; j < kFewMatrix; ++j) ws[j] = ws_row[j][at / kMxGroup];
#pragma unroll
      for (int i = 0; i < R; ++i) xs[i] = xs_row[i][at / kMxGroup];
    }
    __builtin_amdgcn_sched_barrier(0);
    const auto scale = [](uint32_t byte) { return __uint_as_float(byte << 23); };
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const Operand<MX> xo(x[i], scale(xs[i]));
#pragma unroll
      for (int j = 0; j < kFewMatrix; ++j) acc[j][i] = few_dot(Operand<MX>(w[j], scale(ws[j])), xo, acc[j][i]);
    }
  }
#pragma unroll
  for (int j = 0; j < kFewMatrix; ++j)
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const float v = group_sum<64>(acc[j][i]);
      if (lane == 63) s_sum[wave][j * R + i] = v;
    }
  __syncthreads();
  const uint32_t row = tid % R, j = tid / R;
  if (j >= cols || row >= p.rows || col0 + j >= p.n) return;
  float v = 0.0f, up = 0.0f;
  for (uint32_t q = 0; q < waves; ++q) {
    v += s_sum[q][j * R + row];
    if (pairs) up += s_sum[q][(j + kFewMatrix / 2) * R + row];
  }
  finish1(p, row, col0 + j, v, up);
}

// ---------------------------------------------------------------- tiles ---

// Tile (row tile, column tile) of a block: every XCD (blocks b, b + 8, ..) takes a run of tiles, and runs go down columns
// of up to eight row tiles, so that the tiles of one L2 share rows and matrix rows (2048 rows 2048 -> 512 in 32 x 64 tiles
// 11.3 us, row after row 13.1).
__device__ __forceinline__ void tile_of(uint32_t block, uint32_t row_tiles, uint32_t col_tiles, uint32_t* row, uint32_t* col) {
  const uint32_t total = row_tiles * col_tiles, xcd = block & 7u, each = total >> 3, over = total & 7u;
  const uint32_t t = xcd * each + min(xcd, over) + (block >> 3);
  const uint32_t panel = t / (8u * col_tiles), in = t % (8u * col_tiles);
  const uint32_t height = min(8u, row_tiles - panel * 8u);
  *row = panel * 8u + in % height;
  *col = in / height;
}

// LDS of stage J.
template <int J, int BYTES>
__device__ __forceinline__ uint8_t* linear_stage() {
  __shared__ uint4 buf[BYTES / 16];
  return reinterpret_cast<uint8_t*>(buf);
}

// The four scale bytes of chunk c of one row, those behind its end zero.
__device__ __forceinline__ uint32_t scale_bytes(const uint8_t* row, uint32_t c, uint32_t groups, bool whole) {
  if (c * 4u >= groups) return 0;
  if (whole) return ldg_u32(row + c * 4u);
  uint32_t v = 0;
#pragma unroll
  for (uint32_t j = 0; j < 4; ++j)
    if (c * 4u + j < groups) v |= static_cast<uint32_t>(row[c * 4u + j]) << (8u * j);
  return v;
}

// WM x WN x WK waves; each multiplies 16 RF rows by 16 CF matrix rows, over every WK-th chunk; S stages.
template <bool MX, int RF, int CF, int WM, int WN, int WK, int S>
__global__ __launch_bounds__(64 * WM * WN * WK) void k_linear(LinearLaunch p) {
  constexpr int kWaves = WM * WN * WK;
  constexpr uint32_t kRows = 16 * RF * WM, kMatrix = 16 * CF * WN;
  constexpr int kPart = (kRows + kMatrix) * kChunk;           // bytes of one chunk of all rows
  constexpr int kStage = kPart * WK;
  constexpr int kLoads = (kRows + kMatrix) / 8 / (WM * WN);   // 1 KB loads (eight rows) per wave and step
  static_assert(kLoads * 8 * WM * WN == kRows + kMatrix, "whole loads per wave");
  const uint32_t tid = threadIdx.x, lane = tid & 63u, lm = lane & 15u, kb = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t wk = wave / (WM * WN), wmn = wave % (WM * WN), wm = wmn % WM, wn = wmn / WM;
  const bool pairs = p.activation == kActSwiglu;
  const uint32_t cols = pairs ? kMatrix / 2 : kMatrix;        // outputs per block
  uint32_t row_tile, col_tile;
  tile_of(blockIdx.x, (p.rows + kRows - 1) / kRows, (p.n + cols - 1) / cols, &row_tile, &col_tile);
  const uint32_t row0 = row_tile * kRows, col0 = col_tile * cols;
  const auto x_row = [&](uint32_t r) { return static_cast<uint64_t>(min(row0 + r, p.rows - 1)); };
  const auto w_row = [&](uint32_t r) {   // with SwiGLU the second half of the block's matrix rows are up rows
    const bool up = pairs && r >= cols;
    return static_cast<uint64_t>(min(col0 + (up ? r - cols : r), p.n - 1) + (up ? p.n : 0u));
  };

  const uint32_t sub = lane / 8u;
  const uint32_t at = ((lane % 8u) ^ tile_swz(sub)) * 16u;    // byte of the lane's unit in a chunk
  const uint8_t* src[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const uint32_t r = (wmn * kLoads + i) * 8u + sub;
    src[i] = (r < kRows ? p.x + x_row(r) * p.x_stride : p.w + w_row(r - kRows) * p.w_stride) + at;
  }
  constexpr int kXWords = MX ? (RF + 3) / 4 : 1, kWWords = MX ? (CF + 3) / 4 : 1;
  const uint8_t *xs_row[kXWords], *ws_row[kWWords];
  if constexpr (MX) {
#pragma unroll
    for (int s = 0; s < kXWords; ++s)
      xs_row[s] = p.x_scales + x_row(wm * 16 * RF + min(s * 64u + lane, 16u * RF - 1u)) * p.x_scale_stride;
#pragma unroll
    for (int s = 0; s < kWWords; ++s)
      ws_row[s] = p.w_scales + w_row(wn * 16 * CF + min(s * 64u + lane, 16u * CF - 1u)) * p.w_scale_stride;
  }
  const uint32_t chunks = (p.k_bytes + kChunk - 1) / kChunk, groups = p.k_bytes / kMxGroup;
  const uint32_t steps = (chunks + WK - 1) / WK;
  const uint8_t* zeros = reinterpret_cast<const uint8_t*>(g_linear_zeros);
  VM_KEEP(zeros);
  uint32_t held_x[S][kXWords], held_w[S][kWWords];   // the scale bytes of the stages
  const auto begin = [&](auto J, uint32_t step) {
    constexpr int j = decltype(J)::value;
    const uint32_t c = step * WK + wk;
    if constexpr (MX) {
#pragma unroll
      for (int s = 0; s < kXWords; ++s) held_x[j][s] = scale_bytes(xs_row[s], c, groups, p.whole_scales);
#pragma unroll
      for (int s = 0; s < kWWords; ++s) held_w[j][s] = scale_bytes(ws_row[s], c, groups, p.whole_scales);
    }
    __builtin_amdgcn_sched_barrier(0);
    uint8_t* st = linear_stage<j, kStage>() + wk * kPart + wmn * (kLoads * 1024u);
    const bool in = c * kChunk + at < p.k_bytes;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) dma16(in ? src[i] + c * kChunk : zeros, lds_address(st) + i * 1024u);
    __builtin_amdgcn_sched_barrier(0);
  };

  const uint32_t swz = tile_swz(lm);
  const uint32_t unit[2] = {(kb ^ swz) * 16u, ((4u | kb) ^ swz) * 16u};
  const uint32_t x_base = wk * kPart + (wm * (16 * RF) + lm) * kChunk;
  const uint32_t w_base = wk * kPart + (kRows + wn * (16 * CF) + lm) * kChunk;
  f32x4_t acc[RF][CF];
#pragma unroll
  for (int i = 0; i < RF; ++i)
#pragma unroll
    for (int f = 0; f < CF; ++f) acc[i][f] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  const auto compute = [&](auto J) {
    constexpr int j = decltype(J)::value;
    const uint8_t* st = linear_stage<j, kStage>();
    uint32_t xs[RF], ws[CF];
    if constexpr (MX) {
      const auto from = [&](uint32_t r, uint32_t v) {
        return static_cast<uint32_t>(__builtin_amdgcn_ds_bpermute(static_cast<int>(((r & 63u) + lm) * 4u), static_cast<int>(v)));
      };
#pragma unroll
      for (int i = 0; i < RF; ++i) xs[i] = from(i * 16u, held_x[j][i / 4]);
#pragma unroll
      for (int f = 0; f < CF; ++f) ws[f] = from(f * 16u, held_w[j][f / 4]);
    }
    const auto scale = [&](uint32_t bytes, int h) {   // of inputs 16 kb .. +15 of half h of the chunk
      return MX ? __uint_as_float(((bytes >> (16 * h + 8u * (kb >> 1))) & 0xffu) << 23) : 1.0f;
    };
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint4 wv[CF], xv[RF];
#pragma unroll
      for (int f = 0; f < CF; ++f) wv[f] = *reinterpret_cast<const uint4*>(st + w_base + f * 16 * kChunk + unit[h]);
#pragma unroll
      for (int i = 0; i < RF; ++i) xv[i] = *reinterpret_cast<const uint4*>(st + x_base + i * 16 * kChunk + unit[h]);
#pragma unroll
      for (int f = 0; f < CF; ++f) {
        const Operand<MX> w(wv[f], scale(MX ? ws[f] : 0u, h));
#pragma unroll
        for (int i = 0; i < RF; ++i)
          acc[i][f] = unit_mfma<MX>(w, Operand<MX>(xv[i], scale(MX ? xs[i] : 0u, h)), acc[i][f]);
      }
    }
  };

  // One stage is multiplied while the others' steps are on their way (behind the last step zeros, so that every step has
  // as many loads).
  unroll<0, S - 1>([&](auto J) { begin(J, decltype(J)::value); });
  for (uint32_t step = 0; step < steps; step += S) {
    unroll<0, S>([&](auto J) {
      constexpr int j = decltype(J)::value;
      if (step + j >= steps) return;
      wait_vm<(S - 2) * kLoads>();   // this wave's loads of the stage have landed
      wait_lgkm0();                  // its reads of the stage before are done
      bare_barrier();
      begin(std::integral_constant<int, (j + S - 1) % S>{}, step + j + S - 1);
      compute(J);
      __builtin_amdgcn_sched_barrier(0);
    });
  }
  wait_vm<0>();  // no load into LDS outlives the block
  wait_lgkm0();
  bare_barrier();

  // Epilogue, 16 rows of every wave at a time: sums to LDS as [wk][row][matrix row], then eight outputs per thread.
  constexpr uint32_t kLine = kMatrix + 4, kRowsPart = 16 * WM;
  static_assert(WK * kRowsPart * kLine * 4 <= kStage, "a stage holds the sums of 16 rows of every wave");
  float* sums = reinterpret_cast<float*>(linear_stage<0, kStage>());
#pragma unroll
  for (int i = 0; i < RF; ++i) {
    if (i > 0) __syncthreads();
#pragma unroll
    for (int f = 0; f < CF; ++f)
      *reinterpret_cast<f32x4_t*>(sums + (wk * kRowsPart + wm * 16 + lm) * kLine + wn * (16 * CF) + f * 16 + 4 * kb) = acc[i][f];
    __syncthreads();
    const uint32_t per_row = cols / 8;
    for (uint32_t item = tid; item < kRowsPart * per_row; item += 64 * kWaves) {
      const uint32_t line = item / per_row, col = item % per_row * 8u;
      const uint32_t row = row0 + (line / 16u) * (16 * RF) + i * 16u + line % 16u;
      if (row >= p.rows || col0 + col >= p.n) continue;
      float v[8] = {}, up[8] = {};
#pragma unroll
      for (int q = 0; q < WK; ++q) {
        const float* from = sums + (q * kRowsPart + line) * kLine + col;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += from[j];
        if (pairs) {
#pragma unroll
          for (int j = 0; j < 8; ++j) up[j] += from[cols + j];
        }
      }
      finish8(p, row, col0 + col, v, up);
    }
  }
}

// ---------------------------------------------------------- large tiles ---

// Units of a row of 64 bytes lie at unit u ^ strip_swz(row) of it: the four lane groups of a read (lane: row lane % 16,
// unit lane / 16) then meet all 64 banks each.
__device__ __forceinline__ uint32_t strip_swz(uint32_t r) { return (((r >> 1) ^ (r >> 2)) & 2u) | ((r >> 3) & 1u); }

// 16 RF WM rows by 16 CF WN matrix rows; eight waves of 16 RF rows by 16 CF matrix rows in two groups of four, one wave of
// each on a SIMD.  A step of 64 bytes of every row is a slot of reads from LDS and of the loads of the third next step,
// and a slot of MFMAs; the second group runs a slot behind the first, so that one reads while the other multiplies.  Four
// stages hold the step being read and three on their way.  Every wait for loads is the kernel's own: the compiler's, for
// loads that it issued, came before every read and cost a third of the time.
// 8192 x 2560 x 2560 85 to 86 us at 256 x 320 (two stages of 128 bytes 95, half of the matrix rows per slot 90, loads'
// addresses in 64 bits 87), of which the MFMAs take 50 at the 2.0 GHz that it runs at; with bias, SiLU and residual 98, of
// operands that come from HBM 112 in a graph and 115 to 120 traced.  A library's product of this size, without an epilogue,
// took 106.  Of MX 2560 -> 2 x 640 with SwiGLU 54: the MFMAs take 51,200 cycles of a SIMD, 40 % of that at 2.4 GHz, beside 3.4
// other vector instructions to one of them, most of them conversions.  Not kept: loads in
// the MFMAs' slot, waves' priorities the other way round (within 1 %), lines of later steps (4 to 8 ahead) or of the residual
// asked for beforehand (8 % and 1 % slower).
// Fragments of the matrix are dealt in pairs: a lane's eight values of a pair are neighbouring outputs of its row (with
// SwiGLU four gates and four ups of neighbouring outputs), so that sums go from registers to memory.
template <bool MX, int EPI, int RF, int CF, int WM, int WN>
__global__ __launch_bounds__(512, 2) void k_large(LinearLaunch p) {
  static_assert(WM * WN == 8 && CF % 2 == 0, "eight waves, whole pairs");
  constexpr bool kPairs = EPI == kEpiSwiglu;
  constexpr uint32_t kRows = 16 * RF * WM, kMatrix = 16 * CF * WN, kCols = kPairs ? kMatrix / 2 : kMatrix;
  constexpr uint32_t kStrip = 64;                             // bytes of a row per step
  constexpr int kStage = (kRows + kMatrix) * kStrip;
  // 1 KB loads (16 rows) per step: of rows by every wave, of matrix rows by the waves of either group
  constexpr int kLoadsX = kRows / 128, kLoadsW = kMatrix / 64, kFirst = (kLoadsW + 1) / 2, kSecond = kLoadsW / 2;
  constexpr int kWords = MX ? (kRows + kMatrix + 511) / 512 : 0;   // loads of 64 words of scales per wave and step
  static_assert(kLoadsX * 128 == kRows && kLoadsW * 64 == kMatrix, "whole loads per wave");
  const uint32_t tid = threadIdx.x, lane = tid & 63u, lm = lane & 15u, kb = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t second = wave >> 2;                          // group
  const uint32_t wm = wave % WM, wn = wave / WM;
  uint32_t row_tile, col_tile;
  tile_of(blockIdx.x, (p.rows + kRows - 1) / kRows, (p.n + kCols - 1) / kCols, &row_tile, &col_tile);
  const uint32_t row0 = row_tile * kRows, col0 = col_tile * kCols;
  const auto x_row = [&](uint32_t r) { return static_cast<uint64_t>(min(row0 + r, p.rows - 1)); };
  const auto w_row = [&](uint32_t r) {   // matrix row behind the block's row r
    const uint32_t of = r / (16 * CF), f = r % (16 * CF) / 16, q = r / 4 % 4, e = r % 4;
    const uint32_t col = kPairs ? of * (8 * CF) + f / 2 * 16 + 4 * q + e : of * (16 * CF) + f / 2 * 32 + 8 * q + 4 * (f & 1u) + e;
    return static_cast<uint64_t>(min(col0 + col, p.n - 1) + (kPairs && (f & 1u) != 0 ? p.n : 0u));
  };
  const uint32_t sub = lane / 4u;
  const uint32_t at = ((lane % 4u) ^ strip_swz(sub)) * 16u;
  // loads of x rows wave * kLoadsX .., of matrix rows load_w ..; their lanes' offsets from row0's and col0's rows
  const uint32_t load_w = second ? 4 * kFirst + (wave - 4) * kSecond : wave * kFirst;
  const uint8_t* x_rows = p.x + static_cast<uint64_t>(row0) * p.x_stride;
  const uint8_t* w_rows = p.w + static_cast<uint64_t>(col0) * p.w_stride;
  uint32_t x_off[kLoadsX], w_off[kFirst];
#pragma unroll
  for (int i = 0; i < kLoadsX; ++i)
    x_off[i] = static_cast<uint32_t>((x_row((wave * kLoadsX + i) * 16u + sub) - row0) * p.x_stride) + at;
#pragma unroll
  for (int i = 0; i < kFirst; ++i)
    w_off[i] = static_cast<uint32_t>((w_row(min((load_w + i) * 16u + sub, kMatrix - 1u)) - col0) * p.w_stride) + at;
  const uint8_t* words[kWords + 1];
#pragma unroll
  for (int i = 0; i < kWords; ++i) {
    const uint32_t r = min((wave * kWords + i) * 64u + lane, kRows + kMatrix - 1u);
    words[i] = r < kRows ? p.x_scales + x_row(r) * p.x_scale_stride : p.w_scales + w_row(r - kRows) * p.w_scale_stride;
  }
  const uint32_t steps = (p.k_bytes + kStrip - 1) / kStrip;
  constexpr int kScaleStage = kWords * 8 * 256;
  __shared__ uint4 s_stages[4 * kStage / 16], s_scales[MX ? 4 * kScaleStage / 16 : 1];
  const uint32_t stages_at = lds_address(s_stages), scales_at = lds_address(s_scales);
  // Loads of step s; behind the last step that one again, which is not read, so that every step has as many.  Units
  // behind a row's end load its last one and are cleared when that has landed.
  const uint8_t *x_next, *w_next;
  uint32_t back;
  const auto begin = [&](auto J, uint32_t s) {
    constexpr int j = decltype(J)::value;
    const uint32_t from = min(s, steps - 1);
    if constexpr (MX) {   // the word of the step's chunk, of which it needs two bytes
#pragma unroll
      for (int i = 0; i < kWords; ++i) dma4(words[i] + from / 2u * 4u, scales_at + j * kScaleStage + (wave * kWords + i) * 256u);
    }
    const uint32_t st_x = stages_at + j * kStage + wave * (kLoadsX * 1024u);
    const uint32_t st_w = stages_at + j * kStage + kRows * kStrip + load_w * 1024u;
    x_next = x_rows + from * kStrip;
    w_next = w_rows + from * kStrip;
    back = min(at, min(p.k_bytes - from * kStrip, kStrip) - 16u) - at;
#pragma unroll
    for (int i = 0; i < kLoadsX; ++i) dma16(x_next, x_off[i] + back, st_x + i * 1024u);
#pragma unroll
    for (int i = 0; i < kSecond; ++i) dma16(w_next, w_off[i] + back, st_w + i * 1024u);
  };
  // The first group's odd load of matrix rows, behind the others of the step in stage J.
  const auto begin_odd = [&](auto J) {
    constexpr int i = kFirst - 1;
    if constexpr (kFirst > kSecond)
      dma16(w_next, w_off[i] + back, stages_at + decltype(J)::value * kStage + kRows * kStrip + (load_w + i) * 1024u);
  };
  const auto clear = [&](auto J, uint32_t s) {
    if ((s + 1) * kStrip <= p.k_bytes || s >= steps) return;
    uint4* st = s_stages + decltype(J)::value * (kStage / 16) + lane;
    if (s * kStrip + at >= p.k_bytes) {
#pragma unroll
      for (int i = 0; i < kLoadsX; ++i) st[(wave * kLoadsX + i) * 64u] = make_uint4(0, 0, 0, 0);
      for (uint32_t i = 0; i < (second ? kSecond : kFirst); ++i) st[kRows * kStrip / 16 + (load_w + i) * 64u] = make_uint4(0, 0, 0, 0);
    }
    wait_lgkm0();
  };
  // Loads of a wave that may be on their way when the next step's have landed: those of the two steps behind it.
  constexpr int kAheadFirst = 2 * (kLoadsX + kFirst + kWords), kAheadSecond = 2 * (kLoadsX + kSecond + kWords);

  const uint32_t unit = (kb ^ strip_swz(lm)) * 16u;
  const uint32_t x_base = (wm * (16 * RF) + lm) * kStrip + unit;
  const uint32_t w_base = (kRows + wn * (16 * CF) + lm) * kStrip + unit;
  f32x4_t acc[RF][CF];
#pragma unroll
  for (int i = 0; i < RF; ++i)
#pragma unroll
    for (int f = 0; f < CF; ++f) acc[i][f] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};

  // Step s, in stage j.
  const auto step = [&](auto J, uint32_t s) {
    constexpr int j = decltype(J)::value;
    const uint8_t* st = reinterpret_cast<const uint8_t*>(s_stages) + j * kStage;
    const uint8_t* sc = reinterpret_cast<const uint8_t*>(s_scales) + j * kScaleStage;
    // ---- reads
    __builtin_amdgcn_sched_barrier(0);
    uint4 xv[RF], wv[CF];
    float xs[RF], ws[CF];
    const auto scale = [&](uint32_t row) {   // of the unit's group: byte 2 (j % 2) + kb / 2 of the row's word
      return __uint_as_float(static_cast<uint32_t>(sc[row * 4u + 2u * (j % 2) + (kb >> 1)]) << 23);
    };
#pragma unroll
    for (int i = 0; i < RF; ++i) {
      xv[i] = *reinterpret_cast<const uint4*>(st + x_base + i * 16 * kStrip);
      xs[i] = MX ? scale(wm * (16 * RF) + i * 16 + lm) : 1.0f;
    }
#pragma unroll
    for (int f = 0; f < CF; ++f) {
      wv[f] = *reinterpret_cast<const uint4*>(st + w_base + f * 16 * kStrip);
      ws[f] = MX ? scale(kRows + wn * (16 * CF) + f * 16 + lm) : 1.0f;
    }
    __builtin_amdgcn_sched_barrier(0);
    begin(std::integral_constant<int, (j + 3) % 4>{}, s + 3);
    wait_lgkm0();
    if (second) {
      wait_vm<kAheadSecond>();
      clear(std::integral_constant<int, (j + 1) % 4>{}, s + 1);
    }
    __builtin_amdgcn_sched_barrier(0);
    bare_barrier();
    // ---- products
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int f = 0; f < CF; ++f) {
      const Operand<MX> w(wv[f], ws[f]);
#pragma unroll
      for (int i = 0; i < RF; ++i) acc[i][f] = unit_mfma<MX>(w, Operand<MX>(xv[i], xs[i]), acc[i][f]);
    }
    __builtin_amdgcn_s_setprio(0);
    __builtin_amdgcn_sched_barrier(0);
    if (!second) {
      begin_odd(std::integral_constant<int, (j + 3) % 4>{});
      wait_vm<kAheadFirst>();
      clear(std::integral_constant<int, (j + 1) % 4>{}, s + 1);
    }
    bare_barrier();
  };
  unroll<0, 3>([&](auto J) {
    begin(J, decltype(J)::value);
    if (!second) begin_odd(J);
  });
  wait_vm<kAheadSecond>();
  clear(std::integral_constant<int, 0>{}, 0);
  bare_barrier();
  if (second) bare_barrier();
  for (uint32_t s = 0; s < steps; s += 4)
    unroll<0, 4>([&](auto J) {
      if (s + decltype(J)::value < steps) step(J, s + decltype(J)::value);
    });
  if (!second) bare_barrier();
  wait_vm<0>();  // no load into LDS outlives the block, nor meets what the epilogue keeps there
  bare_barrier();

  // Epilogue, a pair of fragments at a time; RES: no residual, bf16 or fp32.  Its loads are issued together, a bf16
  // residual's a pair ahead.
  const SigmoidForm sigmoid(p.activation);
  const float least = p.activation == kActRelu ? 0.0f : -__builtin_huge_valf();
  const uint32_t row = row0 + wm * (16 * RF) + lm;
  constexpr uint32_t kOut = kPairs ? 4 : 8;                   // outputs of a lane and pair
  const auto col_of = [&](int pair) { return col0 + wn * (kCols / WN) + pair * (4 * kOut) + kOut * kb; };
  const auto epilogue = [&](auto RES) {
    constexpr int res = decltype(RES)::value, kAhead = res == 1 ? 2 : 1;
    constexpr int kRaw = res == 0 ? 1 : kOut / (res == 1 ? 8 : 4) + (kOut == 4 && res == 1 ? 1 : 0);
    uint4 raw[kAhead][RF][kRaw];
    const auto load_residual = [&](int pair) {
      const uint32_t col = col_of(pair);
      if (res == 0 || col + kOut > p.n) return;
#pragma unroll
      for (int i = 0; i < RF; ++i) {
        const uint8_t* from = p.residual + min(row + i * 16u, p.rows - 1) * p.residual_stride + static_cast<uint64_t>(col) * (res == 1 ? 2 : 4);
        uint4* to = raw[pair % kAhead][i];
        if constexpr (res == 1 && kOut == 4) {
          const words2 a = *(const __attribute__((address_space(1))) words2*)from;
          to[0] = make_uint4(a[0], a[1], 0, 0);
        } else {
#pragma unroll
          for (int q = 0; q < kRaw; ++q) {
            const words4 a = *(const __attribute__((address_space(1))) words4*)(from + q * 16);
            to[q] = make_uint4(a[0], a[1], a[2], a[3]);
          }
        }
      }
    };
    load_residual(0);
#pragma unroll
    for (int pair = 0; pair < CF / 2; ++pair) {
      const uint32_t col = col_of(pair);
      if (kAhead == 2 && pair + 1 < CF / 2) load_residual(pair + 1);
      if (kAhead == 1 && pair > 0) load_residual(pair);
      if (col + kOut <= p.n) {
        float bias[8] = {};
        if (p.bias != nullptr) {
          load_run<kOut>(p.bias, p.bias_dtype, col, p.n, bias);
          if constexpr (kPairs) load_run<kOut>(p.bias, p.bias_dtype, p.n + col, 2 * p.n, bias + 4);
        }
#pragma unroll
        for (int i = 0; i < RF; ++i) {
          float y[kOut];
#pragma unroll
          for (uint32_t j = 0; j < kOut; ++j) {
            const float v = acc[i][2 * pair + j / 4][j % 4] + bias[j];
            if constexpr (EPI == kEpiSwiglu) y[j] = swiglu(v, acc[i][2 * pair + 1][j] + bias[j + 4]);
            else if constexpr (EPI == kEpiSigmoid) y[j] = sigmoid(v);
            else if constexpr (EPI == kEpiGelu) y[j] = gelu32(v);
            else y[j] = v < least ? least : v;   // NaN stays
            if constexpr (res != 0) {
              const uint4& a = raw[pair % kAhead][i][res == 1 ? 0 : j / 4];
              const uint32_t at = res == 1 ? j / 2 : j % 4;
              const uint32_t w = at == 0 ? a.x : at == 1 ? a.y : at == 2 ? a.z : a.w;
              y[j] += __uint_as_float(res == 2 ? w : j % 2 == 0 ? w << 16 : w & 0xffff0000u);
            }
          }
          if (row + i * 16u < p.rows)
            store_run<kOut>(p.out + (row + i * 16u) * p.out_stride, p.out_dtype, col, col + kOut, y);
        }
      } else if (col < p.n) {   // the row ends within the run: value by value, by way of LDS
        float* line = reinterpret_cast<float*>(s_stages) + tid * 9u;
#pragma unroll
        for (int i = 0; i < RF; ++i) {
#pragma unroll
          for (int j = 0; j < 8; ++j) line[j] = acc[i][2 * pair + j / 4][j % 4];
          __builtin_amdgcn_wave_barrier();
          if (row + i * 16u < p.rows)
            for (uint32_t j = 0; col + j < p.n; ++j) finish1(p, row + i * 16u, col + j, line[j], kPairs ? line[j + 4] : 0.0f);
          __builtin_amdgcn_wave_barrier();
        }
      }
    }
  };
  if (p.residual == nullptr) epilogue(std::integral_constant<int, 0>{});
  else if (p.residual_dtype == 0) epilogue(std::integral_constant<int, 1>{});
  else epilogue(std::integral_constant<int, 2>{});
}

template <class Kernel>
hipError_t go(Kernel kernel, const LinearForm& c, const LinearLaunch& p, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>(c.blocks)), block(c.threads);
  hipEvent_t start = nullptr, stop = nullptr;
  if (timing_events("linear", &start, &stop))
    hipExtLaunchKernelGGL(kernel, grid, block, 0, stream, start, stop, 0, p);
  else
    hipLaunchKernelGGL(kernel, grid, block, 0, stream, p);
  return hipGetLastError();
}

// Whether the form's row in the table is an instance's tile and threads.
template <bool MX, int FORM, int RF, int CF, int WM, int WN, int WK>
constexpr bool is_form() {
  constexpr TileForm t = kTileForms<MX>[FORM];
  return t.rows == 16 * RF * WM && t.matrix == 16 * CF * WN && t.threads == 64 * WM * WN * WK;
}

template <bool MX, int FORM, int RF, int CF, int WM, int WN, int WK, int S>
hipError_t tiles_go(const LinearForm& c, const LinearLaunch& p, hipStream_t stream) {
  static_assert(is_form<MX, FORM, RF, CF, WM, WN, WK>(), "the grid is the form's");
  return go(&k_linear<MX, RF, CF, WM, WN, WK, S>, c, p, stream);
}

template <bool MX, int FORM, int RF, int CF, int WM, int WN>
hipError_t large_go(const LinearForm& c, const LinearLaunch& p, hipStream_t stream) {
  static_assert(is_form<MX, FORM, RF, CF, WM, WN, 1>(), "the grid is the form's");
  switch (p.activation) {
    case kActSwiglu: return go(&k_large<MX, kEpiSwiglu, RF, CF, WM, WN>, c, p, stream);
    case kActGelu: return go(&k_large<MX, kEpiGelu, RF, CF, WM, WN>, c, p, stream);
    case kActNone:
    case kActRelu: return go(&k_large<MX, kEpiPlain, RF, CF, WM, WN>, c, p, stream);
    default: return go(&k_large<MX, kEpiSigmoid, RF, CF, WM, WN>, c, p, stream);
  }
}

template <bool MX>
hipError_t linear_go(const LinearForm& c, const LinearLaunch& p, hipStream_t stream) {
  // More stages than two keep more loads on their way where a CU's LDS would hold no other tile anyway: 64 rows by
  // 2560 x 2560 9.9 to 8.1 us in 32 x 32 tiles with four, 128 rows 14.0 to 9.8 in 32 x 64 with three, 2048 rows 49 to 43 in
  // 64 x 64 with three.  Of MX the scales' registers wait for the loads between: two are the fastest everywhere.
  constexpr int kDeep = MX ? 2 : 3, kDeepest = MX ? 2 : 4;
  switch (c.form) {
    case kFormFew:
      if (p.rows == 1) return go(&k_few<MX, 1>, c, p, stream);
      if (p.rows == 2) return go(&k_few<MX, 2>, c, p, stream);
      return go(&k_few<MX, 4>, c, p, stream);
    case kForm16:
      return c.alone ? tiles_go<MX, kForm16, 1, 1, 1, 1, 8, kDeep>(c, p, stream) : tiles_go<MX, kForm16, 1, 1, 1, 1, 8, 2>(c, p, stream);
    case kForm32:
      return c.alone ? tiles_go<MX, kForm32, 1, 1, 2, 2, 4, kDeepest>(c, p, stream) : tiles_go<MX, kForm32, 1, 1, 2, 2, 4, 2>(c, p, stream);
    case kForm32x64: return tiles_go<MX, kForm32x64, 1, 2, 2, 2, 2, kDeep>(c, p, stream);
    case kForm64: return tiles_go<MX, kForm64, 2, 2, 2, 2, 1, kDeep>(c, p, stream);
    case kForm128: return large_go<MX, kForm128, 2, 4, 4, 2>(c, p, stream);
    case kForm128x320: return large_go<MX, kForm128x320, 2, 10, 4, 2>(c, p, stream);
    default: break;
  }
  if constexpr (!MX) {
    if (c.form == kForm64Deep) return tiles_go<MX, kForm64Deep, 2, 2, 2, 2, 2, kDeep>(c, p, stream);
    if (c.form == kForm256) return large_go<MX, kForm256, 4, 8, 4, 2>(c, p, stream);
    return large_go<MX, kForm256x320, 4, 10, 4, 2>(c, p, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace

}  // namespace vm
