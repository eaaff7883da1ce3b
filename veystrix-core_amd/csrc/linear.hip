// Matrix products with bias, activation and residual in their epilogue (vm_linear):
//   out = activation(x . W^T + bias) + residual, fp32 sums, bf16 or MX operands (vm_mx.h), out in bf16 or fp32.
//
// Both formats move as 128-byte chunks of a row (64 bf16 or 128 e4m3 inputs) made of eight 16-byte units, staged in LDS
// by DMA (vm_dma.h); an MX unit is converted to two bf16 operands in registers (vm_operand.h), so both formats have the
// bf16 unit's sums.  The matrix is the first operand, the rows the second, so a lane receives four neighbouring outputs
// of row lane % 16.  The sums go through LDS to the epilogue, whose threads own eight neighbouring outputs each.

#include <hip/hip_ext.h>
#include <hip/hip_runtime.h>

#include <type_traits>

#include "vm_dma.h"
#include "vm_internal.h"
#include "vm_mx.h"
#include "vm_operand.h"

namespace vm {

namespace {

__device__ uint4 g_linear_zeros[kChunk / 16];  // units at and behind the end of a row load from here

// ------------------------------------------------------------- epilogue ---

// 1 / (1 + e^-v)
__device__ __forceinline__ float sigmoid32(float v) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(v * -0x1.715476p+0f));
}

// Eight neighbouring values of one row from column `col`, those at `n` and behind it left out.
__device__ __forceinline__ void load_outputs(const void* row, uint32_t dtype, bool vector, uint32_t col, uint32_t n, float v[8]) {
  if (vector) {
    const uint8_t* src = static_cast<const uint8_t*>(row) + static_cast<size_t>(col) * (dtype == 0 ? 2u : 4u);
    const uint4 a = ldg16(src);
    if (dtype == 0) {
      const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[2 * j] = __uint_as_float(w[j] << 16);
        v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
      }
    } else {
      const uint4 b = ldg16(src + 16);
      const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(w[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = load_any(row, min(col + j, n - 1), dtype);
  }
}

__device__ __forceinline__ void store_outputs(void* row, uint32_t dtype, bool vector, uint32_t col, uint32_t n, const float v[8]) {
  if (vector) {
    uint8_t* dst = static_cast<uint8_t*>(row) + static_cast<size_t>(col) * (dtype == 0 ? 2u : 4u);
    if (dtype == 0) {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = f32_to_bf16(v[2 * j]) | (f32_to_bf16(v[2 * j + 1]) << 16);
      *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
      reinterpret_cast<float4*>(dst)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4*>(dst)[1] = make_float4(v[4], v[5], v[6], v[7]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (col + j >= n) continue;
      if (dtype == 0) ActBF16::store(row, col + j, v[j]);
      else ActF32::store(row, col + j, v[j]);
    }
  }
}

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
    case kActSilu:
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = swiglu(v[j], 1.0f);
      break;
    case kActGelu:
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = 0.5f * v[j] * erfcf(v[j] * -0x1.6a09e6p-1f);
      break;
    case kActGeluTanh:  // (1 + tanh t) / 2 is the sigmoid of 2 t
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] *= sigmoid32(v[j] * fmaf(v[j] * v[j], 0x1.2444f2p-4f, 0x1.988454p+0f));
      break;
    case kActSigmoid:
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = sigmoid32(v[j]);
      break;
    case kActSwiglu:
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = swiglu(v[j], up[j]);
      break;
    default: break;
  }
  if (p.residual != nullptr) {
    float r[8];
    load_outputs(p.residual + row * p.residual_stride, p.residual_dtype, p.vector, col, p.n, r);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] += r[j];
  }
  store_outputs(p.out + row * p.out_stride, p.out_dtype, p.vector, col, p.n, v);
}

// ---------------------------------------------------------------- tiles ---

template <bool MX>
__device__ __forceinline__ f32x4_t unit_product(const Operand<MX>& w, const Operand<MX>& x, f32x4_t acc) {
#pragma unroll
  for (int i = 0; i < (MX ? 2 : 1); ++i)
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, w.part[i]),
                                                  __builtin_bit_cast(bf16x8_t, x.part[i]), acc, 0, 0, 0);
  return acc;
}

// One LDS object per stage, so that the compiler can tell the stage being read from the one being filled.
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

// WM x WN x WK waves; each multiplies 16 RF rows by 16 CF matrix rows, over every WK-th chunk.
template <bool MX, int RF, int CF, int WM, int WN, int WK>
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
  const uint32_t slices = (p.n + cols - 1) / cols;
  const uint32_t row0 = blockIdx.x / slices * kRows, col0 = blockIdx.x % slices * cols;
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
  uint32_t held_x[2][kXWords], held_w[2][kWWords];   // the scale bytes of the stages
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
    for (int i = 0; i < kLoads; ++i) load_to_lds(in ? src[i] + c * kChunk : zeros, st + i * 1024u);
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
          acc[i][f] = unit_product<MX>(w, Operand<MX>(xv[i], scale(MX ? xs[i] : 0u, h)), acc[i][f]);
      }
    }
  };

  // Two stages: one is multiplied while the next step's chunks are on their way to the other (behind the last step that
  // one again, which is not read).
  begin(std::integral_constant<int, 0>{}, 0);
  for (uint32_t step = 0; step < steps; step += 2) {
    unroll<0, 2>([&](auto J) {
      constexpr int j = decltype(J)::value;
      if (step + j >= steps) return;
      wait_vm<0>();    // this wave's loads of the stage have landed
      wait_lgkm0();    // its reads of the other stage are done
      bare_barrier();
      begin(std::integral_constant<int, 1 - j>{}, min(step + j + 1, steps - 1));
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

template <class Kernel>
hipError_t go(Kernel kernel, uint64_t blocks, uint32_t threads, const LinearLaunch& p, hipStream_t stream) {
  hipEvent_t start = nullptr, stop = nullptr;
  if (timing_events("linear", &start, &stop))
    hipExtLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(blocks)), dim3(threads), 0, stream, start, stop, 0, p);
  else
    hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(blocks)), dim3(threads), 0, stream, p);
  return hipGetLastError();
}

template <bool MX, int RF, int CF, int WM, int WN, int WK>
hipError_t tiles_go(const LinearLaunch& p, hipStream_t stream) {
  const uint32_t rows = 16 * RF * WM, cols = 16 * CF * WN / (p.activation == kActSwiglu ? 2 : 1);
  const uint64_t blocks = uint64_t((p.rows + rows - 1) / rows) * ((p.n + cols - 1) / cols);
  return go(&k_linear<MX, RF, CF, WM, WN, WK>, blocks, 64 * WM * WN * WK, p, stream);
}

template <bool MX>
hipError_t linear_go(const LinearLaunch& p, hipStream_t stream) {
  return tiles_go<MX, 2, 2, 2, 2, 1>(p, stream);
}

}  // namespace

uint64_t linear_blocks(uint32_t rows, uint32_t n) {  // of the smallest tiles
  return (uint64_t(rows) + 63) / 64 * ((uint64_t(n) + 31) / 32);
}

hipError_t launch_linear(const LinearLaunch& p, hipStream_t stream) {
  if (p.rows == 0 || p.n == 0 || p.k_bytes == 0) return hipErrorInvalidValue;
  return p.mx ? linear_go<true>(p, stream) : linear_go<false>(p, stream);
}

}  // namespace vm
