// Root-mean-square norm of rows with the residual's addition in front of it, and rows in MX (vm_mx.h).
//
//   h = x + residual                       fp32; stored rounded to the input's type where sum_out is given
//   y = h * (1 / sqrt(mean(h^2) + eps)) * gain, gain = weight or 1 + weight
//
// The norm reads h as fp32 holds it, before it is rounded to a stored sum.  y is rounded to the input's type, or to e4m3
// under the scale of its group of 32.  Without a weight the rows are only converted to MX.
//
// A row is read once and stays in registers, eight consecutive values per thread and step, so that four lanes hold a
// scale's group and its maximum takes two DPP steps.  Calls are bound by HBM (two rows in, one and a half out, five
// operations a value), to MX by the compensated products that keep values on their side of e4m3's borders, or, with few
// rows, by one row's latency:
//   * many rows: one wave per row, no barrier, four rows per block;
//   * few rows, or rows wider than a wave's registers: one block of 256 threads per row, so that a row's loads are one
//     round trip.
// 8192 rows of 2560 with residual to MX 35.5 to 36.5 us (147 MB, 4.1 TB/s; with plain fp32 products 31.3, the 4.7 of a
// copy), one row 4.2, 37 of 2048 3.3.
// Rows that are not 16-byte aligned, or whose width is not a multiple of eight, take the same code with element loads
// and stores, their values spread over the row's threads unless MX groups have to lie together.

#include <hip/hip_ext.h>
#include <hip/hip_runtime.h>

#include <type_traits>

#include "vm_internal.h"
#include "vm_mx.h"
#include "vm_norm.h"

namespace vm {

namespace {

constexpr int kNormThreads = 256;

// h * (hi + lo) * (gain + rest) of a factor and a gain given as floats and their rests: the nearest float, and what it
// leaves.
__device__ __forceinline__ float exact_product(float h, float hi, float lo, float gain, float rest, float* off = nullptr) {
#pragma clang fp contract(off)
  const float s = hi * gain;
  const float s_rest = fmaf(hi, rest, fmaf(lo, gain, fmaf(hi, gain, -s)));
  const float p = h * s;
  const float p_rest = fmaf(h, s_rest, fmaf(h, s, -p));
  const float f = p + p_rest;
  if (off != nullptr) *off = p_rest - (f - p);
  return f;
}

// TPR threads per row (64 or 256), up to NV steps of eight values per thread.
template <class A, int TPR, int NV, int LIE, bool MXOUT>
__global__ __launch_bounds__(kNormThreads) void k_norm(NormLaunch p) {
  const uint32_t t = threadIdx.x % TPR;
  const uint32_t row = blockIdx.x * (kNormThreads / TPR) + threadIdx.x / TPR;
  if (row >= p.rows) return;  // TPR 64: whole waves; TPR 256: never
  const auto row_of = [&](const void* base, uint64_t stride) {
    return static_cast<const uint8_t*>(base) + static_cast<uint64_t>(row) * stride * A::kBytes;
  };
  // MX rows: a row's factor in 64 bits (of sums of eight squares in 32) and its products with their rests.  In plain
  // fp32 7 to 22 of 8192 x 2560 values came out on the wrong side of an e4m3 border, of these one to four; the call takes
  // 36 us, plain 31.3, all in 64 bits 48.
  // Of fp32 rows to fp32 the factor comes from 64 bits too: in fp32 its mean, sum, root and quotient are a rounding each
  // (64 bits: 0.2 us a call).
  using Real = std::conditional_t<MXOUT || A::kBytes == 4, double, float>;
  static_assert(!MXOUT || LIE != kSpread, "MX rows need a group's values side by side");
  // element of the thread's first value in step i, and between its values
  constexpr uint32_t kStep = LIE == kSpread ? TPR : 1;
  const auto at = [&](int i) { return LIE == kSpread ? i * TPR * 8u + t : (i * TPR + t) * 8u; };
  float h[NV][8];
  const uint8_t* x = row_of(p.x, p.x_stride);
#pragma unroll
  for (int i = 0; i < NV; ++i) load8<A, LIE>(x, at(i), kStep, p.width, h[i]);
  if (p.residual != nullptr) {
    const uint8_t* r = row_of(p.residual, p.residual_stride);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float v[8];
      load8<A, LIE>(r, at(i), kStep, p.width, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) h[i][j] += v[j];
    }
  }
  const bool normed = !MXOUT || p.weight != nullptr;
  Real scale = 1;
  if (normed) {
    Real ss = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float s8 = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) s8 = fmaf(h[i][j], h[i][j], s8);
      ss += s8;
    }
    ss = wave_total(ss);
    if constexpr (TPR > 64) {
      __shared__ Real s_part[TPR / 64];
      if (t % 64 == 0) s_part[t / 64] = ss;
      __syncthreads();
      ss = 0;
#pragma unroll
      for (int w = 0; w < TPR / 64; ++w) ss += s_part[w];
    }
    scale = 1 / sqrt(ss / static_cast<Real>(p.width) + static_cast<Real>(p.eps));
  }
  const float hi = static_cast<float>(scale);
  const float lo = MXOUT ? static_cast<float>(scale - static_cast<Real>(hi)) : 0.0f;
  if (p.sum_out != nullptr) {
    uint8_t* s = const_cast<uint8_t*>(row_of(p.sum_out, p.sum_stride));
#pragma unroll
    for (int i = 0; i < NV; ++i) store8<A, LIE>(s, at(i), kStep, p.width, h[i]);
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (normed) {
      float g[8];
      if (p.weight_dtype == 0) load8<ActBF16, LIE>(p.weight, at(i), kStep, p.width, g);
      else load8<ActF32, LIE>(p.weight, at(i), kStep, p.width, g);
      float g_rest[8] = {};   // of MX rows' gains
      if (!p.one_centered) {
#pragma unroll
        for (int j = 0; j < 8; ++j) g[j] = one_plus(g[j], &g_rest[j]);
      }
      if constexpr (MXOUT) {
        float y[8];
        uint32_t least = ~0u;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          y[j] = exact_product(h[i][j], hi, lo, g[j], g_rest[j]);
          least = min(least, __float_as_uint(y[j]) & kBorderBits);
        }
        if (least == 0) {  // seldom: one of them may lie on a border
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            float off;
            const float f = exact_product(h[i][j], hi, lo, g[j], g_rest[j], &off);
            y[j] = off_border(f, off);
          }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) h[i][j] = y[j];
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) h[i][j] = h[i][j] * hi * g[j];
      }
    }
    if constexpr (!MXOUT) {
      store8<A, LIE>(const_cast<uint8_t*>(row_of(p.out, p.out_stride)), at(i), kStep, p.width, h[i]);
    } else {
      uint32_t m = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) m = max(m, mx_magnitude(h[i][j]));
      m = max(m, dpp_u<kDppQuadXor1>(m));
      m = max(m, dpp_u<kDppQuadXor2>(m));
      const uint32_t e = mx_scale(m);
      if (at(i) < p.width) {  // the width is whole groups, so a lane's eight values are all in it
        const uint64_t first = static_cast<uint64_t>(row) * p.width + at(i);
        *reinterpret_cast<uint2*>(p.values + first) =
            make_uint2(mx_pack4(h[i][0], h[i][1], h[i][2], h[i][3], e), mx_pack4(h[i][4], h[i][5], h[i][6], h[i][7], e));
        if (t % 4 == 0) p.scales[first / kMxGroup] = static_cast<uint8_t>(e);
      }
    }
  }
}

template <class A, int TPR, int NV>
hipError_t norm_go(const NormLaunch& p, hipStream_t stream) {
  const uint32_t per = kNormThreads / TPR;
  const dim3 grid((p.rows + per - 1) / per);
  auto kernel = p.values != nullptr ? (p.vector ? &k_norm<A, TPR, NV, kUnits, true> : &k_norm<A, TPR, NV, kOnes, true>)
                                    : (p.vector ? &k_norm<A, TPR, NV, kUnits, false> : &k_norm<A, TPR, NV, kSpread, false>);
  hipEvent_t start = nullptr, stop = nullptr;
  if (timing_events("norm", &start, &stop))
    hipExtLaunchKernelGGL(kernel, grid, dim3(kNormThreads), 0, stream, start, stop, 0, p);
  else
    hipLaunchKernelGGL(kernel, grid, dim3(kNormThreads), 0, stream, p);
  return hipGetLastError();
}

// Rows from which one wave per row fills the chip (256 CUs of four-row blocks).
constexpr uint32_t kNormWaveRows = 1024;

template <class A>
hipError_t norm_dispatch(const NormLaunch& p, hipStream_t stream) {
  const uint32_t steps = (p.width + 511) / 512;  // of one wave
  if (p.rows >= kNormWaveRows && steps <= 8) {
    switch (steps) {
      case 1: return norm_go<A, 64, 1>(p, stream);
      case 2: return norm_go<A, 64, 2>(p, stream);
      case 3: return norm_go<A, 64, 3>(p, stream);
      case 4: return norm_go<A, 64, 4>(p, stream);
      case 5: return norm_go<A, 64, 5>(p, stream);
      case 6: return norm_go<A, 64, 6>(p, stream);
      default: return norm_go<A, 64, 8>(p, stream);
    }
  }
  if (steps <= 4) return norm_go<A, 256, 1>(p, stream);
  if (steps <= 8) return norm_go<A, 256, 2>(p, stream);
  if (steps <= 16) return norm_go<A, 256, 4>(p, stream);
  return norm_go<A, 256, 8>(p, stream);
}

}  // namespace

hipError_t launch_norm(const NormLaunch& p, hipStream_t stream) {
  if (p.rows == 0 || p.width == 0 || p.width > kNormMaxWidth) return hipErrorInvalidValue;
  return p.act_dtype == 0 ? norm_dispatch<ActBF16>(p, stream) : norm_dispatch<ActF32>(p, stream);
}

}  // namespace vm
