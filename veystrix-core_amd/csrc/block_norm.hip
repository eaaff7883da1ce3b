// The norms before and after a block's boundary in one pass (vm_block_norm).
//
//   n = x / sqrt(mean(x^2) + eps) * post gain      (no post weight: n = x)
//   h = residual_scale * residual + scale * gate * n
//   y = h / sqrt(mean(h^2) + eps) * gain           (no weight: h alone)
//
// gate: none, one per row, per channel or per value, as it is or through a sigmoid; gains are weight or 1 + weight.  The
// second norm reads h as it was computed, before it is rounded to the residual's type.
//
// A row is read once: x and the residual stay in registers from the first sum of squares over the second to the last
// store, eight consecutive values per thread and step (vm_norm.h).  Squares are summed in 64 bits, which no value
// overflows and which costs two operations a value.  Rows to MX are computed in 64 bits throughout, so that e4m3's is
// their one rounding: h is kept as a float and its rest, in the registers that x and the residual leave.
// Bound by HBM (two rows in, two out), or with few rows by one row's latency, which two sums over the row make up.

#include <hip/hip_ext.h>
#include <hip/hip_runtime.h>

#include <type_traits>

#include "vm_internal.h"
#include "vm_mx.h"
#include "vm_norm.h"

namespace vm {

namespace {

constexpr int kBlockNormThreads = 256;

template <int LIE>
__device__ __forceinline__ void load8_any(const void* row, uint32_t dtype, uint32_t at, uint32_t step, uint32_t width,
                                          float v[8]) {
  if (dtype == 0) load8<ActBF16, LIE>(row, at, step, width, v);
  else load8<ActF32, LIE>(row, at, step, width, v);
}
template <int LIE>
__device__ __forceinline__ void store8_any(void* row, uint32_t dtype, uint32_t at, uint32_t step, uint32_t width,
                                           const float v[8]) {
  if (dtype == 0) store8<ActBF16, LIE>(row, at, step, width, v);
  else store8<ActF32, LIE>(row, at, step, width, v);
}

__device__ __forceinline__ const void* row_at(const void* base, uint64_t row, uint64_t stride, uint32_t dtype) {
  return static_cast<const uint8_t*>(base) + row * stride * (dtype == 0 ? 2u : 4u);
}

// Sum over a row's threads, in all of them.
template <int TPR>
__device__ __forceinline__ double row_total(double v, double* part) {
  v = wave_total(v);
  if constexpr (TPR > 64) {
    if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = v;
    __syncthreads();
    v = 0.0;
#pragma unroll
    for (int w = 0; w < TPR / 64; ++w) v += part[w];
  }
  return v;
}

template <class Real>
__device__ __forceinline__ Real gate_sigmoid(float g) {
  if constexpr (sizeof(Real) == 8) return 1.0 / (1.0 + exp(-static_cast<double>(g)));
  else return 1.0f / (1.0f + expf(-g));
}

// TPR threads per row (64 or 256), up to NV steps of eight values per thread.
template <int TPR, int NV, int LIE, bool MXOUT>
__global__ __launch_bounds__(kBlockNormThreads) void k_block_norm(BlockNormLaunch p) {
  static_assert(!MXOUT || LIE != kSpread, "MX rows need a group's values side by side");
  using Real = std::conditional_t<MXOUT, double, float>;
  __shared__ double s_part[2][TPR / 64];
  const uint32_t t = threadIdx.x % TPR;
  const uint32_t row = blockIdx.x * (kBlockNormThreads / TPR) + threadIdx.x / TPR;
  if (row >= p.rows) return;  // TPR 64: whole waves; TPR 256: never
  constexpr uint32_t kStep = LIE == kSpread ? TPR : 1;
  const auto at = [&](int i) { return LIE == kSpread ? i * TPR * 8u + t : (i * TPR + t) * 8u; };
  float h[NV][8], r[NV][8];   // x and the residual, then the sum and, to MX, its rest
  const void* x = row_at(p.x, row, p.x_stride, p.act_dtype);
  const void* res = row_at(p.residual, row, p.residual_stride, p.residual_dtype);
  if (p.act_dtype == 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) load8<ActBF16, LIE>(x, at(i), kStep, p.width, h[i]);
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) load8<ActF32, LIE>(x, at(i), kStep, p.width, h[i]);
  }
  if (p.residual_dtype == 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) load8<ActBF16, LIE>(res, at(i), kStep, p.width, r[i]);
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) load8<ActF32, LIE>(res, at(i), kStep, p.width, r[i]);
  }
  const double width = p.width;
  Real post = 1;
  if (p.post_weight != nullptr) {
    double ss = 0.0;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = fma(static_cast<double>(h[i][j]), static_cast<double>(h[i][j]), ss);
    post = static_cast<Real>(1.0 / sqrt(row_total<TPR>(ss, s_part[0]) / width + p.eps));
  }
  const Real scale = static_cast<Real>(p.scale), residual_scale = static_cast<Real>(p.residual_scale);
  const void* gate = p.gate;
  Real row_gate = 1;
  if (p.gate_kind == kGateRow) {
    const float g = load_any(row_at(p.gate, row, p.gate_stride, p.gate_dtype), 0, p.gate_dtype);
    row_gate = p.sigmoid_gate ? gate_sigmoid<Real>(g) : static_cast<Real>(g);
  } else if (p.gate_kind == kGateValue) {
    gate = row_at(p.gate, row, p.gate_stride, p.gate_dtype);
  }
  double ss = 0.0;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    Real b[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) b[j] = h[i][j];
    if (p.post_weight != nullptr) {
      float w[8];
      load8_any<LIE>(p.post_weight, p.post_dtype, at(i), kStep, p.width, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) b[j] = b[j] * post * (p.one_centered ? static_cast<Real>(w[j]) : 1 + static_cast<Real>(w[j]));
    }
    if (p.gate_kind == kGateChannel || p.gate_kind == kGateValue) {
      float g[8];
      load8_any<LIE>(gate, p.gate_dtype, at(i), kStep, p.width, g);
#pragma unroll
      for (int j = 0; j < 8; ++j) b[j] *= p.sigmoid_gate ? gate_sigmoid<Real>(g[j]) : static_cast<Real>(g[j]);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const Real sum = residual_scale * static_cast<Real>(r[i][j]) + scale * (row_gate * b[j]);
      // values behind the row's end are zeros, but a gate there may have been anything times them
      const bool in = at(i) + j * kStep < p.width;
      h[i][j] = in ? static_cast<float>(sum) : 0.0f;
      if constexpr (MXOUT) r[i][j] = in ? static_cast<float>(sum - static_cast<Real>(h[i][j])) : 0.0f;
      const double wide = in ? static_cast<double>(sum) : 0.0;
      ss = fma(wide, wide, ss);
    }
  }
  if (p.sum_out != nullptr) {
    void* s = const_cast<void*>(row_at(p.sum_out, row, p.sum_stride, p.residual_dtype));
#pragma unroll
    for (int i = 0; i < NV; ++i) store8_any<LIE>(s, p.residual_dtype, at(i), kStep, p.width, h[i]);
  }
  if (p.weight == nullptr) return;
  const Real pre = static_cast<Real>(1.0 / sqrt(row_total<TPR>(ss, s_part[1]) / width + p.eps));
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    float w[8], y[8];
    load8_any<LIE>(p.weight, p.weight_dtype, at(i), kStep, p.width, w);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const Real gain = p.one_centered ? static_cast<Real>(w[j]) : 1 + static_cast<Real>(w[j]);
      if constexpr (MXOUT) {
        const double v = (static_cast<double>(h[i][j]) + static_cast<double>(r[i][j])) * pre * gain;
        y[j] = static_cast<float>(v);
        const double rest = v - static_cast<double>(y[j]);
        y[j] = off_border(y[j], rest > 0.0 ? 1.0f : rest < 0.0 ? -1.0f : 0.0f);
      } else {
        y[j] = h[i][j] * pre * gain;
      }
    }
    if constexpr (!MXOUT) {
      store8_any<LIE>(const_cast<void*>(row_at(p.out, row, p.out_stride, p.act_dtype)), p.act_dtype, at(i), kStep, p.width, y);
    } else {
      uint32_t m = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) m = max(m, mx_magnitude(y[j]));
      m = max(m, dpp_u<kDppQuadXor1>(m));
      m = max(m, dpp_u<kDppQuadXor2>(m));
      const uint32_t e = mx_scale(m);
      if (at(i) < p.width) {  // the width is whole groups, so a lane's eight values are all in it
        const uint64_t first = static_cast<uint64_t>(row) * p.width + at(i);
        *reinterpret_cast<uint2*>(p.values + first) =
            make_uint2(mx_pack4(y[0], y[1], y[2], y[3], e), mx_pack4(y[4], y[5], y[6], y[7], e));
        if (t % 4 == 0) p.scales[first / kMxGroup] = static_cast<uint8_t>(e);
      }
    }
  }
}

template <int TPR, int NV>
hipError_t block_norm_go(const BlockNormLaunch& p, hipStream_t stream) {
  const uint32_t per = kBlockNormThreads / TPR;
  const dim3 grid((p.rows + per - 1) / per);
  auto kernel = p.values != nullptr
                    ? (p.vector ? &k_block_norm<TPR, NV, kUnits, true> : &k_block_norm<TPR, NV, kOnes, true>)
                    : (p.vector ? &k_block_norm<TPR, NV, kUnits, false> : &k_block_norm<TPR, NV, kSpread, false>);
  hipEvent_t start = nullptr, stop = nullptr;
  if (timing_events("norm", &start, &stop))
    hipExtLaunchKernelGGL(kernel, grid, dim3(kBlockNormThreads), 0, stream, start, stop, 0, p);
  else
    hipLaunchKernelGGL(kernel, grid, dim3(kBlockNormThreads), 0, stream, p);
  return hipGetLastError();
}

// Rows from which one wave per row fills the chip (256 CUs of four-row blocks).
constexpr uint32_t kBlockNormWaveRows = 1024;

}  // namespace

hipError_t launch_block_norm(const BlockNormLaunch& p, hipStream_t stream) {
  if (p.rows == 0 || p.width == 0 || p.width > kNormMaxWidth) return hipErrorInvalidValue;
  const uint32_t steps = (p.width + 511) / 512;  // of one wave
  if (p.rows >= kBlockNormWaveRows && steps <= 8) {
    switch (steps) {
      case 1: return block_norm_go<64, 1>(p, stream);
      case 2: return block_norm_go<64, 2>(p, stream);
      case 3:
      case 4: return block_norm_go<64, 4>(p, stream);
      case 5: return block_norm_go<64, 5>(p, stream);
      default: return block_norm_go<64, 8>(p, stream);
    }
  }
  if (steps <= 4) return block_norm_go<256, 1>(p, stream);
  if (steps <= 8) return block_norm_go<256, 2>(p, stream);
  if (steps <= 16) return block_norm_go<256, 4>(p, stream);
  return block_norm_go<256, 8>(p, stream);
}

}  // namespace vm
