// The norms before and after a block's boundary in one pass (vm_block_norm).
//
//   n = x / sqrt(mean(x^2) + eps) * post gain      (no post weight: n = x)
//   h = residual_scale * residual + scale * gate * n
//   y = h / sqrt(mean(h^2) + eps) * gain           (no weight: h alone)
//
// gate: none, one per row, per channel or per value, as it is or through a sigmoid; gains are weight or 1 + weight.  The
// second norm reads h as it was computed, before it is rounded to the residual's type.
//
// A row is read once: x and the residual stay in registers, as they lie in memory, until the first sum of squares is
// known, then h until the second; eight consecutive values per thread and step, at any alignment (vm_any.h).  Squares are
// summed in 64 bits, which no value overflows and which costs two operations a value.  Rows to MX are computed in 64 bits
// throughout, so that e4m3's is their one rounding.
// Bound by HBM (two rows in, two out), or with few rows by one row's latency, which two sums over the row make up: 8192 rows
// of 2560, in a graph over three sets of operands, bf16 36 us (168 MB, 4.7 TB/s), with an fp32 residual 47.5 (252 MB, 5.3); one
// row 5.2.  To MX 39.1 (147 MB, 3.8 TB/s): the vector units are busy half of that time (1582 instructions a row by counter,
// bf16 rows 1140), and the 128 registers of a lane leave four waves a SIMD, which wait 45 % of theirs.  A sigmoid of a gate
// per channel or value costs a 64-bit exponential each to MX: 65 and 68 us, in fp32 45.5 and 52.

#include <hip/hip_ext.h>
#include <hip/hip_runtime.h>

#include <type_traits>

#include "vm_any.h"
#include "vm_internal.h"
#include "vm_mx.h"
#include "vm_norm.h"

namespace vm {

namespace {

constexpr int kBlockNormThreads = 256;

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

// A row's factor, the same in all lanes of the wave: of fp32 values f times 2^past, past being zero but where fp32 would hold
// the factor with fewer bits or not at all, as for rows around 1e30 and a small scale, while its products with the row's
// values may be normal numbers.  (Products in 64 bits instead held up to twice the registers: 8192 fp32 rows of 1024 with a
// gate per value 26.6 to 28.0 us.)
template <class Real>
struct RowFactor {
  Real f;
  int past;
  __device__ __forceinline__ explicit RowFactor(double factor) : past(0) {
    if constexpr (sizeof(Real) == 4) {
      const int e = __builtin_amdgcn_readfirstlane(__builtin_amdgcn_frexp_exp(factor));   // 0 of zero, infinity and NaN
      past = e - max(-120, min(120, e));
      factor = __builtin_amdgcn_ldexp(factor, -past);
    }
    f = static_cast<Real>(factor);
  }
  // Eight values times the factor.
  template <class Values>
  __device__ __forceinline__ void times(const Values& v, Real out[8]) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) out[j] = static_cast<Real>(v[j]) * f;
    if constexpr (sizeof(Real) == 4) {
      if (past != 0) {
#pragma unroll
        for (int j = 0; j < 8; ++j) out[j] = __builtin_amdgcn_ldexpf(out[j], past);
      }
    }
  }
};

// 1 / (1 + e^-g); in fp32 from the exponential of -|g|, which does not overflow where the sigmoid is still a number.
template <class Real>
__device__ __forceinline__ Real gate_sigmoid(float g) {
  if constexpr (sizeof(Real) == 8) return 1.0 / (1.0 + exp(-static_cast<double>(g)));
  const float e = expf(-fabsf(g));
  return (g < 0.0f ? e : 1.0f) / (1.0f + e);
}

// Eight values of a row as they lie in memory, so that a row waits for its sums in half of fp32's registers.
template <class A>
struct RawRun {
  uint32_t w[A::kBytes * 2];
  __device__ __forceinline__ void load(const void* row, uint32_t at, uint32_t width) {
    const uint8_t* from = static_cast<const uint8_t*>(row) + static_cast<size_t>(at) * A::kBytes;
    if (at + 8 <= width) {
#pragma unroll
      for (int q = 0; q < A::kBytes / 2; ++q) {
        const words4 a = *(const __attribute__((address_space(1))) words4*)(from + 16 * q);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[4 * q + i] = a[i];
      }
    } else {
      uint32_t bits[8];
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j) bits[j] = at + j < width ? A::load_bits(row, at + j) : 0u;
#pragma unroll
      for (int i = 0; i < A::kBytes * 2; ++i) w[i] = A::kBytes == 2 ? bits[2 * i % 8] | (bits[(2 * i + 1) % 8] << 16) : bits[i % 8];
    }
  }
  __device__ __forceinline__ float operator[](int j) const {
    if constexpr (A::kBytes == 2) return __uint_as_float(j % 2 == 0 ? w[j / 2] << 16 : w[j / 2] & 0xffff0000u);
    else return __uint_as_float(w[j]);
  }
};

// v as the float that is rounded to e4m3.
__device__ __forceinline__ float towards(double v) {
  const float f = static_cast<float>(v);
  const double rest = v - static_cast<double>(f);
  return off_border(f, rest > 0.0 ? 1.0f : rest < 0.0 ? -1.0f : 0.0f);
}

// Magnitude bits of the largest of the 32 values that four neighbouring lanes hold.
__device__ __forceinline__ uint32_t group_magnitude(const float y[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = max(m, mx_magnitude(y[j]));
  m = max(m, dpp_u<kDppQuadXor1>(m));
  return max(m, dpp_u<kDppQuadXor2>(m));
}

// 2^-80 (off_border knows floats from 2^-101 on, and e4m3 reaches from a group's largest value 2^18 down), zero left out.
constexpr uint32_t kSmallGroup = 0x17800000u - 1u;

// Rows of A and residuals of R; TPR threads per row (64 or 256), up to NV steps of eight values per thread.
template <class A, class R, int TPR, int NV, bool MXOUT>
__global__ __launch_bounds__(kBlockNormThreads) void k_block_norm(BlockNormLaunch p) {
  using Real = std::conditional_t<MXOUT, double, float>;
  __shared__ double s_part[2][TPR / 64];
  const uint32_t t = threadIdx.x % TPR;
  const uint32_t row = blockIdx.x * (kBlockNormThreads / TPR) + threadIdx.x / TPR;
  if (row >= p.rows) return;  // TPR 64: whole waves; TPR 256: never
  const auto at = [&](int i) { return (i * TPR + t) * 8u; };
  RawRun<A> x[NV];
  RawRun<R> r[NV];
  const void* x_row = row_at(p.x, row, p.x_stride, p.act_dtype);
  const void* r_row = row_at(p.residual, row, p.residual_stride, p.residual_dtype);
#pragma unroll
  for (int i = 0; i < NV; ++i) x[i].load(x_row, at(i), p.width);
#pragma unroll
  for (int i = 0; i < NV; ++i) r[i].load(r_row, at(i), p.width);
  const double width = p.width;
  double factor = p.scale;   // of every value of x: its norm's, the row's gate and the scale
  if (p.post_weight != nullptr) {
    double ss = 0.0;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = fma(static_cast<double>(x[i][j]), static_cast<double>(x[i][j]), ss);
    factor /= sqrt(row_total<TPR>(ss, s_part[0]) / width + p.eps);
  }
  const Real residual_scale = static_cast<Real>(p.residual_scale);
  const Real one = p.one_centered ? 0 : 1;
  const void* gate = p.gate;
  if (p.gate_kind == kGateRow) {
    const float g = load_any(row_at(p.gate, row, p.gate_stride, p.gate_dtype), 0, p.gate_dtype);
    factor *= p.sigmoid_gate ? gate_sigmoid<double>(g) : static_cast<double>(g);
  } else if (p.gate_kind == kGateValue) {
    gate = row_at(p.gate, row, p.gate_stride, p.gate_dtype);
  }
  void* sum_out = const_cast<void*>(row_at(p.sum_out, row, p.sum_stride, p.residual_dtype));
  Real h[NV][8];
  double ss = 0.0;
  const RowFactor<Real> of_x(factor);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    of_x.times(x[i], h[i]);
    if (p.post_weight != nullptr) {
      float w[8];
      load_run<8>(p.post_weight, p.post_dtype, at(i), p.width, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) h[i][j] *= one + static_cast<Real>(w[j]);
    }
    if (p.gate_kind == kGateChannel || p.gate_kind == kGateValue) {
      float g[8];
      load_run<8>(gate, p.gate_dtype, at(i), p.width, g);
#pragma unroll
      for (int j = 0; j < 8; ++j) h[i][j] *= p.sigmoid_gate ? gate_sigmoid<Real>(g[j]) : static_cast<Real>(g[j]);
    }
    float sum[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      h[i][j] = fma(residual_scale, static_cast<Real>(r[i][j]), h[i][j]);
      if (at(i) >= p.width) h[i][j] = 0;   // zeros there, but times a scale that is no number
      sum[j] = static_cast<float>(h[i][j]);
    }
    if (p.sum_out != nullptr) store_run<8>(sum_out, p.residual_dtype, at(i), p.width, sum);
    if (at(i) < p.width && at(i) + 8 > p.width) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (at(i) + j >= p.width) h[i][j] = 0;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = fma(static_cast<double>(h[i][j]), static_cast<double>(h[i][j]), ss);
  }
  if (p.weight == nullptr) return;
  const RowFactor<Real> of_h(1.0 / sqrt(row_total<TPR>(ss, s_part[1]) / width + p.eps));
  void* out = const_cast<void*>(row_at(p.out, row, p.out_stride, p.act_dtype));
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    float w[8], y[8];
    load_run<8>(p.weight, p.weight_dtype, at(i), p.width, w);
    uint32_t border = ~0u;
    of_h.times(h[i], h[i]);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      h[i][j] *= one + static_cast<Real>(w[j]);
      y[j] = static_cast<float>(h[i][j]);
      border = min(border, __float_as_uint(y[j]) & kBorderBits);
    }
    if constexpr (!MXOUT) {
      store_run<8>(out, p.act_dtype, at(i), p.width, y);
    } else {
      if (border == 0) {  // seldom: one of them may lie on a border
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = towards(h[i][j]);
      }
      uint32_t m = group_magnitude(y), e = mx_scale(m), up = 0;
      // Groups whose values may lie where fp32's are not whole or not told from borders: 2^100 times theirs, once more.
      if (m - 1u < kSmallGroup) {
        up = 100;
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = towards(__builtin_amdgcn_ldexp(h[i][j], 100));
        e = max(mx_scale(group_magnitude(y)), up);   // scales end at 2^-127
      }
      if (at(i) < p.width) {  // the width is whole groups, so a lane's eight values are all in it
        const uint64_t first = static_cast<uint64_t>(row) * p.width + at(i);
        *reinterpret_cast<uint2*>(p.values + first) =
            make_uint2(mx_pack4(y[0], y[1], y[2], y[3], e), mx_pack4(y[4], y[5], y[6], y[7], e));
        if (t % 4 == 0) p.scales[first / kMxGroup] = static_cast<uint8_t>(e - up);
      }
    }
  }
}

template <class A, class R, int TPR, int NV>
hipError_t block_norm_go(const BlockNormLaunch& p, hipStream_t stream) {
  const uint32_t per = kBlockNormThreads / TPR;
  const dim3 grid((p.rows + per - 1) / per);
  auto kernel = p.values != nullptr ? &k_block_norm<A, R, TPR, NV, true> : &k_block_norm<A, R, TPR, NV, false>;
  hipEvent_t start = nullptr, stop = nullptr;
  if (timing_events("norm", &start, &stop))
    hipExtLaunchKernelGGL(kernel, grid, dim3(kBlockNormThreads), 0, stream, start, stop, 0, p);
  else
    hipLaunchKernelGGL(kernel, grid, dim3(kBlockNormThreads), 0, stream, p);
  return hipGetLastError();
}

// Rows from which one wave per row fills the chip (256 CUs of four-row blocks), and steps of eight values per lane up to
// which it holds them without crowding out other waves: 4000 bf16 rows of 4096 in eight steps of a wave 35.5 us, in two of
// a block 26.6; 8192 of 2560 in five steps 34.5 and 40.
constexpr uint32_t kBlockNormWaveRows = 1024, kBlockNormWaveSteps = 5;

template <class A, class R>
hipError_t block_norm_rows(const BlockNormLaunch& p, hipStream_t stream) {
  const uint32_t steps = (p.width + 511) / 512;  // of one wave
  if (p.rows >= kBlockNormWaveRows && steps <= kBlockNormWaveSteps) {
    switch (steps) {
      case 1: return block_norm_go<A, R, 64, 1>(p, stream);
      case 2: return block_norm_go<A, R, 64, 2>(p, stream);
      case 3:
      case 4: return block_norm_go<A, R, 64, 4>(p, stream);
      default: return block_norm_go<A, R, 64, 5>(p, stream);
    }
  }
  if (steps <= 4) return block_norm_go<A, R, 256, 1>(p, stream);
  if (steps <= 8) return block_norm_go<A, R, 256, 2>(p, stream);
  if (steps <= 12) return block_norm_go<A, R, 256, 3>(p, stream);
  if (steps <= 16) return block_norm_go<A, R, 256, 4>(p, stream);
  return block_norm_go<A, R, 256, 8>(p, stream);
}

}  // namespace

hipError_t launch_block_norm(const BlockNormLaunch& p, hipStream_t stream) {
  if (p.rows == 0 || p.width == 0 || p.width > kNormMaxWidth) return hipErrorInvalidValue;
  if (p.act_dtype == 0)
    return p.residual_dtype == 0 ? block_norm_rows<ActBF16, ActBF16>(p, stream) : block_norm_rows<ActBF16, ActF32>(p, stream);
  return p.residual_dtype == 0 ? block_norm_rows<ActF32, ActBF16>(p, stream) : block_norm_rows<ActF32, ActF32>(p, stream);
}

}  // namespace vm
