// What the norms of rows share: how a row's values lie over its threads, loads and stores of eight values, gains of
// 1 + weight and floats that are rounded once more to e4m3.
#pragma once

#include <hip/hip_runtime.h>

#include "vm_common.h"

namespace vm {

// How a thread's eight values of a step lie in a row: consecutive ones moved as 16-byte units or one by one, or spread
// over the row's threads, so that those moved one by one are neighbours across lanes (3000 rows of 3333 bf16 values and a
// residual 31 to 33 us, eight of them side by side 54; the bytes alone take 17 at a copy's rate, but every value is a load
// of its own, and eight steps of them hold so many registers that one wave runs per SIMD).
enum : int { kUnits = 0, kOnes = 1, kSpread = 2 };

// The eight values of the step at element `at`; those at `width` and behind it are zero.
template <class A, int LIE>
__device__ __forceinline__ void load8(const void* row, uint32_t at, uint32_t step, uint32_t width, float v[8]) {
  if constexpr (LIE == kUnits) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 0.0f;
    if (at >= width) return;
    const uint8_t* src = static_cast<const uint8_t*>(row) + static_cast<size_t>(at) * A::kBytes;
    const uint4 a = ldg16(src);
    if constexpr (A::kBytes == 2) {
      const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[2 * j] = __uint_as_float(w[j] << 16);
        v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
      }
    } else {
      const uint4 b = ldg16(src + 16);
      v[0] = __uint_as_float(a.x); v[1] = __uint_as_float(a.y); v[2] = __uint_as_float(a.z); v[3] = __uint_as_float(a.w);
      v[4] = __uint_as_float(b.x); v[5] = __uint_as_float(b.y); v[6] = __uint_as_float(b.z); v[7] = __uint_as_float(b.w);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {  // no branch: each would wait for its own load
      const uint32_t i = at + j * step;
      const float value = A::from_bits(A::load_bits(row, min(i, width - 1)));
      v[j] = i < width ? value : 0.0f;
    }
  }
}

template <class A, int LIE>
__device__ __forceinline__ void store8(void* row, uint32_t at, uint32_t step, uint32_t width, const float v[8]) {
  if constexpr (LIE == kUnits) {
    if (at >= width) return;
    if constexpr (A::kBytes == 2) {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = f32_to_bf16(v[2 * j]) | (f32_to_bf16(v[2 * j + 1]) << 16);
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(row) + at) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
      float4* dst = reinterpret_cast<float4*>(static_cast<float*>(row) + at);
      dst[0] = make_float4(v[0], v[1], v[2], v[3]);
      dst[1] = make_float4(v[4], v[5], v[6], v[7]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (at + j * step < width) A::store(row, at + j * step, v[j]);
  }
}

__device__ __forceinline__ float wave_total(float v) { return wave_sum_all(v); }
__device__ __forceinline__ double wave_total(double v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
  return v;
}

// 1 + w: the nearest float, and what it leaves.
__device__ __forceinline__ float one_plus(float w, float* rest) {
#pragma clang fp contract(off)
  const float g = 1.0f + w, part = g - 1.0f;
  *rest = (1.0f - (g - part)) + (w - part);
  return g;
}

// A float that is rounded once more, to e4m3, must not lie on a border there that the product itself does not lie on:
// one step towards it then.  Borders have the last 19 bits of a float clear.
constexpr uint32_t kBorderBits = 0x7ffffu;
__device__ __forceinline__ float off_border(float f, float off) {
  const uint32_t bits = __float_as_uint(f);
  const bool finite = (bits & 0x7fffffffu) - 0x0d000000u < 0x7f800000u - 0x0d000000u;  // and far above subnormals
  if ((bits & kBorderBits) != 0 || !finite || off == 0.0f) return f;
  return __uint_as_float((off < 0.0f) == (f < 0.0f) ? bits + 1 : bits - 1);
}

}  // namespace vm
