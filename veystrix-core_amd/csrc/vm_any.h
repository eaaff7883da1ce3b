// Runs of values at any alignment of their type: one load or store of the vector memory unit, which takes any address,
// where the run lies within its row, value by value at a row's end.
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

#include "vm_common.h"

namespace vm {

typedef uint32_t words4 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t words2 __attribute__((ext_vector_type(2), aligned(2)));
template <uint32_t N>
using Words = std::conditional_t<N == 4, words4, words2>;

// N (4 or 8) neighbouring values of one row from `at`; those at `width` and behind it are zero.
template <uint32_t N>
__device__ __forceinline__ void load_run(const void* row, uint32_t dtype, uint32_t at, uint32_t width, float v[N]) {
  if (at + N > width) {
#pragma unroll
    for (uint32_t j = 0; j < N; ++j) v[j] = at + j < width ? load_any(row, at + j, dtype) : 0.0f;
  } else if (dtype == 0) {
    const Words<N / 2> a = *(const __attribute__((address_space(1))) Words<N / 2>*)(static_cast<const uint16_t*>(row) + at);
#pragma unroll
    for (uint32_t j = 0; j < N / 2; ++j) {
      v[2 * j] = __uint_as_float(a[j] << 16);
      v[2 * j + 1] = __uint_as_float(a[j] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (uint32_t j = 0; j < N; j += 4) {
      const Words<4> a = *(const __attribute__((address_space(1))) Words<4>*)(static_cast<const float*>(row) + at + j);
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) v[j + i] = __uint_as_float(a[i]);
    }
  }
}

template <uint32_t N>
__device__ __forceinline__ void store_run(void* row, uint32_t dtype, uint32_t at, uint32_t width, const float v[N]) {
  if (at + N > width) {
#pragma unroll
    for (uint32_t j = 0; j < N; ++j) {
      if (at + j >= width) continue;
      if (dtype == 0) ActBF16::store(row, at + j, v[j]);
      else ActF32::store(row, at + j, v[j]);
    }
  } else if (dtype == 0) {
    Words<N / 2> a;
#pragma unroll
    for (uint32_t j = 0; j < N / 2; ++j) a[j] = f32_to_bf16(v[2 * j]) | (f32_to_bf16(v[2 * j + 1]) << 16);
    *(__attribute__((address_space(1))) Words<N / 2>*)(static_cast<uint16_t*>(row) + at) = a;
  } else {
#pragma unroll
    for (uint32_t j = 0; j < N; j += 4) {
      Words<4> a;
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) a[i] = __float_as_uint(v[j + i]);
      *(__attribute__((address_space(1))) Words<4>*)(static_cast<float*>(row) + at + j) = a;
    }
  }
}

}  // namespace vm
