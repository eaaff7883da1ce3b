// What the products share: MFMA operands of bf16 or MX units, and SwiGLU.
#pragma once

#include <hip/hip_runtime.h>

#include "vm_common.h"

namespace vm {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

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

}  // namespace vm
