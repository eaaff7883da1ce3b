// Matrix products with an epilogue (vm_linear.h): bf16 operands, and the call itself.

#include "vm_linear.h"

namespace vm {

hipError_t launch_linear_mx(const LinearLaunch& p, const LinearForm& form, hipStream_t stream);   // linear_mx.hip

LinearForm linear_form(const LinearLaunch& p) {
  const bool pairs = p.activation == kActSwiglu;
  // the large tiles' offsets are 32 bits from a tile's first row, the up rows of SwiGLU included
  const uint64_t rows = 512, up = pairs ? p.n : 0;
  const bool near = (rows + up) * p.w_stride + p.k_bytes < (1ull << 32) && rows * p.x_stride + p.k_bytes < (1ull << 32);
  return p.mx ? choose_form<true>(p.rows, p.n, p.k_bytes, pairs, near && p.whole_scales)
              : choose_form<false>(p.rows, p.n, p.k_bytes, pairs, near);
}

hipError_t launch_linear(const LinearLaunch& p, const LinearForm& form, hipStream_t stream) {
  if (p.rows == 0 || p.n == 0 || p.k_bytes == 0 || !form.fits()) return hipErrorInvalidValue;
  return p.mx ? launch_linear_mx(p, form, stream) : linear_go<false>(form, p, stream);
}

}  // namespace vm
