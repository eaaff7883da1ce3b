// Matrix products with an epilogue (vm_linear.h): bf16 operands, and the call itself.

#include "vm_linear.h"

namespace vm {

hipError_t launch_linear_mx(const LinearLaunch& p, hipStream_t stream);   // linear_mx.hip

// Of 64 x 64 tiles; smaller ones are chosen where there are few.
uint64_t linear_blocks(uint32_t rows, uint32_t n) { return (uint64_t(rows) + 63) / 64 * ((uint64_t(n) + 31) / 32); }

hipError_t launch_linear(const LinearLaunch& p, hipStream_t stream) {
  if (p.rows == 0 || p.n == 0 || p.k_bytes == 0) return hipErrorInvalidValue;
  return p.mx ? launch_linear_mx(p, stream) : linear_go<false>(p, stream);
}

}  // namespace vm
