// Matrix products with an epilogue (vm_linear.h): MX operands.

#include "vm_linear.h"

namespace vm {

hipError_t launch_linear_mx(const LinearLaunch& p, const LinearForm& form, hipStream_t stream) {
  return linear_go<true>(form, p, stream);
}

}  // namespace vm
