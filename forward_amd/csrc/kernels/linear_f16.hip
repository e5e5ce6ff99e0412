// The linear layer's kernels for fp16 operands (linear_kernels.h).
#include "linear_kernels.h"

namespace fwdmi {

int run_product_f16(Product& P, int layouts, const Plan& plan, bool direct, hipStream_t stream) {
  return run_product<_Float16>(P, layouts, plan, direct, stream);
}
int run_slope_f16(const Slope& S, int parts, hipStream_t stream) { return run_slope<_Float16>(S, parts, stream); }

}  // namespace fwdmi
