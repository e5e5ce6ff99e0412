// The linear layer's kernels for bf16 operands (linear_kernels.h).
#include "linear_kernels.h"

namespace fwdmi {

int run_product_bf16(Product& P, int layouts, const Plan& plan, bool direct, hipStream_t stream) {
  return run_product<__bf16>(P, layouts, plan, direct, stream);
}
int run_gradients_bf16(const Gradients& G, bool direct, hipStream_t stream) { return run_gradients<__bf16>(G, direct, stream); }
int run_slope_bf16(const Slope& S, int parts, hipStream_t stream) { return run_slope<__bf16>(S, parts, stream); }

}  // namespace fwdmi
