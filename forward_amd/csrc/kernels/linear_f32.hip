// The linear layer's kernels for fp32 operands (linear_kernels.h).
#include "linear_kernels.h"

namespace fwdmi {

int run_product_f32(Product& P, int layouts, const Plan& plan, bool direct, hipStream_t stream) {
  return run_product<float>(P, layouts, plan, direct, stream);
}
int run_gradients_f32(const Gradients& G, bool direct, hipStream_t stream) { return run_gradients<float>(G, direct, stream); }
int run_slope_f32(const Slope& S, int parts, hipStream_t stream) { return run_slope<float>(S, parts, stream); }

}  // namespace fwdmi
