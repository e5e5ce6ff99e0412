// The linear layer's kernels for fp16 operands (linear_kernels.h).
#include "linear_kernels.h"

namespace fwdmi {
namespace {

// Bound by memory, a read and a write: 4099 x 1531 and 4096 x 1531 (50 MB in all) take 11 us, and the product behind them then loads
// directly.  Eight elements per lane; an element past the line's end becomes a zero.
__global__ __launch_bounds__(256) void widen_kernel(const Widen W) {
  const uint32_t which = blockIdx.y, per = W.ld_out / 8;
  const uint32_t q = blockIdx.x * 256 + threadIdx.x;  // (a launch holds fewer than 2^32 lanes)
  const int64_t line = q / per;
  if (line >= W.lines[which]) return;
  const int c = (int)(q % per) * 8;
  const uint16_t FWDMI_GLOBAL* const p = gconst<uint16_t>(W.in[which]) + line * W.ld + c;
  Pack<uint16_t, 8> v;
  if (c + 8 <= W.ld) {
    v = load_slice<uint16_t, 8>(p);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v.v[e] = c + e < W.ld ? p[e] : (uint16_t)0;
  }
  store_slice<uint16_t, 8>(gmut<uint16_t>(W.out[which]) + line * W.ld_out + c, v);
}

}  // namespace

int run_widen(const Widen& W, hipStream_t stream) {
  const int64_t most = std::max(W.lines[0], W.lines[1]) * (W.ld_out / 8);
  if (const int rc = check_launch((most + 255) / 256 * 2, 256)) return rc;
  const dim3 grid((unsigned)ceil_div(most, 256), W.in[1] ? 2 : 1);
  hipLaunchKernelGGL(widen_kernel, grid, dim3(256), 0, stream, W);
  FWDMI_HIP_CHECK(hipGetLastError());
  return FWDMI_OK;
}

int run_product_f16(Product& P, int layouts, const Plan& plan, bool direct, hipStream_t stream) {
  return run_product<_Float16>(P, layouts, plan, direct, stream);
}
int run_gradients_f16(const Gradients& G, bool direct, hipStream_t stream) { return run_gradients<_Float16>(G, direct, stream); }
int run_slope_f16(const Slope& S, int parts, hipStream_t stream) { return run_slope<_Float16>(S, parts, stream); }

}  // namespace fwdmi
