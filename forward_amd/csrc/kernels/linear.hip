// Entry points of the linear layer and its gradient: argument checks, plans, workspaces.  The kernels are in
// linear_kernels.h.
#include <hip/hip_runtime.h>

#include "linear_plan.h"
#include "slice.h"

namespace fwdmi {
namespace {

// The tile whose launch fills the CUs best, and how many splits of t it takes to do so when the tiles are few.
Plan make_plan(int ni, int nj, int nt, int elem, bool direct) {
  const int cus = device_cus();
  const int all = ceil_div(nt, kStepBytes / elem);
  Plan p{kSmall, 64, 64, 1, all};
  if (elem == 2 && direct && (int64_t)ceil_div(ni, 256) * ceil_div(nj, 256) >= cus * 3 / 4)
    p = Plan{kBig, 256, 256, 1, all};
  else if ((int64_t)ceil_div(ni, 128) * ceil_div(nj, 128) >= cus * 3 / 4)
    p = Plan{kMid, 128, 128, 1, all};
  const int64_t tiles = (int64_t)ceil_div(ni, p.ti) * ceil_div(nj, p.tj);
  if (tiles < cus && all > 1) {
    // at least four steps each, so that a split is worth its partial tile
    int splits = (int)std::min<int64_t>((2 * cus + tiles - 1) / tiles, std::max(1, all / 4));
    p.steps_per_split = ceil_div(all, splits);
    p.splits = ceil_div(all, p.steps_per_split);
  }
  return p;
}

size_t partial_bytes(const Plan& p, int ni, int nj) {
  return p.splits > 1 ? (size_t)p.splits * ni * nj * sizeof(float) : 0;
}

int run(Product& P, int layouts, int dtype, void* workspace, hipStream_t stream) {
  const int elem = dtype == FWDMI_F32 ? 4 : 2;
  const bool direct = direct_ok(P.a, P.lda, elem, layouts == 2 ? P.ni : P.nt) &&
                      direct_ok(P.b, P.ldb, elem, layouts == 0 ? P.nt : P.nj);
  const Plan plan = make_plan(P.ni, P.nj, P.nt, elem, direct);
  P.partial = plan.splits > 1 ? static_cast<float*>(workspace) : nullptr;
  return dtype == FWDMI_F16    ? run_product_f16(P, layouts, plan, direct, stream)
         : dtype == FWDMI_BF16 ? run_product_bf16(P, layouts, plan, direct, stream)
                               : run_product_f32(P, layouts, plan, direct, stream);
}

// Partial products of either plan (which of the two runs depends on the operands' alignment).
size_t product_bytes(int64_t ni, int64_t nj, int64_t nt, int elem) {
  return std::max(partial_bytes(make_plan((int)ni, (int)nj, (int)nt, elem, true), (int)ni, (int)nj),
                  partial_bytes(make_plan((int)ni, (int)nj, (int)nt, elem, false), (int)ni, (int)nj));
}

int elem_size(int dtype) { return dtype == FWDMI_F32 ? 4 : 2; }
size_t align256(size_t v) { return (v + 255) / 256 * 256; }

constexpr int64_t kMaxDim = (int64_t)1 << 30;  // of each of m, n, k: tile numbers and row ends stay in 31 bits
bool dims_ok(int64_t m, int64_t n, int64_t k) {
  return m >= 0 && n >= 0 && k >= 0 && m <= kMaxDim && n <= kMaxDim && k <= kMaxDim;
}

int slope_parts(int64_t m, int64_t n) {
  const int64_t blocks = (n + 511) / 512;
  const int64_t want = std::max<int64_t>(1, 1024 / std::max<int64_t>(1, blocks));
  return (int)std::max<int64_t>(1, std::min<int64_t>((m + 3) / 4, std::min<int64_t>(want, 256)));
}

// Workspace of the backward pass: dz, its column sums' partials, then the larger of the two products' partials.
struct BackwardSpace {
  size_t dz, part, product;
  size_t total() const { return dz + part + product; }
};
BackwardSpace backward_space(int64_t m, int64_t n, int64_t k, int act, int dtype) {
  const int elem = elem_size(dtype);
  BackwardSpace s{0, 0, 0};
  if (m == 0 || n == 0) return s;
  if (act != FWDMI_ACT_NONE) s.dz = align256((size_t)m * n * elem);
  s.part = align256((size_t)slope_parts(m, n) * n * sizeof(float));
  if (k > 0)
    s.product = std::max(product_bytes(m, k, n, elem), product_bytes(n, k, m, elem));
  return s;
}

}  // namespace
}  // namespace fwdmi

extern "C" {

size_t fwdmi_linear_workspace(int64_t m, int64_t n, int64_t k, int32_t dtype) {
  using namespace fwdmi;
  if (!is_train_dtype(dtype) || !dims_ok(m, n, k) || m == 0 || n == 0) return 0;
  return product_bytes(m, n, k, elem_size(dtype));
}

int fwdmi_linear(void* stream, int64_t m, int64_t n, int64_t k, const void* x, const void* w, const float* bias,
                 const void* residual, void* y, void* preact, int32_t act, int32_t dtype, void* workspace,
                 size_t workspace_size) {
  using namespace fwdmi;
  clear_error();
  if (!is_train_dtype(dtype)) return set_error(FWDMI_ERR_UNSUPPORTED, "linear: unsupported dtype %d", dtype);
  FWDMI_REQUIRE(act >= FWDMI_ACT_NONE && act <= FWDMI_ACT_SILU, "linear: unknown activation %d", act);
  FWDMI_REQUIRE(dims_ok(m, n, k), "linear: m=%lld n=%lld k=%lld", (long long)m, (long long)n, (long long)k);
  if (m == 0 || n == 0) return FWDMI_OK;
  FWDMI_REQUIRE(y && (k == 0 || (x && w)), "linear: null pointer");
  const size_t need = fwdmi_linear_workspace(m, n, k, dtype);
  FWDMI_REQUIRE(need == 0 || (workspace && workspace_size >= need && reinterpret_cast<uintptr_t>(workspace) % 16 == 0),
                "linear: workspace of %zu bytes, %zu needed", workspace ? workspace_size : (size_t)0, need);
  Product P{};
  P.a = x;
  P.b = w;
  P.lda = P.ldb = k;
  P.ni = (int)m;
  P.nj = (int)n;
  P.nt = (int)k;
  P.c = y;
  P.preact = preact;
  P.bias = bias;
  P.residual = residual;
  P.act = act;
  return run(P, 0, dtype, workspace, static_cast<hipStream_t>(stream));
}

size_t fwdmi_linear_backward_workspace(int64_t m, int64_t n, int64_t k, int32_t act, int32_t dtype) {
  using namespace fwdmi;
  if (!is_train_dtype(dtype) || !dims_ok(m, n, k)) return 0;
  return backward_space(m, n, k, act, dtype).total();
}

int fwdmi_linear_backward(void* stream, int64_t m, int64_t n, int64_t k, const void* dy, const void* x, const void* w,
                          const void* preact, void* dx, void* dw, float* dbias, int32_t act, int32_t dtype,
                          void* workspace, size_t workspace_size) {
  using namespace fwdmi;
  clear_error();
  if (!is_train_dtype(dtype)) return set_error(FWDMI_ERR_UNSUPPORTED, "linear backward: unsupported dtype %d", dtype);
  FWDMI_REQUIRE(act >= FWDMI_ACT_NONE && act <= FWDMI_ACT_SILU, "linear backward: unknown activation %d", act);
  FWDMI_REQUIRE(dims_ok(m, n, k), "linear backward: m=%lld n=%lld k=%lld", (long long)m, (long long)n, (long long)k);
  const bool any = m > 0 && n > 0;
  FWDMI_REQUIRE(!any || dy, "linear backward: null dy");
  FWDMI_REQUIRE(!any || act == FWDMI_ACT_NONE || preact, "linear backward: an activation needs its pre-activation");
  FWDMI_REQUIRE(!dx || !any || k == 0 || w, "linear backward: dx needs w");
  FWDMI_REQUIRE(!dw || !any || k == 0 || x, "linear backward: dw needs x");
  const BackwardSpace space = backward_space(m, n, k, act, dtype);
  FWDMI_REQUIRE(space.total() == 0 || (workspace && workspace_size >= space.total() &&
                                       reinterpret_cast<uintptr_t>(workspace) % 16 == 0),
                "linear backward: workspace of %zu bytes, %zu needed", workspace ? workspace_size : (size_t)0, space.total());
  hipStream_t s = static_cast<hipStream_t>(stream);
  char* const ws = static_cast<char*>(workspace);
  const int parts = any ? slope_parts(m, n) : 0;
  const void* dz = dy;
  int rc = FWDMI_OK;
  if (any && (act != FWDMI_ACT_NONE || dbias)) {
    Slope S{};
    S.dy = dy;
    if (act != FWDMI_ACT_NONE) {
      S.z = preact;
      S.dz = ws;
      dz = ws;
    }
    S.part = dbias ? reinterpret_cast<float*>(ws + space.dz) : nullptr;
    S.m = m;
    S.n = (int)n;
    S.act = act;
    rc = dtype == FWDMI_F16    ? run_slope_f16(S, parts, s)
         : dtype == FWDMI_BF16 ? run_slope_bf16(S, parts, s)
                               : run_slope_f32(S, parts, s);
    if (rc != FWDMI_OK) return rc;
  }
  if (dbias && n > 0) {
    ColumnSums C{};
    C.part = reinterpret_cast<const float*>(ws + space.dz);
    C.out[0] = dbias;
    C.parts = parts;
    C.ld = (int)n;
    C.kinds = 1;
    rc = launch_column_sums(C, s);
    if (rc != FWDMI_OK) return rc;
  }
  void* const partial = ws + space.dz + space.part;
  Product P{};
  P.a = dz;
  P.lda = n;
  P.ldb = k;
  P.nj = (int)k;
  if (dx && m > 0 && k > 0) {  // (n == 0: an empty sum, zeros)
    P.b = w;
    P.ni = (int)m;
    P.nt = (int)n;
    P.c = dx;
    rc = run(P, 1, dtype, partial, s);
    if (rc != FWDMI_OK) return rc;
  }
  if (dw && n > 0 && k > 0) {
    P.b = x;
    P.ni = (int)n;
    P.nt = (int)m;
    P.c = dw;
    rc = run(P, 2, dtype, partial, s);
  }
  return rc;
}

}  // extern "C"
