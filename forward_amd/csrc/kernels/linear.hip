// Entry points of the linear layer and its gradient: argument checks, plans, workspaces.  The kernels are in
// linear_kernels.h.
#include <hip/hip_runtime.h>

#include "linear_plan.h"
#include "slice.h"

namespace fwdmi {
namespace {

// What bounds a product's operands: the layouts (0 both along t, 1 a along and b across, 2 both across), whether they
// may be loaded directly and, if so, how the end of t is (through registers: kTail).
struct Operands {
  int layouts, elem;
  bool direct;
  End end;
};

// The tile and the number of splits of t with the shortest estimated time.  A CU's time is its workgroups' steps: each as
// long as its loads (direct ones reach 90 KB/us per CU, those through registers 40) or its matrix instructions take
// (kRate: flop/us per CU that the steps of each tile sustain in bf16, by layout; in fp32 kStep32, per workgroup when a CU has one and when it has several), plus what a round of tiles spends
// outside its steps and, with splits, the second launch and the partial products' way through the caches.  Measured, us:
//   bf16  8192 x 4096 x 1024                  64 with 256 x 256, 74 with 256 x 128, 84 with 128 x 128
//         8192 x 1024 x 4096, b across        66 with 256 x 128, 81 with 128 x 128
//         4096 x 1024 x 8192, both across     63 + 13 to add the splits with 256 x 256 and four, 72 + 9 with 256 x 128 and two
//         4096 x 1024 x 4096                  42 with 128 x 128 in turns, 45 with four waves, 48 with 256 x 128 on half the CUs
//         the same, b across or both          52 with 128 x 128 in turns, 63 with four waves, 58 with 64 x 64
//         1024 x 1024 x 4096                  15 with 64 x 64 and three buffers, 23 with two
//         the same, b across or both          22 and 24 with 64 x 64 and steps of 512 bytes, 27 with 256 and two or three buffers
//         512 x 1024 x 4096                   10 with 64 x 32, 13 with 32 x 32, 18 with 48 x 32 (two workgroups on some CUs)
//         384 x 1024 x 4096                   10 with 48 x 32, 11 with 64 x 32, 14 with 32 x 32, 15 with 64 x 64
//         256 x 1024 x 4096                   8 with 32 x 32, 9 with 48 x 32, 10 with 64 x 32
//   fp32  512 x 512 x 512                     7 with 32 x 32, 9 with 64 x 32, 13 with 64 x 64
//         1003 x 517 x 1024                   15 with 48 x 48, 20 with 32 x 32, 23 with 64 x 64
//         256 x 1024 x 4096                   26 with 64 x 64 and four splits, 27 with 32 x 32 and two, 48 with 32 x 32 alone
//         768 x 768 x 768                     13 with 48 x 48, 16 with 32 x 32, 17 with 64 x 64
//         1024 x 1024 x 1024                  23 with 64 x 64 and steps of 512 bytes, 24 with 256
//         100 x 1024 x 1024                   9 with 32 x 32 and steps of 512 bytes, 10 with 256
const double kRate[3][kTileKinds] = {{6.0e6, 4.6e6, 3.7e6, 3.5e6, 4.0e6, 3.5e6, 3.0e6, 0, 3.0e6, 2.0e6, 0},
                                     {6.0e6, 4.6e6, 2.9e6, 1.9e6, 3.7e6, 3.0e6, 1.4e6, 0, 0, 0.9e6, 0},
                                     {6.0e6, 4.3e6, 2.9e6, 1.8e6, 2.2e6, 2.8e6, 1.4e6, 0, 0, 0.8e6, 0}};
const double kStep32[2][kTileKinds] = {{0, 0, 0, 2.4, 2.2, 1.2, 0.8, 1.55, 0, 0.78, 0.5},
                                       {0, 0, 0, 2.4, 2.1, 1.15, 0.65, 1.6, 0, 0.78, 0.36}};
const double kRound[kTileKinds] = {9.0, 4.0, 3.0, 1.5, 3.0, 1.5, 1.0, 1.5, 1.0, 1.0, 1.0};

// Where a tile is offered, with `wgs` workgroups on the fullest CU.  Tiles that fill a CU's LDS with one workgroup's deep or
// many buffers replace those of which several fit a CU where there is no second one to fit.
bool offered(TileKind kind, const Operands& o, double wgs) {
  const bool half = o.elem == 2, alone = wgs <= 1;
  switch (kind) {
    case k256x256:
    case k256x128: return half && o.direct;
    case k128x128Turns: return half && o.direct && alone;
    case k64x64Alone: return o.direct && alone;
    case k128x128: return !(half && o.direct && alone);
    case k64x64: return !(o.direct && alone);
    case k48x48: return !half && o.direct && o.layouts == 0;
    case k48x32: return half && o.direct && o.layouts == 0;
    case k32x32Deep: return o.direct && (half || alone);
    case k32x32: return !half && !(o.direct && alone);
    default: return true;
  }
}

// One step of each of `wgs` workgroups on a CU.
double step_us(TileKind kind, const Operands& o, double wgs) {
  const TileShape t = kTiles[kind];
  const int bytes = step_bytes(kind, o.layouts, o.elem, o.direct);
  const double load = wgs * (t.ti + t.tj) * bytes / ((o.direct ? 90.0 : 40.0) * 1024);
  if (o.elem == 4) return std::max(load, std::max(kStep32[0][kind], wgs * kStep32[1][kind]));
  return std::max(load, wgs * 2.0 * t.ti * t.tj * (bytes / 2) / kRate[o.layouts][kind]);
}
// A few rows: whole rows of w per workgroup, unless there are so few workgroups and so long rows that a second launch to
// add splits costs less than it gains.  A CU draws w and x at 38 KB/us through registers: 16 x 4096 x 1024 fp32 takes 16 us
// on 64 CUs, 9 with four splits and their sum.  No tile competes with it up to 32 rows, which is right where w has enough
// rows (replayed from a graph, 32 x 4096 x 1024 fp16 5.0 us, 33 rows in tiles 4.3; one row 3.4) and not where w has few: 32 x
// 1024 x 4096 fp16 12.8 us, 33 rows in tiles 7.9, one row 6.5; fp32 10.7, 12.4 and 6.9.
Plan few_plan(int ni, int nj, int nt, int elem) {
  const int pieces = nt / (128 / elem), wgs = ceil_div(nj, 16);
  const double us = (16.0 + (ni <= 16 ? 16 : 32)) * nt * elem / (38.0 * 1024);
  int splits = 1;
  if (us > 11.0) splits = std::max(1, std::min(std::min(8, device_cus() / wgs), pieces / 16));
  const int per = std::max(1, ceil_div(pieces, splits));
  return Plan{kFew, std::max(1, ceil_div(pieces, per)), 0, 0, per, us};
}

Plan make_plan(int ni, int nj, int nt, const Operands& o) {
  if (o.layouts == 0 && ni <= kFewRows) return few_plan(ni, nj, nt, o.elem);
  // (a call plans up to ten times before its launch: few divisions, none of 64 bits in the common case)
  const int cus = device_cus();
  Plan best{};
  best.us = 1e30;
  for (int i = 0; i < kTileKinds; ++i) {
    const TileKind kind = (TileKind)i;
    if (!offered(kind, o, 1.0) && !offered(kind, o, 2.0)) continue;
    const TileShape t = kTiles[kind];
    const int depth = step_bytes(kind, o.layouts, o.elem, o.direct) / o.elem;
    const int all = (int)(((unsigned)nt + (unsigned)depth - 1) >> __builtin_ctz(depth));  // steps, whatever their end
    const int64_t tiles = (int64_t)(((unsigned)ni + t.ti - 1) / (unsigned)t.ti) * (((unsigned)nj + t.tj - 1) / (unsigned)t.tj);
    for (int target = 0; target <= 2; ++target) {  // one workgroup per tile, or splits for one or two per CU
      int splits = 1, per = std::max(1, all);
      if (target > 0) {
        if (tiles * 2 > (int64_t)target * cus) continue;
        const int want = std::min(target * cus / (int)tiles, all / 2);
        if (want < 2) continue;
        per = (all + want - 1) / want;
        splits = (all + per - 1) / per;
      }
      const int64_t total = tiles * splits;
      const double wgs = total <= cus ? 1 : ceil_div(total, cus);
      if (!offered(kind, o, wgs)) continue;
      double us = 2.0 + wgs * kRound[kind] + per * step_us(kind, o, wgs);
      if (splits > 1) us += 3.0 + 6.0 * splits * ni * nj / 5.0e6;
      if (us < best.us) best = Plan{kind, splits, 0, 0, per, us};
    }
  }
  tail_of(nt, step_bytes(best.tile, o.layouts, o.elem, o.direct) / o.elem, o.end, best.whole_steps, best.tail);
  return best;
}

size_t partial_bytes(const Plan& p, int ni, int nj) {
  return p.splits > 1 ? (size_t)p.splits * ni * nj * sizeof(float) : 0;
}

End end_of(int layouts, int ni, int nj, int nt, int64_t lda, int64_t ldb, int elem) {
  const int chunk = 16 / elem;
  // (lines longer than their contents are copies made here, with zeros behind)
  auto part = [&](int n, int64_t ld) { return n % chunk != 0 && ld < (int64_t)ceil_div(n, chunk) * chunk; };
  if ((layouts == 2 && part(ni, lda)) || (layouts >= 1 && part(nj, ldb))) return kTailLine;
  return (layouts <= 1 && part(nt, lda)) || (layouts == 0 && part(nt, ldb)) ? kTail : kWhole;
}

Operands operands_of(const Product& P, int layouts, int elem) {
  const bool direct = direct_ok(P.a, P.lda, elem) && direct_ok(P.b, P.ldb, elem);
  return Operands{layouts, elem, direct, direct ? end_of(layouts, P.ni, P.nj, P.nt, P.lda, P.ldb, elem) : kTail};
}

int elem_size(int dtype) { return dtype == FWDMI_F32 ? 4 : 2; }

int run(Product& P, int layouts, int dtype, void* workspace, hipStream_t stream) {
  const Operands o = operands_of(P, layouts, elem_size(dtype));
  const Plan plan = make_plan(P.ni, P.nj, P.nt, o);
  P.partial = plan.splits > 1 ? static_cast<float*>(workspace) : nullptr;
  return dtype == FWDMI_F16    ? run_product_f16(P, layouts, plan, o.direct, stream)
         : dtype == FWDMI_BF16 ? run_product_bf16(P, layouts, plan, o.direct, stream)
                               : run_product_f32(P, layouts, plan, o.direct, stream);
}

// Whether the launches that `run` would make hold this product (asked for where a call makes several, before the first).
int check_product(const Product& P, int layouts, int dtype) {
  constexpr int kMost = 512;  // work-items of a workgroup; the smallest tile is 32 x 32, and what is split has few tiles
  if (launchable(((int64_t)P.ni + 31) / 32 * (((int64_t)P.nj + 31) / 32), kMost)) return FWDMI_OK;
  const Plan plan = make_plan(P.ni, P.nj, P.nt, operands_of(P, layouts, elem_size(dtype)));
  const TileShape t = kTiles[plan.tile];
  return check_launch((int64_t)ceil_div(P.ni, t.ti) * ceil_div(P.nj, t.tj) * plan.splits, kMost);
}

// Fills in P as one unsplit pass over tiles of `kind`; returns the number of tiles.
int64_t whole_tiles(Product& P, TileKind kind, const Operands& o) {
  const TileShape t = kTiles[kind];
  tail_of(P.nt, step_bytes(kind, o.layouts, o.elem, o.direct) / o.elem, o.end, P.whole_steps, P.tail);
  P.steps_per_split = P.whole_steps + (P.tail > 0);
  P.tiles_i = ceil_div(P.ni, t.ti);
  P.tiles_j = ceil_div(P.nj, t.tj);
  return (int64_t)P.tiles_i * P.tiles_j;
}

// Whether both products of a gradient are faster in one launch of unsplit tiles than in launches of their own (whose gap
// is about 3 us), and if so that launch, but for dbias.  771 x 1011 x 768 fp16: 12 us together, 10 and 8 us apart.  (Tiles of
// both and the columns of dbias that one launch cannot hold stay apart, where each product may still fit.)
bool together(const Product& x, const Product& w, int dtype, Gradients& G, bool& direct) {
  const int elem = elem_size(dtype), cus = device_cus();
  Operands ox = operands_of(x, 1, elem), ow = operands_of(w, 2, elem);
  double best = make_plan(x.ni, x.nj, x.nt, ox).us + make_plan(w.ni, w.nj, w.nt, ow).us + 3.0;
  direct = ox.direct && ow.direct;
  if (!direct) {
    ox.direct = ow.direct = false;
    ox.end = ow.end = kTail;
  }
  bool found = false;
  for (TileKind kind : {k64x64, k32x32}) {
    if (kind == k32x32 && elem == 2) break;
    Product px = x, pw = w;
    const int64_t tx = whole_tiles(px, kind, ox), tw = whole_tiles(pw, kind, ow);
    if (!launchable(tx + tw + ceil_div(w.ni, 64), kTiles[kind].ti * 8)) continue;
    const int sx = px.steps_per_split, sw = pw.steps_per_split;
    const double wgs = ceil_div(tx + tw, cus), mean = ((double)tx * sx + (double)tw * sw) / (double)(tx + tw);
    const double us = 2.0 + wgs * kRound[kind] +
                      std::max(std::max(sx, sw) * step_us(kind, ow, 1.0), mean * step_us(kind, ow, wgs));
    if (us < best) {
      best = us;
      found = true;
      G.x = px;
      G.w = pw;
      G.tile = kind;
      G.blocks_x = (int)tx;
      G.blocks_w = (int)tw;
    }
  }
  return found;
}

// Partial products of any plan that `run` may choose for these sizes: that depends on the operands' alignment too, but not
// on how the end of t is loaded.
size_t product_bytes(int layouts, int64_t ni, int64_t nj, int64_t nt, int elem) {
  size_t bytes = 0;
  for (const Operands& o : {Operands{layouts, elem, true, kWhole}, Operands{layouts, elem, false, kTail}})
    bytes = std::max(bytes, partial_bytes(make_plan((int)ni, (int)nj, (int)nt, o), (int)ni, (int)nj));
  return bytes;
}

size_t align256(size_t v) { return (v + 255) / 256 * 256; }
int64_t widened(int64_t ld) { return (ld + 7) / 8 * 8; }

// Lines of an odd number of 16-bit elements cannot be loaded directly.  Where copies with whole lines cost less than
// direct loads gain (an estimate from the sizes alone, so that the workspace's size follows from them too), operands are
// copied first.  `us`: what the products are estimated to take through registers and directly.
bool widening_pays(int64_t ld, int elem, double lines, double registers_us, double direct_us) {
  if (elem != 2 || ld % 2 == 0) return false;
  return direct_us + 4.0 + lines * (double)ld * 2 * elem / 4.0e6 < registers_us;
}
bool widen_forward(int64_t m, int64_t n, int64_t k, int elem) {
  if (m <= kFewRows || elem != 2 || k % 2 == 0) return false;
  return widening_pays(k, elem, (double)(m + n), make_plan((int)m, (int)n, (int)k, Operands{0, elem, false, kTail}).us,
                       make_plan((int)m, (int)n, (int)k, Operands{0, elem, true, kWhole}).us);
}
bool widen_backward(int64_t m, int64_t n, int64_t k, int elem) {
  if (elem != 2 || k % 2 == 0) return false;
  auto both = [&](bool direct) {
    return make_plan((int)m, (int)k, (int)n, Operands{1, elem, direct, direct ? kWhole : kTail}).us +
           make_plan((int)n, (int)k, (int)m, Operands{2, elem, direct, direct ? kWhole : kTail}).us;
  };
  return widening_pays(k, elem, (double)(m + n), both(false), both(true));
}

constexpr int64_t kMaxDim = (int64_t)1 << 30;   // of each of m, n, k, and of their products in pairs: tile numbers and
constexpr double kMaxPlane = 1099511627776.0;   // launch sizes stay in 31 bits
bool dims_ok(int64_t m, int64_t n, int64_t k) {
  return m >= 0 && n >= 0 && k >= 0 && m <= kMaxDim && n <= kMaxDim && k <= kMaxDim && (double)m * n <= kMaxPlane &&
         (double)m * k <= kMaxPlane && (double)n * k <= kMaxPlane;
}

int slope_parts(int64_t m, int64_t n) {
  const int64_t blocks = (n + 511) / 512;
  const int64_t want = std::max<int64_t>(1, 1024 / std::max<int64_t>(1, blocks));
  return (int)std::max<int64_t>(1, std::min<int64_t>((m + 3) / 4, std::min<int64_t>(want, 256)));
}

// Workspace of the forward pass: copies of x and w with whole lines, then the partial products.
struct ForwardSpace {
  size_t x, w, product;
  size_t total() const { return x + w + product; }
};
ForwardSpace forward_space(int64_t m, int64_t n, int64_t k, int dtype) {
  const int elem = elem_size(dtype);
  ForwardSpace s{0, 0, 0};
  if (m == 0 || n == 0) return s;
  if (widen_forward(m, n, k, elem)) {
    s.x = align256((size_t)m * widened(k) * elem);
    s.w = align256((size_t)n * widened(k) * elem);
  }
  s.product = product_bytes(0, m, n, k, elem);
  return s;
}

// Workspace of the backward pass: dz (with an activation, or where dy's lines are odd), its column sums' partials, copies
// of x and w with whole lines, then the larger of the two products' partials.
struct BackwardSpace {
  size_t dz, part, x, w, product;
  int64_t ld_dz;
  size_t total() const { return dz + part + x + w + product; }
};
BackwardSpace backward_space(int64_t m, int64_t n, int64_t k, int act, int dtype) {
  const int elem = elem_size(dtype);
  BackwardSpace s{0, 0, 0, 0, 0, n};
  if (m == 0 || n == 0) return s;
  if (elem == 2 && n % 2 != 0) s.ld_dz = widened(n);
  if (act != FWDMI_ACT_NONE || s.ld_dz != n) s.dz = align256((size_t)m * s.ld_dz * elem);
  s.part = align256((size_t)slope_parts(m, n) * n * sizeof(float));
  if (k > 0) {
    if (widen_backward(m, n, k, elem)) {
      s.x = align256((size_t)m * widened(k) * elem);
      s.w = align256((size_t)n * widened(k) * elem);
    }
    s.product = std::max(product_bytes(1, m, k, n, elem), product_bytes(2, n, k, m, elem));
  }
  return s;
}

// What the forward product reads: x and w, or their copies with whole lines at the workspace's beginning.
Product forward_product(int64_t m, int64_t n, int64_t k, const ForwardSpace& space, const void* x, const void* w, char* ws) {
  Product P{};
  P.a = space.x ? ws : x;
  P.b = space.x ? ws + space.x : w;
  P.lda = P.ldb = space.x ? widened(k) : k;
  P.ni = (int)m;
  P.nj = (int)n;
  P.nt = (int)k;
  return P;
}

// What the gradient's products read: dz or dy, and x and w or their copies with whole lines behind dz and its partials.
void backward_products(int64_t m, int64_t n, int64_t k, const BackwardSpace& space, const void* dy, const void* x,
                       const void* w, char* ws, bool copy, bool widen, Product& X, Product& W) {
  char* const wide = ws + space.dz + space.part;
  X.a = W.a = copy ? ws : dy;
  X.lda = W.lda = space.ld_dz;
  X.b = widen ? wide + space.x : w;
  W.b = widen ? wide : x;
  X.ldb = W.ldb = widen ? widened(k) : k;
  X.ni = W.nt = (int)m;
  X.nt = W.ni = (int)n;
  X.nj = W.nj = (int)k;
}

}  // namespace
}  // namespace fwdmi

extern "C" {

size_t fwdmi_linear_workspace(int64_t m, int64_t n, int64_t k, int32_t dtype) {
  using namespace fwdmi;
  if (!is_train_dtype(dtype) || !dims_ok(m, n, k) || m == 0 || n == 0) return 0;
  return forward_space(m, n, k, dtype).total();
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
  const ForwardSpace space = forward_space(m, n, k, dtype);
  FWDMI_REQUIRE(space.total() == 0 || (workspace && workspace_size >= space.total() &&
                                       reinterpret_cast<uintptr_t>(workspace) % 16 == 0),
                "linear: workspace of %zu bytes, %zu needed", workspace ? workspace_size : (size_t)0, space.total());
  hipStream_t s = static_cast<hipStream_t>(stream);
  char* const ws = static_cast<char*>(workspace);
  if (space.x) {
    const int rc = run_widen(Widen{{x, w}, {ws, ws + space.x}, {m, n}, (int)k, (int)widened(k)}, s);
    if (rc != FWDMI_OK) return rc;
  }
  Product P = forward_product(m, n, k, space, x, w, ws);
  P.c = y;
  P.preact = preact;
  P.bias = bias;
  P.residual = residual;
  P.act = act;
  return run(P, 0, dtype, ws + space.x + space.w, s);
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
  float* const part = reinterpret_cast<float*>(ws + space.dz);
  char* const wide = ws + space.dz + space.part;
  void* const partial = wide + space.x + space.w;
  dx = m > 0 && k > 0 ? dx : nullptr;  // (n == 0 leaves zeros: an empty sum)
  dw = n > 0 && k > 0 ? dw : nullptr;  // (m == 0 likewise)
  const bool copy = space.dz && (dx || dw), widen = space.x && (dx || dw);
  Product X{}, W{};
  backward_products(m, n, k, space, dy, x, w, ws, copy, widen, X, W);
  X.c = dx;
  W.c = dw;
  Gradients G{};
  bool direct = false;
  const bool joint = any && dx && dw && together(X, W, dtype, G, direct);
  // few rows are summed straight from dy by the joint launch
  const bool sum_dy = joint && act == FWDMI_ACT_NONE && m <= 1024;
  int rc = FWDMI_OK;
  if (!joint) {  // (a joint launch is one that holds both)
    if (dx) rc = check_product(X, 1, dtype);
    if (dw && rc == FWDMI_OK) rc = check_product(W, 2, dtype);
    if (rc != FWDMI_OK) return rc;
  }
  if (copy && act == FWDMI_ACT_NONE && (sum_dy || !dbias)) {  // (a plain copy, 4 us for 771 x 1011; 5 with partial sums)
    rc = run_widen(Widen{{dy, nullptr}, {ws, nullptr}, {m, 0}, (int)n, (int)space.ld_dz}, s);
    if (rc != FWDMI_OK) return rc;
  } else if (any && (copy || (dbias && !sum_dy))) {
    Slope S{};
    S.dy = dy;
    S.z = act != FWDMI_ACT_NONE ? preact : nullptr;
    S.dz = copy ? ws : nullptr;
    S.part = dbias ? part : nullptr;
    S.m = m;
    S.n = (int)n;
    S.ld_dz = (int)space.ld_dz;
    S.act = act;
    rc = dtype == FWDMI_F16    ? run_slope_f16(S, parts, s)
         : dtype == FWDMI_BF16 ? run_slope_bf16(S, parts, s)
                               : run_slope_f32(S, parts, s);
    if (rc != FWDMI_OK) return rc;
  }
  if (widen) {
    rc = dx && dw ? run_widen(Widen{{x, w}, {wide, wide + space.x}, {m, n}, (int)k, (int)widened(k)}, s)
         : dw     ? run_widen(Widen{{x, nullptr}, {wide, nullptr}, {m, 0}, (int)k, (int)widened(k)}, s)
                  : run_widen(Widen{{w, nullptr}, {wide + space.x, nullptr}, {n, 0}, (int)k, (int)widened(k)}, s);
    if (rc != FWDMI_OK) return rc;
  }
  if (joint) {
    G.dbias = dbias;
    G.part = sum_dy ? nullptr : part;
    G.dy = dy;
    G.parts = sum_dy ? m : parts;
    G.n = (int)n;
    return dtype == FWDMI_F16    ? run_gradients_f16(G, direct, s)
           : dtype == FWDMI_BF16 ? run_gradients_bf16(G, direct, s)
                                 : run_gradients_f32(G, direct, s);
  }
  if (dbias && n > 0) {
    ColumnSums C{};
    C.part = part;
    C.out[0] = dbias;
    C.parts = parts;
    C.ld = (int)n;
    C.kinds = 1;
    rc = launch_column_sums(C, s);
    if (rc != FWDMI_OK) return rc;
  }
  if (dx) {
    rc = run(X, 1, dtype, partial, s);
    if (rc != FWDMI_OK) return rc;
  }
  return dw ? run(W, 2, dtype, partial, s) : FWDMI_OK;
}

int fwdmi_linear_plan(int64_t m, int64_t n, int64_t k, int32_t what, int32_t act, int32_t dtype, int32_t on_boundary,
                      fwdmi_linear_plan_info* plan) {
  using namespace fwdmi;
  clear_error();
  if (!is_train_dtype(dtype)) return set_error(FWDMI_ERR_UNSUPPORTED, "linear plan: unsupported dtype %d", dtype);
  FWDMI_REQUIRE(plan && what >= 0 && what <= 3 && act >= FWDMI_ACT_NONE && act <= FWDMI_ACT_SILU, "linear plan: null plan, or unknown product %d or activation %d", what, act);
  FWDMI_REQUIRE(dims_ok(m, n, k) && m > 0 && n > 0 && k > 0, "linear plan: m=%lld n=%lld k=%lld", (long long)m, (long long)n,
                (long long)k);
  *plan = fwdmi_linear_plan_info{};
  // (addresses that are looked at and never read: on a boundary, or one element past it)
  const int elem = elem_size(dtype);
  char* const ws = reinterpret_cast<char*>((uintptr_t)1 << 20);
  const char* const at = ws + (on_boundary ? 0 : elem);
  Plan p{};
  Operands o{};
  if (what == 0) {
    const Product P = forward_product(m, n, k, forward_space(m, n, k, dtype), at, at, ws);
    o = operands_of(P, 0, elem);
    p = make_plan(P.ni, P.nj, P.nt, o);
  } else {
    const BackwardSpace space = backward_space(m, n, k, act, dtype);
    Product X{}, W{};
    backward_products(m, n, k, space, at, at, at, ws, space.dz != 0, space.x != 0, X, W);
    if (what == 3) {
      Gradients G{};
      if (!together(X, W, dtype, G, o.direct)) return FWDMI_OK;  // (zeros: each product in a launch of its own)
      p.tile = G.tile;
      p.splits = 1;
      o.end = o.direct ? std::max(operands_of(X, 1, elem).end, operands_of(W, 2, elem).end) : kTail;
    } else {
      const Product& P = what == 1 ? X : W;
      o = operands_of(P, what, elem);
      p = make_plan(P.ni, P.nj, P.nt, o);
    }
  }
  plan->tile = p.tile;
  plan->tile_rows = p.tile == kFew ? (m <= 16 ? 16 : kFewRows) : kTiles[p.tile].ti;
  plan->tile_columns = p.tile == kFew ? 16 : kTiles[p.tile].tj;
  plan->splits = p.splits;
  plan->direct = p.tile != kFew && o.direct;
  plan->end = p.tile == kFew ? 0 : o.end;
  return FWDMI_OK;
}

}  // extern "C"
