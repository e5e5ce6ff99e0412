"""linear / linear_backward on the GPU against their definitions in fp64.

Bounds (u = 2^-24, eps_T = torch.finfo(T).eps, a rounding to T is off by at most eps_T / 2 relative):
  products of two 16-bit operands are exact in fp32, of two fp32 ones rounded once; a sum over t of n products takes at
  most n additions, each off by at most one unit of its result (2u, matrix instructions are not said to round to nearest):
  |dz| <= (n + 8) 2u S with S the sum of the products' magnitudes (8: bias, the product's own rounding, the last splits).
  The activations' slopes are at most 1.13; their evaluation (a reciprocal, an exponential of 1 ulp, a polynomial whose
  error is 1.5e-7 of erf in 16-bit types) is off by at most 16u (|z| + |y|), the slope functions by 32u.
Where the operands are small whole numbers every sum is exact, and results have to be equal.
"""
import math

import pytest
import torch

from forward_amd import lib, ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = [torch.float32, torch.float16, torch.bfloat16]
ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]
# (m, n, k): single elements, rows that are no whole 16-byte lines, tile edges on every side, empty sums, long sums of
# few tiles (split), and enough tiles for each tile size
SHAPES = [(1, 1, 1), (1, 1, 4111), (1, 17, 5), (3, 64, 64), (5, 130, 72), (16, 24, 0), (64, 64, 64), (65, 63, 129), (128, 128, 8),
          (1, 1024, 2048), (9, 40, 9001), (30, 136, 8200), (7, 264, 4104), (200, 1000, 136), (257, 511, 1031), (1000, 517, 1001), (300, 4096, 1024),
          (250, 1000, 1034), (380, 1002, 520), (500, 1000, 2050), (900, 1026, 2050), (1000, 7, 8000), (1111, 2048, 72), (1931, 1930, 2042), (4000, 3336, 136)]


def half(dtype):
    return 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2


def check(got, want, bound, what):
    err = (got.double() - want).abs()
    worst = (err - bound).max().item() if err.numel() else 0.0
    assert not torch.isnan(err).any() and worst <= 0.0, "%s: %g past its bound" % (what, worst)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def make(m, n, k, dtype, seed, offset=0):
    g = gen(seed)

    def plane(rows, cols, std):
        t = torch.empty(rows * cols + offset, dtype=dtype, device="cuda")
        t.copy_(torch.randn(t.shape, generator=g, device="cuda") * std)
        return t[offset:].view(rows, cols)

    return dict(x=plane(m, k, 1.0), w=plane(n, k, 1.0 / math.sqrt(max(k, 1))), b=(torch.randn(n + offset, generator=g, device="cuda"))[offset:],
                r=plane(m, n, 1.0), dy=plane(m, n, 1.0))


def act64(z, name):
    if name == "relu":
        return z.clamp(min=0), (z > 0).double()
    if name == "gelu":
        p = torch.special.ndtr(z)
        return z * p, p + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        p = torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
        return z * p, p + z * p * (1 - p) * 2 * math.sqrt(2 / math.pi) * (1 + 0.134145 * z * z)
    if name == "silu":
        p = torch.sigmoid(z)
        return z * p, p + z * p * (1 - p)
    return z, torch.ones_like(z)


def check_linear(s, act, bias, residual, preact):
    x, w = s["x"], s["w"]
    k, e = x.shape[1], half(x.dtype)
    tiny = torch.finfo(x.dtype).tiny
    z = x.double() @ w.double().t()
    S = x.double().abs() @ w.double().abs().t()
    if bias:
        z, S = z + s["b"].double(), S + s["b"].double().abs()
    bz = (k + 8) * 2 * U * S
    a = act64(z, act)[0]
    y = a + (s["r"].double() if residual else 0.0)
    by = 1.13 * bz + 16 * U * (z.abs() + a.abs()) + 2 * U * y.abs()
    got = ops.linear(x, w, bias=s["b"] if bias else None, activation=act, residual=s["r"] if residual else None, want_preact=preact)
    if preact:
        got, gz = got
        check(gz, z, bz + e * (z.abs() + bz) + tiny, "preact")
    check(got, y, by + e * (y.abs() + by) + tiny, "y")
    return (got, gz) if preact else got


def check_backward(s, act, bias=True):
    x, w, dy = s["x"], s["w"], s["dy"]
    (m, k), n, e = x.shape, w.shape[0], half(x.dtype)
    tiny = torch.finfo(x.dtype).tiny
    z = s["r"] if act != "none" else None            # any values do as the pre-activation
    dz = dy.double() * (act64(z.double(), act)[1] if z is not None else 1.0)
    bdz = (32 * U * dy.double().abs() + e * dz.abs() + tiny) if z is not None else torch.zeros_like(dz)
    got = ops.linear_backward(dy, x, w, preact=z, activation=act, want_dbias=bias)
    A = dz.abs() + bdz
    dx, Sx = dz @ w.double(), A @ w.double().abs()
    bx = (n + 8) * 2 * U * Sx + bdz @ w.double().abs()
    check(got[0], dx, bx + e * (dx.abs() + bx) + tiny, "dx")
    dw, Sw = dz.t() @ x.double(), A.t() @ x.double().abs()
    bw = (m + 8) * 2 * U * Sw + bdz.t() @ x.double().abs()
    check(got[1], dw, bw + e * (dw.abs() + bw) + tiny, "dw")
    if bias:
        check(got[2], dz.sum(0), ((m + 8) * 2 * U * dz.abs() + 32 * U * dy.double().abs()).sum(0), "dbias")
    assert len(got) == (3 if bias else 2)
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_whole_numbers_are_exact(shape, dtype):
    m, n, k = shape
    g = gen(m + n + k)
    ints = lambda *s: torch.randint(-3, 4, s, generator=g, device="cuda").to(dtype)
    x, w, dy = ints(m, k), ints(n, k), ints(m, n)
    b = torch.randint(-3, 4, (n,), generator=g, device="cuda").float()
    r = ints(m, n)
    z = x.double() @ w.double().t() + b.double()
    y, gz = ops.linear(x, w, bias=b, activation="relu", residual=r, want_preact=True)
    # |sums| < 9 * 4104 + ...: exact in fp32, one rounding to the type
    assert torch.equal(gz, z.to(dtype)) and torch.equal(y, (z.clamp(min=0) + r.double()).to(dtype))
    dx, dw, db = ops.linear_backward(dy, x, w)
    assert torch.equal(dx, (dy.double() @ w.double()).to(dtype))
    assert torch.equal(dw, (dy.double().t() @ x.double()).to(dtype))
    assert torch.equal(db.double(), dy.double().sum(0))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_shapes(shape, dtype):
    m, n, k = shape
    s = make(m, n, k, dtype, m * 7 + n + k)
    check_linear(s, ACTS[(m + n) % 5], bias=n % 2 == 0, residual=m % 2 == 1, preact=k % 2 == 0)
    check_backward(s, ACTS[(m + k) % 5], bias=k % 2 == 0)


# (rows, columns, sum): each tile with one workgroup per CU and several, with the sum whole and split, and ends of a step; a
# line of more than 4 MiB; a sum of fewer elements than a load
PRODUCTS = [(36, 38, 36), (36, 38, 1962), (194, 1154, 36), (98, 332, 2934), (114, 334, 3916), (132, 2732, 38), (226, 424, 4272),
            (514, 1808, 46), (1154, 860, 2624), (200, 4222, 66), (2658, 3056, 38), (4828, 772, 38), (1306, 966, 4102), (2882, 2840, 138),
            (2380, 3382, 76), (800, 2840, 4842), (4892, 848, 3442), (36, 2097154, 36), (36, 38, 5), (194, 1154, 5), (132, 2732, 5), (660, 2990, 5)]


@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", PRODUCTS)
def test_each_product_alone(shape, dtype, offset):
    """y, dx and dw of these sizes, each in a call of its own; with the offset 16-bit operands go through registers."""
    ni, nj, nt = shape
    e, tiny, seed = half(dtype), torch.finfo(dtype).tiny, ni + nj + nt
    check_linear(make(ni, nj, nt, dtype, seed, offset), "silu", bias=True, residual=True, preact=True)
    s = make(ni, nt, nj, dtype, seed + 1, offset)
    dx, = ops.linear_backward(s["dy"], s["x"], s["w"], want_dweight=False, want_dbias=False)
    dy, w = s["dy"].double(), s["w"].double()
    want, bound = dy @ w, (nt + 8) * 2 * U * (dy.abs() @ w.abs())
    check(dx, want, bound + e * (want.abs() + bound) + tiny, "dx")
    s = make(nt, ni, nj, dtype, seed + 2, offset)
    dw, = ops.linear_backward(s["dy"], s["x"], s["w"], want_dx=False, want_dbias=False)
    dy, x = s["dy"].double().t(), s["x"].double()
    want, bound = dy @ x, (nt + 8) * 2 * U * (dy.abs() @ x.abs())
    check(dw, want, bound + e * (want.abs() + bound) + tiny, "dw")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ACTS)
def test_activations(act, dtype):
    s = make(130, 264, 64, dtype, 3)
    s["x"].mul_(4)                                    # pre-activations out to +-16
    s["r"].mul_(4)
    check_linear(s, act, bias=True, residual=True, preact=True)
    check_backward(s, act)
    s = make(9, 33, 4096, dtype, 4)                   # the same through split sums
    check_linear(s, act, bias=True, residual=False, preact=True)
    check_backward(s, act)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ACTS)
def test_far_pre_activations(act, dtype):
    """Where every activation is z or 0 and its slope 1 or 0, up to the ends of the type."""
    big = torch.finfo(dtype).max
    z = torch.tensor([[100.0, min(1e20, big), big, -100.0, -min(1e20, big), -big]], device="cuda").to(dtype)
    one, eye = torch.ones(1, 6, dtype=dtype, device="cuda"), torch.eye(6, dtype=dtype, device="cuda")
    want = torch.where((z > 0) | torch.tensor(act == "none", device="cuda"), z, torch.zeros_like(z))
    assert torch.equal(ops.linear(z, eye, activation=act), want)         # (products with zeros are exact)
    dx, _, db = ops.linear_backward(one, z, eye, preact=z if act != "none" else None, activation=act)
    slope = (want != 0).to(dtype)
    assert torch.equal(dx, slope) and torch.equal(db, slope.float()[0])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset", [1, 2, 3, 7])
def test_operands_start_at_any_element(offset, dtype):
    s = make(70, 136, 200, dtype, offset, offset=offset)
    check_linear(s, "gelu", bias=True, residual=True, preact=True)
    check_backward(s, "silu")


def test_leading_axes():
    g = gen(1)
    x = torch.randn(3, 5, 64, generator=g, device="cuda").half()
    w = torch.randn(40, 64, generator=g, device="cuda").half()
    y = ops.linear(x, w)
    assert y.shape == (3, 5, 40) and torch.equal(y.view(15, 40), ops.linear(x.view(15, 64), w))
    v = ops.linear(x[0, 0], w)
    assert v.shape == (40,)
    dy = torch.randn(3, 5, 40, generator=g, device="cuda").half()
    dx, dw, db = ops.linear_backward(dy, x, w)
    assert dx.shape == x.shape and dw.shape == w.shape and db.shape == (40,)
    assert torch.equal(ops.linear_backward(dy, x, w, want_dx=False, want_dbias=False)[0], dw)
    assert torch.equal(ops.linear_backward(dy, x, w, want_dweight=False)[0], dx)


@pytest.mark.parametrize("dtype", TYPES)
def test_empty_axes(dtype):
    z = lambda *s: torch.zeros(s, dtype=dtype, device="cuda")
    assert ops.linear(z(0, 8), z(4, 8)).shape == (0, 4)
    assert ops.linear(z(5, 8), z(0, 8)).shape == (5, 0)
    b = torch.tensor([1.0, -2.0, 3.0], device="cuda")
    assert torch.equal(ops.linear(z(2, 0), z(3, 0), bias=b, activation="relu").float(), b.clamp(min=0).expand(2, 3))
    dx, dw, db = ops.linear_backward(z(0, 4), z(0, 8), z(4, 8))
    assert dx.shape == (0, 8) and not dw.any() and not db.any()
    dx, dw, db = ops.linear_backward(z(5, 0), z(5, 8), z(0, 8))
    assert dx.shape == (5, 8) and not dx.any() and dw.shape == (0, 8) and db.shape == (0,)
    dx, dw, db = ops.linear_backward(z(5, 4) + 1, z(5, 0), z(4, 0))
    assert dx.shape == (5, 0) and dw.shape == (4, 0) and torch.equal(db, torch.full((4,), 5.0, device="cuda"))


@pytest.mark.parametrize("dtype", TYPES)
def test_nan_and_infinity_stay_in_their_rows(dtype):
    s = make(150, 200, 264, dtype, 5)
    want = ops.linear(s["x"], s["w"], activation="relu")
    s["x"][3, 7] = float("nan")
    s["x"][70, 1] = float("inf")
    s["x"][149, 263] = float("nan")
    y = ops.linear(s["x"], s["w"], activation="relu")
    keep = [i for i in range(150) if i not in (3, 70, 149)]
    assert torch.equal(y[keep], want[keep]) and torch.isnan(y[3]).all() and torch.isnan(y[149]).all()
    assert not torch.isfinite(y[70][y[70] != 0]).any()
    s["dy"][2, 5] = float("nan")
    s["x"].nan_to_num_(0, 0, 0)
    dx, dw, db = ops.linear_backward(s["dy"], s["x"], s["w"])
    rows, cols = torch.isnan(dx).any(1), torch.isnan(dw).any(1)
    assert rows[2] and rows.sum() == 1 and cols[5] and cols.sum() == 1 and torch.isnan(db).sum() == 1


def test_nothing_past_the_result_is_written():
    for m, n, k in ((5, 130, 72), (65, 63, 129), (3, 24, 4096)):
        s = make(m, n, k, torch.float16, 2)
        room = torch.full((m * n + 64,), 7.0, dtype=torch.float16, device="cuda")
        size = lib.dll.fwdmi_linear_workspace(m, n, k, lib.F16)
        ws = torch.full((size + 64,), 77, dtype=torch.uint8, device="cuda")
        p = ops._p
        lib.check(lib.dll.fwdmi_linear(ops._stream(None), m, n, k, p(s["x"]), p(s["w"]), None, None, p(room[32:]), None,
                                       lib.ACT_NONE, lib.F16, p(ws), size))
        assert torch.equal(room[32:32 + m * n].view(m, n), ops.linear(s["x"], s["w"]))
        assert (room[:32] == 7).all() and (room[32 + m * n:] == 7).all() and (ws[size:] == 77).all()


def test_results_repeat_bit_for_bit():
    s = make(771, 1011, 768, torch.float16, 9)
    a = ops.linear_backward(s["dy"], s["x"], s["w"], preact=s["r"], activation="gelu")
    y = ops.linear(s["x"], s["w"], bias=s["b"], activation="gelu")
    for _ in range(3):
        b = ops.linear_backward(s["dy"], s["x"], s["w"], preact=s["r"], activation="gelu")
        assert all(torch.equal(p, q) for p, q in zip(a, b))
        assert torch.equal(y, ops.linear(s["x"], s["w"], bias=s["b"], activation="gelu"))


@pytest.mark.parametrize("act", ACTS[2:])
def test_against_differences(act):
    """dx, dw and dbias against central differences of the fp64 definition (the smooth activations)."""
    g = gen(21)
    x, w = torch.randn(3, 6, generator=g, device="cuda"), torch.randn(5, 6, generator=g, device="cuda")
    b, dy = torch.randn(5, generator=g, device="cuda"), torch.randn(3, 5, generator=g, device="cuda")
    _, z = ops.linear(x, w, bias=b, activation=act, want_preact=True)
    grads = [t.double().cpu() for t in ops.linear_backward(dy, x, w, preact=z, activation=act)]
    p = [t.double().cpu() for t in (x, w, b)]
    loss = lambda: (act64(p[0] @ p[1].t() + p[2], act)[0] * dy.double().cpu()).sum().item()
    step = 1e-5          # truncation ~ step^2, cancellation ~ 1e-16 / step: 1e-10 both; fp32 results ~ 1e-6
    for t, grad in zip(p, grads):
        flat = t.view(-1)
        for i in range(flat.numel()):
            old = flat[i].item()
            flat[i] = old + step
            up = loss()
            flat[i] = old - step
            down = loss()
            flat[i] = old
            assert abs((up - down) / (2 * step) - grad.reshape(-1)[i].item()) < 2e-5, (act, i)


def test_on_another_stream():
    side = torch.cuda.Stream()
    s = make(384, 1024, 4096, torch.bfloat16, 8)
    want = ops.linear(s["x"], s["w"], bias=s["b"], residual=s["r"])
    wantb = ops.linear_backward(s["dy"], s["x"], s["w"], preact=s["r"], activation="gelu")
    side.wait_stream(torch.cuda.current_stream())
    got = ops.linear(s["x"], s["w"], bias=s["b"], residual=s["r"], stream=side)
    gotb = ops.linear_backward(s["dy"], s["x"], s["w"], preact=s["r"], activation="gelu", stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(want, got) and all(torch.equal(a, b) for a, b in zip(wantb, gotb))


def test_captured_into_a_graph():
    """The feed-forward half of a layer, forward and backward, replayed on new values."""
    names = dict(x=(200, 256), w1=(1024, 256), w2=(256, 1024), dy=(200, 256))

    def values(seed):
        g = gen(seed)
        v = {k: (torch.randn(*s, generator=g, device="cuda") * (0.05 if k[0] == "w" else 1.0)).half() for k, s in names.items()}
        v["b1"], v["b2"] = torch.randn(1024, generator=g, device="cuda") * 0.1, torch.randn(256, generator=g, device="cuda") * 0.1
        v["gamma"], v["beta"] = torch.randn(256, generator=g, device="cuda") + 1, torch.randn(256, generator=g, device="cuda")
        return v

    s = values(0)

    def step():
        h, z = ops.linear(s["x"], s["w1"], bias=s["b1"], activation="gelu", want_preact=True)
        f = ops.linear(h, s["w2"], bias=s["b2"])
        y, mean, rstd = ops.layer_norm_forward(f, s["gamma"], s["beta"], skip=s["x"], eps=1e-5)
        df, dg, db = ops.layer_norm_backward(s["dy"], f, s["gamma"], mean, rstd, skip=s["x"])
        dh, dw2, db2 = ops.linear_backward(df, h, s["w2"])
        dx, dw1, db1 = ops.linear_backward(dh, s["x"], s["w1"], preact=z, activation="gelu")
        return y, dg, db, dw2, db2, dx, dw1, db1

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(1, 5):
        for k, v in values(seed).items():
            s[k].copy_(v)
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), seed
