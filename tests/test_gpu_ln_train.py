"""layer_norm_forward / layer_norm_backward on the GPU against their definitions in fp64.

Bounds (u = 2^-24, eps_T = torch.finfo(T).eps, a rounding to T is off by at most eps_T / 2 relative):
  h = x + skip + bias takes two fp32 additions: |dh| <= 2u H with H = |x| + |skip| + |bias|.
  A row sum adds at most 48 terms in sequence in a lane (rows up to 24576 elements over 512 lanes, or 32 elements a
  lane) and then 6 + 7 across lanes and waves: relative error at most 61u of the sum of magnitudes; products in front of
  the sum, the division by n and the 1-ulp reciprocal square root add less than 8 more.  N = 72 covers them.
  So mean is off by at most N u mean(H), xhat by D = N u rstd (H + mean(H)) + N u |xhat|, y by |gamma| D + 2u |y| and
  its rounding.  The backward pass takes mean and rstd as given: xhat is off by D' = 8u rstd (H + |mean|);
  dx by rstd (N u (|g| + mean|g| + |xhat| mean|g xhat|) + D' mean|g xhat| + |xhat| mean(|g| D')) and its rounding.
  Column sums add at most 64 rows in sequence in a lane, 64 groups, 16 parts and 16 waves at these sizes: C = 168 additions
  and products, so they are off by at most C u sum|terms| plus the terms' own errors.
"""
import numpy as np
import pytest
import torch

from forward_amd import lib, ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
N, C = 72, 168
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def make(rows, ld, dtype, seed, skip=True, bias=True, dsum=False, offset=0, scale=1.0, shift=0.0):
    """Inputs; ``offset`` elements of the allocation lie in front of every [rows, ld] operand (unaligned starts)."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def plane(std=1.0, mean=0.0):
        t = torch.empty(rows * ld + offset, dtype=dtype, device="cuda")
        t.copy_(torch.randn(t.shape, generator=g, device="cuda") * std + mean)
        return t[offset:].view(rows, ld)

    def vec(mean, std):
        t = torch.randn(ld + offset, generator=g, device="cuda") * std + mean
        return t[offset:]

    return dict(x=plane(scale, shift), skip=plane(scale) if skip else None, bias=vec(0.0, 0.5) if bias else None,
                gamma=vec(1.0, 0.3), beta=vec(0.0, 0.3), dy=plane(0.5), dsum=plane(0.5) if dsum else None)


def d(t):
    return 0.0 if t is None else t.double()


def check(got, want, bound, what):
    err = (got.double() - want).abs()
    worst = (err - bound).max().item() if err.numel() else 0.0
    assert not torch.isnan(err).any() and worst <= 0.0, "%s: %g past its bound" % (what, worst)


def half(dtype):
    return 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2


def check_forward(s, eps, want_sum):
    x = s["x"]
    h = d(x) + d(s["skip"]) + d(s["bias"])
    H = d(x).abs() + (d(s["skip"]).abs() if s["skip"] is not None else 0) + (d(s["bias"]).abs() if s["bias"] is not None else 0)
    var, mean = torch.var_mean(h, 1, correction=0, keepdim=True)
    rstd = (var + eps) ** -0.5
    xh = (h - mean) * rstd
    D = N * U * (rstd * (H + H.mean(1, keepdim=True)) + xh.abs())
    y = xh * d(s["gamma"]) + d(s["beta"])
    out = ops.layer_norm_forward(x, s["gamma"], s["beta"], skip=s["skip"], bias=s["bias"], eps=eps, want_sum=want_sum)
    e = half(x.dtype)
    by = d(s["gamma"]).abs() * D + 4 * U * (y.abs() + d(s["beta"]).abs())
    check(out[0], y, by + e * (y.abs() + by) + torch.finfo(x.dtype).tiny, "y")
    check(out[1], mean[:, 0], (N * U * H.mean(1)), "mean")
    # d(rstd) / rstd = d(var) / (2 (var + eps)); var's error: N u var + 2 |dh| |h - mean| averaged
    dv = N * U * var[:, 0] + 2 * ((2 * U * H + N * U * H.mean(1, keepdim=True)) * (h - mean).abs()).mean(1)
    check(out[2], rstd[:, 0], rstd[:, 0] * (dv / (var[:, 0] + eps) + 4 * U), "rstd")
    if want_sum:
        check(out[3], h, 2 * U * H + e * (h.abs() + 2 * U * H) + torch.finfo(x.dtype).tiny, "sum")
    return out


def check_backward(s, mean, rstd):
    x = s["x"]
    h = d(x) + d(s["skip"]) + d(s["bias"])
    H = d(x).abs() + (d(s["skip"]).abs() if s["skip"] is not None else 0) + (d(s["bias"]).abs() if s["bias"] is not None else 0)
    m, r = d(mean)[:, None], d(rstd)[:, None]
    xh = (h - m) * r
    D = 8 * U * r * (H + m.abs())
    g = d(s["dy"]) * d(s["gamma"])
    c1, c2 = (g * xh).mean(1, keepdim=True), g.mean(1, keepdim=True)
    dh = r * (g - c2 - xh * c1)
    dx = dh + d(s["dsum"])
    m1 = (g * xh).abs().mean(1, keepdim=True)
    bh = r * (N * U * (g.abs() + g.abs().mean(1, keepdim=True) + xh.abs() * m1) + D * m1 + xh.abs() * (g.abs() * D).mean(1, keepdim=True))
    bx = bh + 2 * U * (dx.abs() + (d(s["dsum"]).abs() if s["dsum"] is not None else 0))
    out = ops.layer_norm_backward(s["dy"], x, s["gamma"], mean, rstd, skip=s["skip"], bias=s["bias"], dsum=s["dsum"])
    e = half(x.dtype)
    check(out[0], dx, bx + e * (dx.abs() + bx) + torch.finfo(x.dtype).tiny, "dx")
    dy = d(s["dy"])
    check(out[1], (dy * xh).sum(0), (C * U * (dy * xh).abs() + dy.abs() * D).sum(0), "dgamma")
    check(out[2], dy.sum(0), C * U * dy.abs().sum(0), "dbeta")
    assert len(out) == (4 if s["bias"] is not None else 3)
    if s["bias"] is not None:
        check(out[3], dx.sum(0), (C * U * dx.abs() + bx).sum(0), "dbias")
    return out


# every lane layout: parts of a wavefront, whole ones, four and eight of them, streamed; full and ragged
WIDTHS = [1, 3, 4, 7, 8, 9, 31, 32, 64, 100, 127, 128, 200, 256, 257, 500, 512, 768, 1000, 1024, 1025, 1531, 2048, 2050,
          4096, 4097, 8192, 9999, 16384, 16400, 24576]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ld", WIDTHS)
def test_widths(ld, dtype):
    rows = 37 if ld <= 4096 else 9
    s = make(rows, ld, dtype, ld, skip=ld % 2 == 0, bias=ld % 3 != 0, dsum=ld % 5 == 0)
    _, mean, rstd, _ = check_forward(s, 1e-5, True)
    check_backward(s, mean, rstd)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 2, 8, 9, 64, 257, 2049, 5000])
def test_rows(rows, dtype):
    for ld, flags in ((64, dict(skip=False, bias=False)), (1024, dict(skip=True, bias=True, dsum=True)),
                      (1531, dict(skip=True, bias=False))):
        if rows * ld > 3000000:
            continue
        s = make(rows, ld, dtype, rows + ld, **flags)
        _, mean, rstd = check_forward(s, 1e-5, False)
        check_backward(s, mean, rstd)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ld", [3, 64, 128, 200, 512, 768, 1024, 1030, 1531, 2048, 4096, 8192])
@pytest.mark.parametrize("bias", [False, True])
def test_more_rows_than_one_launch_sums(ld, bias, dtype):
    s = make(1027, ld, dtype, ld + bias, skip=ld % 3 == 0, bias=bias, dsum=ld % 4 == 0)
    _, mean, rstd = check_forward(s, 1e-5, False)
    check_backward(s, mean, rstd)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset", [1, 2, 3, 7])
def test_operands_start_at_any_element(offset, dtype):
    for ld in (5, 96, 1024, 1040):
        s = make(33, ld, dtype, offset, dsum=True, offset=offset)
        _, mean, rstd, _ = check_forward(s, 1e-6, True)
        check_backward(s, mean, rstd)


@pytest.mark.parametrize("dtype", TYPES)
def test_large_means_and_scales(dtype):
    for scale, shift in ((1e-3, 0.0), (100.0, 0.0), (1.0, 50.0)):
        s = make(65, 768, dtype, 5, bias=False, scale=scale, shift=shift)
        _, mean, rstd = check_forward(s, 1e-12, False)
        check_backward(s, mean, rstd)


def test_sum_alone_serves_the_backward_pass():
    """Backward from the stored fp32 sum equals backward from its parts: dx bit for bit (the same fp32 operations on the
    same h), the column sums as far as two orders of adding them agree (each is within C u of the exact sum)."""
    s = make(50, 512, torch.float32, 3)
    y, mean, rstd, h = ops.layer_norm_forward(s["x"], s["gamma"], s["beta"], skip=s["skip"], bias=s["bias"], eps=1e-5, want_sum=True)
    a = ops.layer_norm_backward(s["dy"], s["x"], s["gamma"], mean, rstd, skip=s["skip"], bias=s["bias"])
    b = ops.layer_norm_backward(s["dy"], h, s["gamma"], mean, rstd)
    assert torch.equal(a[0], b[0])
    xh = (d(h) - d(mean)[:, None]) * d(rstd)[:, None]
    check(a[1], d(b[1]), 2 * C * U * (d(s["dy"]) * xh).abs().sum(0), "dgamma")
    check(a[2], d(b[2]), 2 * C * U * d(s["dy"]).abs().sum(0), "dbeta")


def test_against_differences():
    """dx and the parameter gradients against central differences of the fp64 definition."""
    s = make(3, 40, torch.float32, 11)
    eps = 1e-5
    _, mean, rstd = ops.layer_norm_forward(s["x"], s["gamma"], s["beta"], skip=s["skip"], bias=s["bias"], eps=eps)
    dx, dgamma, dbeta, dbias = (t.double().cpu() for t in ops.layer_norm_backward(
        s["dy"], s["x"], s["gamma"], mean, rstd, skip=s["skip"], bias=s["bias"]))
    p = {k: v.double().cpu() for k, v in s.items() if v is not None}

    def loss(q):
        h = q["x"] + q["skip"] + q["bias"]
        var, m = torch.var_mean(h, 1, correction=0, keepdim=True)
        return (((h - m) * (var + eps) ** -0.5 * q["gamma"] + q["beta"]) * q["dy"]).sum().item()

    step = 1e-5      # truncation ~ step^2 = 1e-10, cancellation ~ 1e-16 * |loss| / step = 1e-10; fp32 results ~ 1e-6
    for name, grad in (("x", dx), ("skip", dx), ("gamma", dgamma), ("beta", dbeta), ("bias", dbias)):
        flat = p[name].reshape(-1)
        for i in range(0, flat.numel(), 7):
            old = flat[i].item()
            flat[i] = old + step
            up = loss(p)
            flat[i] = old - step
            down = loss(p)
            flat[i] = old
            assert abs((up - down) / (2 * step) - grad.reshape(-1)[i].item()) < 2e-5, (name, i)


@pytest.mark.parametrize("dtype", TYPES)
def test_no_rows(dtype):
    s = make(0, 24, dtype, 1)
    y, mean, rstd = ops.layer_norm_forward(s["x"], s["gamma"], s["beta"], eps=1e-5)
    assert y.shape == (0, 24) and mean.numel() == 0
    dx, dg, db, dh = ops.layer_norm_backward(s["dy"], s["x"], s["gamma"], mean, rstd, bias=s["bias"])
    assert dx.shape == (0, 24) and not dg.any() and not db.any() and not dh.any()


def test_a_row_of_nan_stays_its_own():
    for ld in (64, 1000, 4096):
        s = make(40, ld, torch.float16, 2, dsum=True)
        clean = ops.layer_norm_forward(s["x"], s["gamma"], s["beta"], skip=s["skip"], eps=1e-5)
        s["x"][7, 3] = float("nan")
        s["x"][9, 5] = float("inf")
        got = ops.layer_norm_forward(s["x"], s["gamma"], s["beta"], skip=s["skip"], eps=1e-5)
        keep = [i for i in range(40) if i not in (7, 9)]
        for a, b in zip(got, clean):
            assert torch.equal(a[keep], b[keep]) and torch.isnan(a[7]).all()
        dx = ops.layer_norm_backward(s["dy"], s["x"], s["gamma"], got[1], got[2], skip=s["skip"])[0]
        assert not torch.isnan(dx[keep]).any() and torch.isnan(dx[7]).all()


def test_constant_rows_have_no_variance():
    x = torch.full((5, 96), 3.0, device="cuda")
    g, b = torch.ones(96, device="cuda"), torch.full((96,), 0.25, device="cuda")
    y, mean, rstd = ops.layer_norm_forward(x, g, b, eps=1e-5)
    assert torch.equal(y, torch.full_like(x, 0.25)) and torch.equal(mean, torch.full_like(mean, 3.0))
    dx = ops.layer_norm_backward(torch.ones_like(x), x, g, mean, rstd)[0]
    assert dx.abs().max().item() <= 96 * U * rstd.max().item()          # g - mean(g) = 0 up to the mean's rounding


def test_results_repeat_bit_for_bit_and_agree_with_the_inference_launch():
    s = make(3001, 1024, torch.float16, 6)
    first = ops.layer_norm_forward(s["x"], s["gamma"], s["beta"], skip=s["skip"], bias=s["bias"], eps=1e-5)
    grads = ops.layer_norm_backward(s["dy"], s["x"], s["gamma"], first[1], first[2], skip=s["skip"], bias=s["bias"])
    for _ in range(3):
        again = ops.layer_norm_backward(s["dy"], s["x"], s["gamma"], first[1], first[2], skip=s["skip"], bias=s["bias"])
        assert all(torch.equal(a, b) for a, b in zip(grads, again))
    infer = ops.skip_layer_norm(s["x"], s["gamma"], s["beta"], skip=s["skip"], bias=s["bias"], eps=1e-5)
    # Both are within `by` of the definition before their rounding (the inference launch adds 16 terms a lane and merges
    # six times, inside N as well), so they are at most 2 by apart, plus half a step of each rounding: near a sum
    # gamma xhat + beta that cancels, by is what counts, not a step of the small result.
    H = (d(s["x"]).abs() + d(s["skip"]).abs() + d(s["bias"]).abs())
    h = d(s["x"]) + d(s["skip"]) + d(s["bias"])
    r = d(first[2])[:, None]
    xh = (h - d(first[1])[:, None]) * r
    by = d(s["gamma"]).abs() * N * U * (r * (H + H.mean(1, keepdim=True)) + xh.abs()) \
        + 4 * U * ((xh * d(s["gamma"]) + d(s["beta"])).abs() + d(s["beta"]).abs())
    a, b = d(first[0]), d(infer)
    check(first[0], b, 2 * by + half(torch.float16) * (a.abs() + b.abs()) + 2.0 ** -24, "inference launch")


def test_on_another_stream():
    side = torch.cuda.Stream()
    s = make(512, 1024, torch.bfloat16, 8)
    want = ops.layer_norm_forward(s["x"], s["gamma"], s["beta"], skip=s["skip"], eps=1e-5)
    wantb = ops.layer_norm_backward(s["dy"], s["x"], s["gamma"], want[1], want[2], skip=s["skip"])
    side.wait_stream(torch.cuda.current_stream())
    got = ops.layer_norm_forward(s["x"], s["gamma"], s["beta"], skip=s["skip"], eps=1e-5, stream=side)
    gotb = ops.layer_norm_backward(s["dy"], s["x"], s["gamma"], got[1], got[2], skip=s["skip"], stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want + wantb, got + gotb))


def test_captured_into_a_graph():
    s = make(700, 768, torch.float16, 12, dsum=True)

    def step():
        f = ops.layer_norm_forward(s["x"], s["gamma"], s["beta"], skip=s["skip"], bias=s["bias"], eps=1e-5, want_sum=True)
        return f + ops.layer_norm_backward(s["dy"], s["x"], s["gamma"], f[1], f[2], skip=s["skip"], bias=s["bias"], dsum=s["dsum"])

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(4):
        new = make(700, 768, torch.float16, 100 + seed, dsum=True)
        for k in new:
            s[k].copy_(new[k])
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), seed


def test_workspace_of_the_wrong_size_is_refused():
    s = make(3000, 64, torch.float32, 1)
    ld, n = 64, 3000 * 64
    need = lib.dll.fwdmi_layer_norm_backward_workspace(ld, n, 0, lib.F32)
    assert need > 0
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    _, mean, rstd = ops.layer_norm_forward(s["x"], s["gamma"], s["beta"], eps=1e-5)
    out = [torch.zeros_like(s["gamma"]) for _ in range(2)]
    p = ops._p
    rc = lib.dll.fwdmi_layer_norm_backward(None, ld, n, p(s["dy"]), p(s["x"]), None, None, p(s["gamma"]), None, p(mean),
                                           p(rstd), p(torch.empty_like(s["x"])), p(out[0]), p(out[1]), None, p(ws), need - 1,
                                           lib.F32)
    assert rc == lib.ERR_BAD_ARG and "workspace" in lib.last_error()
