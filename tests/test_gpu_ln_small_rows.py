"""layer_norm_forward on rows whose variance lies at the lower end of fp32, without an eps, against the definition in fp64.

Bounds (u = 2^-24; H, N, D as in test_gpu_ln_train.py): squares and sums below 2^-126 are rounded to multiples of 2^-149, so
each of a row's additions is off by at most 2^-150 more, and so is the mean of the squares: var by
dv = N u var + 2 mean(|dh| |h - mean|) + 2^-149 (its own last rounding included), rstd by rstd dv / (2 var) in first order
(dv / var covers the second), and xhat by |xhat| times that beside D.
"""
import pytest
import torch

from forward_amd import ops

pytestmark = pytest.mark.gpu
U, N = 2.0 ** -24, 72


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("ld", [3, 96, 1000, 1531, 4096, 16400])
@pytest.mark.parametrize("scale", [1e-17, 1e-19, 3e-20, 1e-20])
def test_small_rows_without_eps(scale, ld, dtype):
    g = torch.Generator(device="cuda").manual_seed(ld)
    x = (torch.randn(9, ld, generator=g, device="cuda") * scale).to(dtype)
    gamma = torch.randn(ld, generator=g, device="cuda") + 1
    beta = torch.randn(ld, generator=g, device="cuda")
    y, mean, rstd = ops.layer_norm_forward(x, gamma, beta, eps=0.0)
    h = x.double()
    H = h.abs()
    var, mu = torch.var_mean(h, 1, correction=0, keepdim=True)
    r = var ** -0.5
    dh = 2 * U * H + N * U * H.mean(1, keepdim=True)
    off = (N * U * var + 2 * (dh * (h - mu).abs()).mean(1, keepdim=True) + 2.0 ** -149) / var + 4 * U
    assert (off < 0.01).all() and torch.isfinite(y).all()
    assert ((rstd.double() - r[:, 0]).abs() <= r[:, 0] * off[:, 0]).all()
    xh = (h - mu) * r
    D = N * U * (r * (H + H.mean(1, keepdim=True)) + xh.abs()) + xh.abs() * off
    want = xh * gamma.double() + beta.double()
    bound = gamma.double().abs() * D + 4 * U * (want.abs() + beta.double().abs())
    half = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    assert ((y.double() - want).abs() <= bound + half * (want.abs() + bound)).all()
    # and back: the statistics as given, finite gradients of the same magnitude as rstd
    dy = torch.randn(9, ld, generator=g, device="cuda").to(dtype)
    dx, dgamma, dbeta = ops.layer_norm_backward(dy, x, gamma, mean, rstd)
    assert all(torch.isfinite(t).all() for t in (dx, dgamma, dbeta))


def test_rows_without_any_variance_are_as_before():
    """var = 0 and no eps: rstd is infinite, as the definition's quotient is."""
    x = torch.full((2, 64), 3.0, device="cuda")
    _, mean, rstd = ops.layer_norm_forward(x, torch.ones(64, device="cuda"), torch.zeros(64, device="cuda"), eps=0.0)
    assert torch.isinf(rstd).all() and (rstd > 0).all() and torch.equal(mean, torch.full_like(mean, 3.0))
