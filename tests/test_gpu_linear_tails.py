"""The activations and their slopes against 64 bits relative to their own value, far into the tails where that value is small.

The pre-activations pass through an identity weight, so z is exact, and a slope is read from dbias over one row.  Bounds
(u = 2^-24), fp32: an exponential is off by at most 3 units in the last place (6u), erfc by 16 (32u), what OpenCL asks of
both; a reciprocal by one (2u), every other operation by u; arguments are exact to 2^-48 of themselves.
  logistic p = t r or r, r = 1 / (1 + t), t = e^-|a|: t 6u + 1u for its low part, 1 + t u more, the reciprocal 2u, t r u, t in
  the sum 7u again: 18u;  silu = z p: 19u;  tanh-GELU likewise
  Phi = erfc / 2: 32u, its correction's own rounding and the sum 2u: 34u;  gelu = z Phi: 35u
  slopes p (1 + z rest), p + z p rest 2 sqrt(2 / pi) (1 + 0.134145 z^2) and Phi + z phi: no factor off by more than 18u (35u),
  at most two such and six operations: 2 * 18u + 6u = 42u of the sum of magnitudes (gelu: 35u and 6u + 6u, so 42u as well).
A logistic below 2^-126 is 0 by definition here (silu(-100) is -0): off by at most 2^-126, which the value has times |z| and
the slope times 1 + |z| 2 sqrt(2 / pi) (1 + 0.134145 z^2), the largest factor of the three (1 + 1.6 |z| (1 + 0.14 z^2) below);
results that are subnormal themselves are multiples of 2^-149, which that covers.
16-bit results: half a step, and for GELU the error of its polynomial as stated beside it.
"""
import math

import pytest
import torch

from forward_amd import ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
SPANS = [(-110, -60), (-60, -16), (-16, -12), (-12, -8), (-8, -6), (-6, -4), (-4, -1), (-1, 1), (1, 4), (4, 16), (16, 110)]


def exact(z, act):
    """The activation, its slope and the slope's magnitude (on the CPU: erfc there keeps its tail)."""
    z = z.double().cpu()
    if act == "gelu":
        p, b = 0.5 * torch.special.erfc(-z * math.sqrt(0.5)), z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    else:
        a = z if act == "silu" else 2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
        p, rest = torch.sigmoid(a), torch.sigmoid(-a)
        b = z * p * rest * (1.0 if act == "silu" else 2 * math.sqrt(2 / math.pi) * (1 + 0.134145 * z * z))
    return z * p, p + b, p + b.abs()


def least(z):
    return 2.0 ** -126 * (1 + 1.6 * z.abs() * (1 + 0.14 * z * z))


def through(z, act):
    n, dt = z.numel(), z.dtype
    y = ops.linear(z.view(-1, 64), torch.eye(64, device="cuda", dtype=dt), activation=act)
    one = torch.ones(1, n, device="cuda", dtype=dt)
    _, _, slope = ops.linear_backward(one, torch.zeros(1, 8, device="cuda", dtype=dt), torch.zeros(n, 8, device="cuda", dtype=dt),
                                      preact=z.view(1, n), activation=act)
    return y.double().cpu().view(-1), slope.double().cpu()


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("span", SPANS)
def test_fp32_keeps_its_digits(span, act):
    z = torch.linspace(*span, 4096, device="cuda")
    y, slope = through(z, act)
    a, s, m = exact(z, act)
    tiny = least(z.double().cpu())
    worst = lambda got, want, bound: ((got - want).abs() - bound).max().item()
    assert worst(y, a, (35 if act == "gelu" else 19) * U * a.abs() + tiny) <= 0
    assert worst(slope, s, 42 * U * m + tiny) <= 0


# relative error of 16-bit GELU's lower tail between one point and the next
TAIL = [(-3, 0.00006), (-4, 0.0005), (-5, 0.0016), (-6, 0.0036), (-8, 0.0103), (-13, 0.0371)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
def test_16_bit_results_and_the_stated_tail_of_gelu(act, dtype):
    z = torch.linspace(-13, 13, 8192, device="cuda").to(dtype)
    y, slope = through(z, act)
    a, s, m = exact(z, act)
    zd = z.double().cpu()
    tail = torch.zeros_like(zd)
    if act == "gelu":
        for at, most in TAIL[::-1]:
            tail[zd >= at] = most
        tail[zd >= 0] = 0
    half = torch.finfo(dtype).eps / 2
    # an exponent's argument is rounded: at most 3u of it; |a| <= 4 z^2 + 2 |z| covers the three
    rough = (40 + 3 * (4 * zd * zd * (1 + zd.abs() * (act == "gelu_tanh") / 8) + 2 * zd.abs())) * U
    err = rough + tail + half * (1 + tail + rough)
    none = least(zd)
    small = torch.finfo(dtype).tiny * torch.finfo(dtype).eps + none
    assert ((y - a).abs() - err * a.abs() - small).max().item() <= 0
    # the polynomial's 1.5e-7 is of erf, twice what it is of Phi; slopes come back in fp32
    assert ((slope - s).abs() - rough * m - (7.5e-8 if act == "gelu" else 0.0) - none).max().item() <= 0
