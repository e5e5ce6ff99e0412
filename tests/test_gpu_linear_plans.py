"""Every variant of the linear layer's kernels against 64 bits: y, dx, dw and both gradients together, each in a call of its own.

Bounds as derived in test_gpu_linear.py; the gradients' with an activation count the rounding of dz to the type as well.
"""
import pytest
import torch
from linear_sizes import SIZES, drawn, variants
from test_gpu_linear import TYPES, U, act64, check, check_linear, half, make

from forward_amd import ops

pytestmark = pytest.mark.gpu


def test_the_tested_sizes_reach_every_variant_on_this_device():
    tested = set().union(*(variants(*s) for s in SIZES))
    missing = {}
    for s in drawn(20000, 4):
        for v in variants(*s) - tested:
            missing.setdefault(v, s)
    assert not missing, missing


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", SIZES)
def test_products(size, dtype):
    m, n, k, on_boundary, with_act = size
    s = make(m, n, k, dtype, m + 3 * n + 7 * k, 0 if on_boundary else 1)
    act = "gelu" if with_act else "none"
    check_linear(s, act, bias=True, residual=True, preact=bool(with_act))
    x, w, dy, e, tiny = s["x"], s["w"], s["dy"], half(dtype), torch.finfo(dtype).tiny
    z = s["r"] if with_act else None
    grads = dict(preact=z, activation=act)
    dz = dy.double()
    off = torch.zeros_like(dz)
    if with_act:
        dz = dz * act64(z.double(), act)[1]
        off = 32 * U * dy.double().abs() + e * dz.abs() + tiny
    A = dz.abs() + off
    dx, dw = dz @ w.double(), dz.t() @ x.double()
    bx = (n + 8) * 2 * U * (A @ w.double().abs()) + off @ w.double().abs()
    bw = (m + 8) * 2 * U * (A.t() @ x.double().abs()) + off.t() @ x.double().abs()
    bx, bw = bx + e * (dx.abs() + bx) + tiny, bw + e * (dw.abs() + bw) + tiny
    bb = ((m + 8) * 2 * U * dz.abs() + 32 * U * dy.double().abs() * with_act).sum(0)
    db = dz.sum(0)
    del dz, off, A
    check(ops.linear_backward(dy, x, w, want_dweight=False, want_dbias=False, **grads)[0], dx, bx, "dx alone")
    check(ops.linear_backward(dy, x, w, want_dx=False, want_dbias=False, **grads)[0], dw, bw, "dw alone")
    got = ops.linear_backward(dy, x, w, **grads)
    check(got[0], dx, bx, "dx")
    check(got[1], dw, bw, "dw")
    check(got[2], db, bb, "dbias")
