"""Argument checks of the training launchers and their tensor-level wrappers: what they refuse, without a GPU."""
import pytest
import torch

from forward_amd import lib, ops


@pytest.fixture(autouse=True)
def host_tensors_pass_as_device(monkeypatch):
    def dev(t, name):
        if not isinstance(t, torch.Tensor):
            raise RuntimeError(name)
        if not t.is_contiguous():
            raise ValueError(name)
        return t
    monkeypatch.setattr(ops, "_dev", dev)


def z(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


def test_layer_norm_forward_refuses():
    good = dict(x=z(4, 16), gamma=z(16), beta=z(16))
    for change in (dict(gamma=z(15)), dict(beta=z(17)), dict(gamma=z(16, dtype=torch.float16)), dict(skip=z(4, 8)),
                   dict(skip=z(4, 16, dtype=torch.float16)), dict(bias=z(8)), dict(x=z(4, 0), gamma=z(0), beta=z(0)),
                   dict(x=z(16, 4).t())):
        with pytest.raises(ValueError):
            ops.layer_norm_forward(**{**good, **change})
    with pytest.raises(TypeError):
        ops.layer_norm_forward(z(4, 16, dtype=torch.float64), z(16), z(16))


def test_layer_norm_backward_refuses():
    good = dict(dy=z(4, 16), x=z(4, 16), gamma=z(16), mean=z(4), rstd=z(4))
    for change in (dict(dy=z(4, 15)), dict(dy=z(4, 16, dtype=torch.float16)), dict(mean=z(3)), dict(rstd=z(5)),
                   dict(mean=z(4, dtype=torch.float16)), dict(skip=z(2, 16)), dict(bias=z(4)), dict(dsum=z(4, 17)),
                   dict(gamma=z(8))):
        with pytest.raises(ValueError):
            ops.layer_norm_backward(**{**good, **change})


def test_layer_norm_launchers_refuse():
    d = lib.dll
    one = 64   # stands for a pointer: the calls below return before anything is read through it
    assert d.fwdmi_layer_norm_forward(None, 10, 25, *[None] * 9, lib.F32, 0.0) == lib.ERR_BAD_ARG
    assert d.fwdmi_layer_norm_forward(None, 0, 0, *[None] * 9, lib.F32, 0.0) == lib.ERR_BAD_ARG
    assert d.fwdmi_layer_norm_forward(None, 10, -10, *[None] * 9, lib.F32, 0.0) == lib.ERR_BAD_ARG
    assert d.fwdmi_layer_norm_forward(None, 10, 20, *[None] * 9, lib.I8, 0.0) == lib.ERR_UNSUPPORTED
    assert d.fwdmi_layer_norm_forward(None, 10, 20, *[None] * 9, lib.BF16, 0.0) == lib.ERR_BAD_ARG     # null pointers
    assert d.fwdmi_layer_norm_forward(None, 10, 0, *[None] * 9, lib.BF16, 0.0) == lib.OK               # nothing to do
    assert d.fwdmi_layer_norm_backward(None, 10, 20, *[None] * 13, 0, lib.I32) == lib.ERR_UNSUPPORTED
    assert d.fwdmi_layer_norm_backward(None, 10, 20, *[None] * 13, 0, lib.F16) == lib.ERR_BAD_ARG
    # a bias without room for its gradient, and the other way round
    args = [one] * 4 + [one, one, one, one, one, one, one, None, one]
    assert d.fwdmi_layer_norm_backward(None, 10, 20, *args, 1 << 20, lib.F16) == lib.ERR_BAD_ARG
    args[5], args[11] = None, one
    assert d.fwdmi_layer_norm_backward(None, 10, 20, *args, 1 << 20, lib.F16) == lib.ERR_BAD_ARG
    # no workspace
    args[11], args[12] = None, None
    assert d.fwdmi_layer_norm_backward(None, 10, 100000, *args, 1 << 20, lib.F16) == lib.ERR_BAD_ARG
    assert "workspace" in lib.last_error()


def test_layer_norm_workspace_sizes():
    f = lib.dll.fwdmi_layer_norm_backward_workspace
    assert f(16, 0, 1, lib.F32) == 0 and f(0, 16, 1, lib.F32) == 0 and f(16, 17, 1, lib.F32) == 0 and f(16, 16, 1, lib.I8) == 0
    assert f(1024, 8192 * 1024, 1, lib.F16) >= 2 * 3 * 1024 * 4 and f(1024, 1024, 1, lib.F16) == 0
    assert f(100000, 50 * 100000, 0, lib.F32) >= 50 * 8 + 2 * 2 * 100000 * 4


def test_linear_refuses():
    good = dict(x=z(4, 16), weight=z(8, 16))
    for change in (dict(weight=z(8, 15)), dict(weight=z(8, 16, dtype=torch.float16)), dict(weight=z(8, 16, 1)), dict(bias=z(16)),
                   dict(bias=z(8, dtype=torch.float16)), dict(residual=z(4, 16)), dict(residual=z(4, 8, dtype=torch.float16)),
                   dict(activation="tanh"), dict(weight=z(16, 8).t())):
        with pytest.raises(ValueError):
            ops.linear(**{**good, **change})
    with pytest.raises(TypeError):
        ops.linear(z(4, 16, dtype=torch.float64), z(8, 16, dtype=torch.float64))


def test_linear_backward_refuses():
    good = dict(dy=z(4, 8), x=z(4, 16), weight=z(8, 16), preact=z(4, 8), activation="gelu")
    for change in (dict(dy=z(4, 16)), dict(dy=z(4, 8, dtype=torch.float16)), dict(preact=None), dict(preact=z(4, 16)),
                   dict(preact=z(4, 8, dtype=torch.bfloat16)), dict(weight=z(8, 8)), dict(activation="")):
        with pytest.raises(ValueError):
            ops.linear_backward(**{**good, **change})


def test_linear_launchers_refuse():
    d = lib.dll
    none6 = [None] * 6
    assert d.fwdmi_linear(None, 4, 8, 16, *none6, lib.ACT_NONE, lib.I8, None, 0) == lib.ERR_UNSUPPORTED
    assert d.fwdmi_linear(None, 4, 8, 16, *none6, 9, lib.F16, None, 0) == lib.ERR_BAD_ARG
    assert d.fwdmi_linear(None, 4, 8, 16, *none6, -1, lib.F16, None, 0) == lib.ERR_BAD_ARG
    assert d.fwdmi_linear(None, -4, 8, 16, *none6, 0, lib.F16, None, 0) == lib.ERR_BAD_ARG
    assert d.fwdmi_linear(None, 4, 8, 1 << 40, *none6, 0, lib.F16, None, 0) == lib.ERR_BAD_ARG
    assert d.fwdmi_linear(None, 4, 8, 16, *none6, 0, lib.F16, None, 0) == lib.ERR_BAD_ARG            # null pointers
    assert d.fwdmi_linear(None, 0, 8, 16, *none6, 0, lib.F16, None, 0) == lib.OK                     # nothing to do
    need = d.fwdmi_linear_workspace(64, 64, 1 << 16, lib.F16)
    assert need > 0                                                                                # a long sum is split
    some = [64, 64, None, None, 64, None]
    assert d.fwdmi_linear(None, 64, 64, 1 << 16, *some, 0, lib.F16, 64, need - 1) == lib.ERR_BAD_ARG
    assert "workspace" in lib.last_error()
    assert d.fwdmi_linear(None, 64, 64, 1 << 16, *some, 0, lib.F16, 72, need) == lib.ERR_BAD_ARG     # off its boundary
    none7 = [None] * 7
    assert d.fwdmi_linear_backward(None, 4, 8, 16, *none7, 0, lib.BOOL, None, 0) == lib.ERR_UNSUPPORTED
    assert d.fwdmi_linear_backward(None, 4, 8, 16, *none7, 0, lib.F16, None, 0) == lib.ERR_BAD_ARG
    args = [64, 64, 64, None, 64, 64, 64]
    assert d.fwdmi_linear_backward(None, 4, 8, 16, *args, lib.ACT_GELU, lib.F16, 64, 1 << 20) == lib.ERR_BAD_ARG
    assert "pre-activation" in lib.last_error()
    assert d.fwdmi_linear_backward(None, 4, 8, 16, *args, lib.ACT_NONE, lib.F16, None, 0) == lib.ERR_BAD_ARG
    assert "workspace" in lib.last_error()


def test_linear_workspace_sizes():
    d = lib.dll
    assert d.fwdmi_linear_workspace(0, 8, 8, lib.F16) == 0 and d.fwdmi_linear_workspace(8, 8, -1, lib.F16) == 0
    assert d.fwdmi_linear_workspace(8, 8, 8, lib.I32) == 0
    # dz and the column sums' partials at least
    assert d.fwdmi_linear_backward_workspace(100, 64, 64, lib.ACT_GELU, lib.F16) >= 100 * 64 * 2 + 64 * 4
    assert d.fwdmi_linear_backward_workspace(0, 64, 64, lib.ACT_GELU, lib.F16) == 0


@pytest.mark.skipif(lib.dll.fwdmi_device_count() > 0, reason="made-up addresses: only where nothing can be launched")
def test_launches_that_a_device_cannot_hold_are_refused():
    d, p, big = lib.dll, 1 << 20, (1 << 64) - 1
    call = lambda m, n, k, ptr=p: d.fwdmi_linear(None, m, n, k, p, p, None, None, ptr, None, 0, lib.F16, p, big)
    assert call(1, 1 << 26, 8) == lib.ERR_HIP            # (no device here: it got as far as the launch)
    assert call(1, 1 << 30, 8) == lib.ERR_UNSUPPORTED    # 2^26 workgroups of 256
    assert call(33, 1 << 30, 8) == lib.ERR_UNSUPPORTED
    back = lambda m, n, k: d.fwdmi_linear_backward(None, m, n, k, p, p, p, None, p, None, None, 0, lib.F16, p, big)
    assert back(1 << 20, 8, 1 << 10) == lib.ERR_HIP      # (dx alone)
    assert back(1 << 30, 8, 1 << 10) == lib.ERR_UNSUPPORTED
    width = (1 << 26) + 1
    assert d.fwdmi_layer_norm_forward(None, width, width, *[p] * 9, lib.F16, 1e-5) == lib.ERR_BAD_ARG
    assert d.fwdmi_layer_norm_backward(None, width, width, *[p] * 12, p, big, lib.F16) == lib.ERR_BAD_ARG
    assert d.fwdmi_layer_norm_forward(None, width - 1, width - 1, *[p] * 9, lib.F16, 1e-5) == lib.ERR_HIP


@pytest.mark.skipif(lib.dll.fwdmi_device_count() > 0, reason="made-up addresses: only where nothing can be launched")
def test_arguments_at_the_ends_of_their_types_return_a_status():
    """Every call below returns: refused, nothing to do, or (no device here) a launch that the runtime turns down; and the
    workspace sizes neither wrap round nor fall short of what a call then asks for."""
    import itertools
    import random
    rng = random.Random(3)
    d = lib.dll
    ends = [0, 1, 2, 7, 8, 63, 64, 1000, 4095, 1 << 16, (1 << 30) - 1, 1 << 30, (1 << 30) + 1, (1 << 31) - 1, (1 << 62), -1, -(1 << 62)]
    dtypes = [lib.F32, lib.F16, lib.BF16, lib.I8, lib.I64, -5, 1 << 30]
    allowed = {lib.OK, lib.ERR_BAD_ARG, lib.ERR_UNSUPPORTED, lib.ERR_HIP}
    p = 1 << 20
    for m, n, k in itertools.chain(itertools.product(ends, repeat=3), ((rng.choice(ends) + rng.randint(-3, 3),) * 3 for _ in range(500))):
        dt = rng.choice(dtypes)
        size = d.fwdmi_linear_workspace(m, n, k, dt)
        back = d.fwdmi_linear_backward_workspace(m, n, k, rng.choice([0, 2]), dt)
        assert size < 1 << 60 and back < 1 << 60
        rc = d.fwdmi_linear(None, m, n, k, p, p, p, p, p, p, rng.choice([0, 1, 2, 3, 4, 5, -1]), dt, p, (1 << 64) - 1)
        assert rc in allowed
        if rc == lib.ERR_HIP and size:
            assert d.fwdmi_linear(None, m, n, k, p, p, p, p, p, p, 0, dt, p, size - 1) == lib.ERR_BAD_ARG
            assert d.fwdmi_linear(None, m, n, k, p, p, p, p, p, p, 0, dt, p, size) == lib.ERR_HIP
        rc = d.fwdmi_linear_backward(None, m, n, k, p, p, p, p, p, p, p, rng.choice([0, 1, 2, 3, 4, 5, -1]), dt, p, (1 << 64) - 1)
        assert rc in allowed
    for ld, rows in itertools.product([e for e in ends if abs(e) < 1 << 31], ends):
        n = ld * rows
        if abs(n) >= 1 << 63:
            continue
        dt = rng.choice(dtypes)
        assert d.fwdmi_layer_norm_forward(None, ld, n, *[p] * 9, dt, 1e-5) in allowed
        size = d.fwdmi_layer_norm_backward_workspace(ld, n, 1, dt)
        rc = d.fwdmi_layer_norm_backward(None, ld, n, *[p] * 12, p, (1 << 64) - 1, dt)
        assert rc in allowed
        if rc == lib.ERR_HIP and size:
            assert d.fwdmi_layer_norm_backward(None, ld, n, *[p] * 12, p, size - 1, dt) == lib.ERR_BAD_ARG
