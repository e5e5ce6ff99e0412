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
    assert d.fwdmi_layer_norm_backward(None, 10, 20, *args, 1 << 20, lib.F16) == lib.ERR_BAD_ARG
    assert "workspace" in lib.last_error()


def test_layer_norm_workspace_sizes():
    f = lib.dll.fwdmi_layer_norm_backward_workspace
    assert f(16, 0, lib.F32) == 0 and f(0, 16, lib.F32) == 0 and f(16, 17, lib.F32) == 0 and f(16, 16, lib.I8) == 0
    assert f(1024, 8192 * 1024, lib.F16) >= 3 * 1024 * 4
    assert f(100000, 5 * 100000, lib.F32) >= 5 * 8 + 3 * 100000 * 4
