"""Rows longer than the norm's launchers take, without a GPU: refused by the tensor-level wrappers, whose lengths have 64 bits
where the launcher's argument has 32."""
import pytest
import torch

from forward_amd import ops


@pytest.fixture(autouse=True)
def shapes_alone(monkeypatch):
    monkeypatch.setattr(ops, "_dev", lambda t, name: t)
    monkeypatch.setattr(ops, "_away", lambda x, stream: None)
    monkeypatch.setattr(ops, "_raw_stream", lambda device: 0)


@pytest.mark.parametrize("ld", [(1 << 26) + 1, (1 << 31) + 8, (1 << 32) + 8, (1 << 33)])
def test_rows_past_the_limit_are_refused(ld):
    plane = lambda: torch.empty(1, ld, dtype=torch.float16, device="meta")
    vec, one = torch.empty(ld, device="meta"), torch.empty(1, device="meta")
    with pytest.raises(ValueError, match="2\\^26"):
        ops.layer_norm_forward(plane(), vec, vec)
    with pytest.raises(ValueError, match="2\\^26"):
        ops.layer_norm_backward(plane(), plane(), vec, one, one)
