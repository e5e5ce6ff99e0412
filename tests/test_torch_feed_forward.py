"""The feed-forward block calls its modules as modules: what is hooked to them takes part.  Shapes alone, without a GPU."""
import pytest
import torch
from torch.nn.utils import weight_norm

from forward_amd import torch_ops


def test_hooks_of_every_part_run():
    block, seen = torch_ops.FeedForward(16, 32, device="meta"), []
    for name in ("up", "down", "norm"):
        getattr(block, name).register_forward_hook(lambda m, args, out, name=name: seen.append((name, tuple(out.shape))))
    assert block(torch.empty(3, 5, 16, device="meta")).shape == (3, 5, 16)
    assert seen == [("up", (3, 5, 32)), ("down", (3, 5, 16)), ("norm", (3, 5, 16))]


@pytest.mark.filterwarnings("ignore")          # (PyTorch's newer names for weight_norm)
@pytest.mark.parametrize("part", ["up", "down"])
def test_a_recomputed_weight_is_recomputed_at_every_call(part):
    block = torch_ops.FeedForward(16, 32, device="meta")
    weight_norm(getattr(block, part))
    first = getattr(block, part).weight
    block(torch.empty(3, 16, device="meta"))
    assert getattr(block, part).weight is not first


def test_a_product_without_its_bias(monkeypatch):
    lin, seen = torch_ops.Linear(16, 8, activation="gelu", device="meta"), []
    op = torch.ops.fwdmi.linear_preact
    monkeypatch.setattr(torch.ops.fwdmi, "linear_preact", lambda x, w, bias, *rest: (seen.append(bias), op(x, w, bias, *rest))[1])
    for add in (False, True):
        lin(torch.empty(2, 16, device="meta"), add_bias=add)
    assert seen[0] is None and seen[1] is lin.bias
