"""replace_dense_modules and the from_torch constructors on layers that are more than their parameters, without a GPU."""
import copy

import pytest
import torch
from torch.nn.utils import parametrize, prune, spectral_norm, weight_norm

from forward_amd import torch_ops


class Twice(torch.nn.Module):
    def forward(self, w):
        return w * 2


def forward_of_its_own(m):
    m.forward = lambda x: x
    return m


def hooked(kind):
    def add(m):
        getattr(m, kind)(lambda *args: None)
        return m
    return add


def parametrized(m):
    parametrize.register_parametrization(m, "weight", Twice())
    return m


def pruned(m):
    prune.l1_unstructured(m, "weight", amount=0.5)
    return m


CHANGES = {
    "weight_norm": weight_norm, "spectral_norm": spectral_norm, "prune": pruned, "parametrization": parametrized,
    "forward": forward_of_its_own, "buffer": lambda m: (m.register_buffer("scale", torch.ones(1)), m)[1],
    "child": lambda m: (m.add_module("adapter", torch.nn.Identity()), m)[1],
}
CHANGES.update({k: hooked(k) for k in ("register_forward_hook", "register_forward_pre_hook", "register_full_backward_hook",
                                       "register_full_backward_pre_hook", "register_state_dict_pre_hook",
                                       "register_load_state_dict_post_hook")})


@pytest.mark.filterwarnings("ignore")          # (PyTorch's newer names for weight_norm)
@pytest.mark.parametrize("change", list(CHANGES))
def test_layers_that_are_more_than_their_parameters_stay(change):
    layer = CHANGES[change](torch.nn.Linear(6, 4))
    model = torch.nn.Sequential(layer, torch.nn.Linear(4, 4))
    keys, x = list(model.state_dict()), torch.randn(3, 6)
    params = dict(model.named_parameters())
    want = layer(x).detach().clone()
    torch_ops.replace_dense_modules(model)
    assert model[0] is layer and isinstance(model[1], torch_ops.Linear)
    assert list(model.state_dict()) == keys
    after = dict(model.named_parameters())
    assert list(after) == list(params) and all(after[k] is params[k] for k in params)
    if change != "spectral_norm":              # (a power iteration moves its weight at every call)
        assert torch.equal(model[0](x), want)
    with pytest.raises(NotImplementedError):
        torch_ops.Linear.from_torch(layer)


@pytest.mark.parametrize("change", ["forward", "register_forward_hook", "register_forward_pre_hook", "register_full_backward_hook", "buffer"])
def test_norms_that_are_more_than_their_parameters_stay(change):
    norm = CHANGES[change](torch.nn.LayerNorm(4))
    model = torch.nn.Sequential(norm, torch.nn.LayerNorm(4), torch.nn.LayerNorm(4, bias=False), torch.nn.LayerNorm(4, elementwise_affine=False))
    torch_ops.replace_dense_modules(model)
    assert model[0] is norm and isinstance(model[1], torch_ops.LayerNorm)
    assert type(model[2]) is torch.nn.LayerNorm and type(model[3]) is torch.nn.LayerNorm
    with pytest.raises(NotImplementedError):
        torch_ops.LayerNorm.from_torch(norm)


@pytest.mark.filterwarnings("ignore")
def test_a_weight_under_weight_norm_still_trains_and_loads():
    model = torch.nn.Sequential(weight_norm(torch.nn.Linear(5, 3)))
    other = copy.deepcopy(model.state_dict())
    torch_ops.replace_dense_modules(model)
    x = torch.randn(2, 5)
    before = model(x)
    before.square().sum().backward()
    assert all(p.grad is not None for p in model.parameters())
    torch.optim.SGD(model.parameters(), lr=0.1).step()
    assert not torch.equal(model(x), before)
    model.load_state_dict(other)
    assert torch.equal(model(x), before)


def test_the_training_flag_goes_along():
    model = torch.nn.Sequential(torch.nn.Linear(4, 4), torch.nn.LayerNorm(4)).eval()
    torch_ops.replace_dense_modules(model)
    assert isinstance(model[0], torch_ops.Linear) and not any(m.training for m in model.modules())
    assert torch_ops.Linear.from_torch(torch.nn.Linear(4, 4)).training


def test_a_layer_in_two_places_stays_one():
    layer, norm = torch.nn.Linear(4, 4), torch.nn.LayerNorm(4)
    model = torch.nn.Sequential(layer, norm, layer, torch.nn.Sequential(layer, norm), torch.nn.ModuleDict({"a": layer}))
    count = sum(1 for _ in model.parameters())
    torch_ops.replace_dense_modules(model)
    assert isinstance(model[0], torch_ops.Linear) and isinstance(model[1], torch_ops.LayerNorm)
    assert model[2] is model[0] and model[3][0] is model[0] and model[3][1] is model[1] and model[4]["a"] is model[0]
    assert sum(1 for _ in model.parameters()) == count and model[0].weight is layer.weight


def test_the_model_itself_is_returned_as_it_is():
    layer = torch.nn.Linear(4, 4)
    assert torch_ops.replace_dense_modules(layer) is layer and type(layer) is torch.nn.Linear
