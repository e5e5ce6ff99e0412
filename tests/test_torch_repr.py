"""What the dense modules print, without a GPU: as much as the modules they stand in for."""
import torch

from forward_amd import torch_ops


def test_swapped_modules_print_what_they_are():
    model = torch.nn.Sequential(torch.nn.Linear(6, 4, bias=False), torch.nn.LayerNorm(4, eps=1e-6))
    torch_ops.replace_dense_modules(model)
    assert repr(model[0]) == "Linear(in_features=6, out_features=4, bias=False)"
    assert repr(model[1]) == "LayerNorm((4,), eps=1e-06)"
    assert repr(torch_ops.Linear(6, 4, activation="gelu")) == "Linear(in_features=6, out_features=4, bias=True, activation='gelu')"
    assert repr(torch_ops.LayerNorm(4, keep_sum=True)) == "LayerNorm((4,), eps=1e-05, keep_sum=True)"
