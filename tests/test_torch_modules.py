"""The dense modules as replacements of PyTorch's, without a GPU: names, sharing, attributes."""
import copy

import torch

from forward_amd import torch_ops


def test_swapped_modules_keep_names_and_parameters():
    model = torch.nn.TransformerEncoderLayer(16, 2, dim_feedforward=32, activation="gelu", batch_first=True)
    ref = copy.deepcopy(model)
    before, keys = dict(model.named_parameters()), list(model.state_dict())
    torch_ops.replace_dense_modules(model)
    assert isinstance(model.linear1, torch_ops.Linear) and isinstance(model.norm2, torch_ops.LayerNorm)
    after = dict(model.named_parameters())
    assert list(model.state_dict()) == keys and all(after[k] is before[k] for k in before)
    model.load_state_dict(ref.state_dict())
    assert (model.linear1.in_features, model.linear1.out_features) == (16, 32)
    assert model.norm1.normalized_shape == (16,) and model.norm1.gamma is model.norm1.weight and model.norm1.beta is model.norm1.bias


def test_what_reads_a_swapped_layers_attributes_still_finds_them():
    model = torch.nn.TransformerEncoderLayer(16, 2, dim_feedforward=32, batch_first=True).eval()
    x = torch.randn(3, 5, 16)
    with torch.no_grad():                       # (PyTorch's own fused layer, which takes the parameters themselves)
        want = model(x)
        torch_ops.replace_dense_modules(model)
        assert torch.equal(model(x), want)


def test_bias_is_optional_and_kept_so():
    m = torch_ops.Linear.from_torch(torch.nn.Linear(4, 6, bias=False))
    assert m.bias is None and list(m.state_dict()) == ["weight"]
    assert list(torch_ops.Linear(4, 6).state_dict()) == ["weight", "bias"]
    assert list(torch_ops.LayerNorm(4).state_dict()) == ["weight", "bias"]
    n = torch.nn.LayerNorm((2, 4))
    assert type(torch_ops.replace_dense_modules(torch.nn.Sequential(n))[0]) is torch.nn.LayerNorm
