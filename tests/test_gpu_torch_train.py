"""The differentiable torch ops and modules (linear, layer norm, feed-forward block) against PyTorch's own modules in fp64,
and runs of the embedding launch, the products and the norms together as a model uses them.

Bound of the fp32 comparisons: a sum of n products is off by at most (n + 8) 2^-23 of its magnitudes' sum, which is at most
sqrt(n) times larger than the result's norm for these random operands; four such sums of at most 256 terms lie between an
input and a gradient here, so results agree to 4 * 264 * 16 * 2^-23 = 2e-3 of their largest value at the very worst.
fp16: every stored tensor (at most eight in a row) adds half a step, 2^-12 of its values, and sums of n roundings at
most sqrt(n) more of their norm: 8 * 16 * 2^-12 = 3e-2.
"""
import copy

import numpy as np
import pytest
import torch

from forward_amd import ops, torch_ops, workloads

pytestmark = pytest.mark.gpu
TOL = {torch.float32: 2e-3, torch.float16: 3e-2}


def close(got, want, tol, what):
    got, want = got.detach().double(), want.detach().double()
    assert got.shape == want.shape, what
    err = (got - want).abs().max().item()
    assert err <= tol * max(want.abs().max().item(), 1e-6), "%s: off by %g of %g" % (what, err, want.abs().max().item())


class Reference(torch.nn.Module):
    """The feed-forward block from PyTorch's modules."""

    def __init__(self, hidden, inner, activation):
        super().__init__()
        self.up, self.down = torch.nn.Linear(hidden, inner), torch.nn.Linear(inner, hidden)
        self.norm = torch.nn.LayerNorm(hidden, eps=1e-5)
        self.act = {"gelu": torch.nn.functional.gelu, "silu": torch.nn.functional.silu, "relu": torch.relu,
                    "gelu_tanh": lambda z: torch.nn.functional.gelu(z, approximate="tanh")}[activation]

    def forward(self, x):
        return self.norm(x + self.down(self.act(self.up(x))))


def pair(hidden, inner, activation, dtype, seed=0):
    """A FeedForward of `dtype` and the fp64 reference with the same parameters."""
    torch.manual_seed(seed)
    ref = Reference(hidden, inner, activation).cuda()
    with torch.no_grad():
        ref.norm.weight.normal_(1.0, 0.2)
        ref.norm.bias.normal_(0.0, 0.2)
    mine = torch_ops.FeedForward(hidden, inner, activation=activation, eps=1e-5, device="cuda", dtype=dtype)
    names = (("up.weight",) * 2, ("up.bias",) * 2, ("down.weight",) * 2, ("down.bias",) * 2, ("norm.weight",) * 2,
             ("norm.bias",) * 2)
    own, theirs = dict(mine.named_parameters()), dict(ref.named_parameters())
    with torch.no_grad():
        for a, b in names:
            own[a].copy_(theirs[b])
            theirs[b].copy_(own[a].float())       # what the narrower type holds
    return mine, ref.double(), [(own[a], theirs[b], a) for a, b in names]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("activation", ["gelu", "relu", "silu", "gelu_tanh"])
@pytest.mark.parametrize("tokens", [1, 77])
def test_feed_forward_and_its_gradients(tokens, activation, dtype):
    mine, ref, params = pair(64, 256, activation, dtype, seed=tokens)
    x = torch.randn(tokens, 64, device="cuda").to(dtype).requires_grad_()
    x64 = x.detach().double().requires_grad_()
    dy = torch.randn(tokens, 64, device="cuda").to(dtype)
    y, y64 = mine(x), ref(x64)
    close(y, y64, TOL[dtype], "y")
    y.backward(dy)
    y64.backward(dy.double())
    close(x.grad, x64.grad, TOL[dtype], "x")
    for p, q, name in params:
        assert p.grad.dtype == p.dtype
        close(p.grad, q.grad, TOL[dtype], name)
    with torch.no_grad():
        assert torch.equal(mine(x), y)


def test_pre_norm_residual_stream():
    """Two pre-norm steps: the sum each norm keeps goes on, its gradient comes back through dsum; with and without bias."""
    torch.manual_seed(3)
    for biased in (False, True):
        norms = [torch_ops.LayerNorm(48, keep_sum=True, device="cuda") for _ in range(2)]
        lin = torch_ops.Linear(48, 48, activation="gelu", device="cuda")
        ref = [torch.nn.LayerNorm(48).cuda().double() for _ in range(2)]
        lin64 = copy.deepcopy(torch.nn.Linear(48, 48)).cuda().double()
        with torch.no_grad():
            lin64.weight.copy_(lin.weight)
            lin64.bias.copy_(lin.bias)
        b = torch.randn(48, device="cuda", requires_grad=True)
        x = torch.randn(30, 48, device="cuda", requires_grad=True)
        b64, x64 = (t.detach().double().requires_grad_() for t in (b, x))
        n1, h1 = norms[0](x, bias=b if biased else None)
        n2, h2 = norms[1](lin(n1), skip=h1)
        (n2 * 2 + h2.sin()).sum().backward()
        g1 = x64 + b64 if biased else x64
        g2 = torch.nn.functional.gelu(lin64(ref[0](g1))) + g1
        (ref[1](g2) * 2 + g2.sin()).sum().backward()
        close(h2, g2, 2e-3, "sum")
        close(x.grad, x64.grad, 2e-3, "x")
        close(lin.weight.grad, lin64.weight.grad, 2e-3, "weight")
        close(norms[0].gamma.grad, ref[0].weight.grad, 2e-3, "gamma")
        if biased:
            close(b.grad, b64.grad, 2e-3, "bias")


def test_gradients_of_the_residual_and_of_parts_alone():
    torch.manual_seed(4)
    lin = torch_ops.Linear(32, 24, activation="silu", device="cuda")
    x, r = torch.randn(9, 32, device="cuda"), torch.randn(9, 24, device="cuda", requires_grad=True)
    lin.weight.requires_grad_(False)
    lin(x, residual=r).sum().backward()
    assert torch.equal(r.grad, torch.ones_like(r)) and lin.weight.grad is None and lin.bias.grad is not None
    lin.bias.requires_grad_(False)
    x.requires_grad_()
    lin(x).sum().backward()
    z = x.detach().double() @ lin.weight.double().t() + lin.bias.double()
    p = torch.sigmoid(z)
    close(x.grad, (p * (1 + z * (1 - p))) @ lin.weight.double(), 2e-3, "x alone")
    h, s = torch_ops.LayerNorm(32, keep_sum=True, device="cuda")(x, skip=x.detach())
    x.grad = None
    s.sum().backward()                              # the sum alone: the norm's output is not used
    assert torch.equal(x.grad, torch.ones_like(x))


def test_an_activation_without_its_preactivation_is_refused():
    x = torch.randn(4, 16, device="cuda", requires_grad=True)
    w = torch.randn(8, 16, device="cuda")
    with pytest.raises(RuntimeError, match="linear_preact"):
        torch.ops.fwdmi.linear(x, w, None, None, "gelu")
    with torch.no_grad():
        torch.ops.fwdmi.linear(x, w, None, None, "gelu")
    torch.ops.fwdmi.linear(x, w, None, None, "none").sum().backward()
    assert x.grad is not None


def test_parameters_of_another_type_and_strided_inputs():
    torch.manual_seed(6)
    lin = torch_ops.Linear(40, 56, device="cuda", dtype=torch.float16)      # half bias
    norm = torch_ops.LayerNorm(56, device="cuda", dtype=torch.bfloat16)     # bf16 gamma and beta under fp16 rows
    x = torch.randn(40, 33, device="cuda", dtype=torch.float16).t().requires_grad_()
    y = norm(lin(x))
    y.backward(torch.randn(56, 33, device="cuda", dtype=torch.float16).t())
    assert lin.bias.grad.dtype == torch.float16 and norm.gamma.grad.dtype == torch.bfloat16 and x.grad.shape == x.shape
    want = torch.nn.functional.layer_norm(x.double() @ lin.weight.double().t() + lin.bias.double(), (56,),
                                          norm.gamma.double(), norm.beta.double(), 1e-5)
    close(y, want, 3e-2, "y")


def test_ops_pass_pytorchs_own_checks():
    x = torch.randn(6, 32, device="cuda", requires_grad=True)
    w, b = torch.randn(16, 32, device="cuda", requires_grad=True), torch.randn(16, device="cuda", requires_grad=True)
    r, g = torch.randn(6, 16, device="cuda"), torch.ones(32, device="cuda", requires_grad=True)
    checks = ("test_schema", "test_autograd_registration", "test_faketensor")
    torch.library.opcheck(torch.ops.fwdmi.linear.default, (x, w, b, r, "none"), test_utils=checks)
    torch.library.opcheck(torch.ops.fwdmi.linear_preact.default, (x, w, b, None, "gelu"), test_utils=checks)
    torch.library.opcheck(torch.ops.fwdmi.layer_norm_train.default, (x, None, g, g, None, 1e-5), test_utils=checks)
    torch.library.opcheck(torch.ops.fwdmi.layer_norm_train_sum.default, (x, x.detach(), g, g, g, 1e-5), test_utils=checks)


def test_swapped_modules_train():
    torch.manual_seed(8)
    model = torch.nn.Sequential(torch.nn.Linear(24, 64), torch.nn.ReLU(), torch.nn.LayerNorm(64), torch.nn.Linear(64, 8)).cuda()
    ref = copy.deepcopy(model).double()
    opt = torch.optim.SGD(model.parameters(), lr=0.1)
    torch_ops.replace_dense_modules(model)
    assert isinstance(model[0], torch_ops.Linear) and isinstance(model[2], torch_ops.LayerNorm)
    x = torch.randn(50, 24, device="cuda")
    model(x).square().mean().backward()
    ref(x.double()).square().mean().backward()
    for p, q in zip(model.parameters(), ref.parameters()):
        close(p.grad, q.grad, 2e-3, "gradient")
    before = [p.detach().clone() for p in model.parameters()]
    opt.step()
    assert all(not torch.equal(a, b) for a, b in zip(before, model.parameters()))


def test_embedding_launch_products_and_norms_together():
    """A BERT layer's dense half behind the embedding launch, on the BERT-base workload's tables: fp16, no gradients."""
    wl = workloads.config3(variant=2, batch=4, seq=32)
    f32 = lambda a: torch.from_numpy(np.asarray(a, np.float32)).cuda()
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()
    emb = torch_ops.BertEmbeddings(dev(wl.word), dev(wl.pos), dev(wl.tok), f32(wl.gamma), f32(wl.beta), eps=wl.eps)
    mine, ref, _ = pair(768, 1024, "gelu", torch.float16, seed=2)
    ids, seg, msk = (dev(a.T.astype(np.int64)) for a in (wl.input_ids, wl.segment_ids, wl.input_mask))
    with torch.no_grad():
        h, _ = emb(ids, seg, msk)
        y = mine(h)
        # the inference launch of the framework takes the same place as the norm
        f = torch.ops.fwdmi.linear(mine.up(h), mine.down.weight, None, None, "none")
        z = torch.ops.fwdmi.skip_layer_norm(f, h, mine.norm.gamma, mine.norm.beta, mine.down.bias, 1e-5)
        want = ref(h.double())
    assert y.shape == (4, 32, 768)
    close(y, want, 3e-2, "feed-forward")
    close(z, want, 3e-2, "through skip_layer_norm")


def test_a_training_step_captured_into_a_graph():
    """Forward and backward of the block in one graph, replayed on new values.  Nothing of an eager run of the same
    parameters is alive during the capture: the eager results come from a copy of the block."""
    mine, _, _ = pair(96, 160, "gelu", torch.float16, seed=9)
    eager = copy.deepcopy(mine)
    x, dy = torch.zeros(64, 96, device="cuda", dtype=torch.float16), torch.zeros(64, 96, device="cuda", dtype=torch.float16)

    def step(block, a, b):
        a = a.detach().requires_grad_()
        y = block(a)
        grads = torch.autograd.grad(y, [a] + list(block.parameters()), b)
        return (y.detach(),) + grads

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            out = step(mine, x, dy)
    torch.cuda.current_stream().wait_stream(side)
    del out
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(mine, x, dy)
    for seed in range(4):
        torch.manual_seed(seed)
        x.copy_(torch.randn_like(x))
        dy.copy_(torch.randn_like(dy))
        want = step(eager, x, dy)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), seed


def test_gradients_on_another_stream():
    mine, _, _ = pair(96, 160, "gelu", torch.float32, seed=10)
    x = torch.randn(200, 96, device="cuda")
    mine(x).square().sum().backward()
    want = [p.grad.clone() for p in mine.parameters()]
    mine.zero_grad()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        mine(x).square().sum().backward()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p.grad, w) for p, w in zip(mine.parameters(), want))
