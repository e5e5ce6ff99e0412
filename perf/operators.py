"""Cases of the dense half of a transformer layer: layer norm and the fused linear layer, each forward and backward.

``run`` computes an operator either in its plain form (elementary torch operations in fp32, rounded once at the
end) or, with ``own`` set, through ``forward_amd.ops``.  ``exact`` evaluates the definitions in fp64.

    layer norm   h = x (+ skip) (+ bias);  y = gamma * (h - mean) * rstd + beta,  rstd = 1 / sqrt(var + eps)
                 outputs y, mean, rstd and, for pre-norm layers, h itself
    its gradient dx = rstd * (g - mean(g) - xhat * mean(g * xhat)) (+ dsum),  g = dy * gamma;
                 dgamma = sum dy * xhat, dbeta = sum dy, dbias = sum of dx without dsum, over the rows
    linear       z = x w^T + b;  y = act(z) (+ residual);  z is kept where a backward pass follows
    its gradient dz = dy * act'(z);  dx = dz w, dw = dz^T x, db = sum of dz over the rows
"""
import math

import torch

own = False

_TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def _size(case):
    return 4 if case["type"] == "fp32" else 2


# ---- cases -------------------------------------------------------------------------------------------------

def listed():
    return [
        # one token of a BERT-large encoder: what its latency costs
        dict(name="norm forward one token", op="norm_forward", type="fp16", rows=1, width=1024,
             skip=True, bias=True, keep_sum=False),
        # a batch of 16 sequences of 512 tokens, post-norm, the previous product's bias folded in
        dict(name="norm forward 8192 tokens post-norm", op="norm_forward", type="fp16", rows=8192, width=1024,
             skip=True, bias=True, keep_sum=False),
        # the residual stream of a wide pre-norm layer: the sum goes on beside the normalised rows
        dict(name="norm forward wide pre-norm", op="norm_forward", type="bf16", rows=8192, width=4096,
             skip=True, bias=False, keep_sum=True),
        # a ragged batch at BERT-base's width, master precision
        dict(name="norm backward 509 tokens", op="norm_backward", type="fp32", rows=509, width=768,
             skip=False, bias=False, keep_sum=False),
        # a training step's post-norm at BERT-large's width
        dict(name="norm backward 8192 tokens post-norm", op="norm_backward", type="bf16", rows=8192, width=1024,
             skip=True, bias=True, keep_sum=False),
        # the gradient that comes down the residual stream joins in; rows that do not cut into vectors
        dict(name="norm backward odd width pre-norm", op="norm_backward", type="fp16", rows=4099, width=1531,
             skip=False, bias=False, keep_sum=True),
        # one token through the first product of a feed-forward block: a pass over the weights
        dict(name="linear one token", op="linear", type="fp16", tokens=1, width=1024, out=4096,
             act="gelu", bias=True, residual=False, keep_z=False),
        # a short batch through the second product, the residual added on the way out
        dict(name="linear 384 tokens with residual", op="linear", type="fp16", tokens=384, width=4096, out=1024,
             act="none", bias=True, residual=True, keep_z=False),
        # training: the first product of a feed-forward block, pre-activation kept
        dict(name="linear 8192 tokens training", op="linear", type="bf16", tokens=8192, width=1024, out=4096,
             act="gelu", bias=True, residual=False, keep_z=True),
        # a head of odd sizes in master precision
        dict(name="linear odd sizes fp32", op="linear", type="fp32", tokens=1003, width=1001, out=517,
             act="relu", bias=True, residual=True, keep_z=False),
        # the gradient of a projection at BERT-base's width, a ragged batch
        dict(name="linear backward 771 tokens", op="linear_backward", type="fp16", tokens=771, width=768, out=1011,
             act="none", bias=True),
        # the gradient of the training case above
        dict(name="linear backward 8192 tokens", op="linear_backward", type="bf16", tokens=8192, width=1024, out=4096,
             act="gelu", bias=True),
    ]


_MOST_ELEMENTS = 8192 * 4096               # the largest listed norm
_MOST_PRODUCTS = 8192 * 1024 * 4096        # the largest listed product


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A width between lo and hi: mostly a multiple of 8 or of 64, as models have them, else any number."""
    n = _log_int(rng, lo, hi)
    step = rng.choice([64, 64, 8, 1])
    return min(hi, max(lo, n // step * step))


def draw(rng):
    op = rng.choice(["norm_forward", "norm_backward", "linear", "linear_backward"])
    kind = rng.choice(["fp16", "bf16", "fp32"])
    if op.startswith("norm"):
        width = _width(rng, 32, 12288)
        rows = min(_log_int(rng, 1, 32768), _MOST_ELEMENTS // width)
        skip = rng.random() < 0.6
        return dict(op=op, type=kind, rows=rows, width=width, skip=skip, bias=rng.random() < 0.4,
                    keep_sum=rng.random() < 0.4)
    width, out = _width(rng, 64, 8192), _width(rng, 64, 8192)
    tokens = _log_int(rng, 1, 16384)
    # fp32 products run at about a sixteenth of the 16-bit rate: a share of the size keeps a case's cost in bounds
    most = _MOST_PRODUCTS // (8 if kind == "fp32" else 1)
    tokens = max(1, min(tokens, most // (width * out)))
    case = dict(op=op, type=kind, tokens=tokens, width=width, out=out,
                act=rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]), bias=rng.random() < 0.7)
    if op == "linear":
        case.update(residual=rng.random() < 0.4, keep_z=rng.random() < 0.4)
    return case


# ---- inputs ------------------------------------------------------------------------------------------------

def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind = _TYPES[case["type"]]

    def normal(*shape, mean=0.0, std=1.0, type=kind):
        return (torch.randn(shape, generator=gen, device="cuda") * std + mean).to(type)

    s = dict(case=case)
    if case["op"].startswith("norm"):
        rows, width = case["rows"], case["width"]
        s["eps"] = 1e-5
        s["x"] = normal(rows, width)
        if case["op"] == "norm_forward" or not case["keep_sum"]:
            # (the backward pass of a layer that kept its sum reads the sum as x)
            s["skip"] = normal(rows, width) if case["skip"] else None
            s["bias"] = normal(width, std=0.02, type=torch.float32) if case["bias"] else None
        else:
            s["skip"] = s["bias"] = None
        s["gamma"] = normal(width, mean=1.0, std=0.1, type=torch.float32)
        s["beta"] = normal(width, std=0.1, type=torch.float32)
        if case["op"] == "norm_backward":
            s["dy"] = normal(rows, width, std=0.1)
            s["dsum"] = normal(rows, width, std=0.1) if case["keep_sum"] else None
            h = s["x"].double()
            if s["skip"] is not None:
                h += s["skip"].double()
            if s["bias"] is not None:
                h += s["bias"].double()
            s["mean"] = h.mean(1).float()
            s["rstd"] = (h.var(1, unbiased=False) + s["eps"]).rsqrt().float()
        return s
    tokens, width, out = case["tokens"], case["width"], case["out"]
    s["x"] = normal(tokens, width)
    s["w"] = normal(out, width, std=0.02)
    s["b"] = normal(out, std=0.02, type=torch.float32) if case["bias"] else None
    if case["op"] == "linear":
        s["residual"] = normal(tokens, out) if case["residual"] else None
    else:
        s["dy"] = normal(tokens, out, std=0.1)
        s["z"] = None
        if case["act"] != "none":
            z = s["x"].float() @ s["w"].float().t()
            s["z"] = (z if s["b"] is None else z + s["b"]).to(kind)
    return s


# ---- one pass ----------------------------------------------------------------------------------------------

def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    from forward_amd import ops
    case = s["case"]
    if case["op"] == "norm_forward":
        return ops.layer_norm_forward(s["x"], s["gamma"], s["beta"], skip=s["skip"], bias=s["bias"], eps=s["eps"],
                                      want_sum=case["keep_sum"])
    if case["op"] == "norm_backward":
        return ops.layer_norm_backward(s["dy"], s["x"], s["gamma"], s["mean"], s["rstd"], skip=s["skip"],
                                       bias=s["bias"], dsum=s["dsum"])
    if case["op"] == "linear":
        return ops.linear(s["x"], s["w"], bias=s["b"], activation=case["act"], residual=s["residual"],
                          want_preact=case["keep_z"])
    return ops.linear_backward(s["dy"], s["x"], s["w"], preact=s["z"], activation=case["act"],
                               want_dbias=case["bias"])


_SQRT_2_OVER_PI = math.sqrt(2.0 / math.pi)


def _act(z, name):
    if name == "relu":
        return torch.clamp(z, min=0)
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(_SQRT_2_OVER_PI * (z + 0.044715 * z * z * z)))
    if name == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _act_slope(z, name):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        t = torch.tanh(_SQRT_2_OVER_PI * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * _SQRT_2_OVER_PI * (1 + 3 * 0.044715 * z * z)
    p = 1 / (1 + torch.exp(-z))
    return p * (1 + z * (1 - p))


def _norm_input(s):
    h = s["x"].float()
    if s["skip"] is not None:
        h = h + s["skip"].float()
    if s["bias"] is not None:
        h = h + s["bias"]
    return h


def _run_plain(s):
    case = s["case"]
    kind = _TYPES[case["type"]]
    if case["op"] == "norm_forward":
        h = _norm_input(s)
        mean = h.mean(1)
        c = h - mean[:, None]
        rstd = 1 / torch.sqrt((c * c).mean(1) + s["eps"])
        y = (c * rstd[:, None] * s["gamma"] + s["beta"]).to(kind)
        return (y, mean, rstd, h.to(kind)) if case["keep_sum"] else (y, mean, rstd)
    if case["op"] == "norm_backward":
        xhat = (_norm_input(s) - s["mean"][:, None]) * s["rstd"][:, None]
        dy = s["dy"].float()
        g = dy * s["gamma"]
        dh = (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True)) * s["rstd"][:, None]
        dx = (dh if s["dsum"] is None else dh + s["dsum"].float()).to(kind)
        out = (dx, (dy * xhat).sum(0), dy.sum(0))
        return out if s["bias"] is None else out + (dh.sum(0),)
    x, w = s["x"].float(), s["w"].float()
    if case["op"] == "linear":
        z = torch.matmul(x, w.t())
        if s["b"] is not None:
            z = z + s["b"]
        y = _act(z, case["act"])
        if s["residual"] is not None:
            y = y + s["residual"].float()
        return (y.to(kind), z.to(kind)) if case["keep_z"] else y.to(kind)
    dz = s["dy"].float()
    if s["z"] is not None:
        dz = dz * _act_slope(s["z"].float(), case["act"])
    out = (torch.matmul(dz, w).to(kind), torch.matmul(dz.t(), x).to(kind))
    return out + (dz.sum(0),) if case["bias"] else out


# ---- cost and exact values -----------------------------------------------------------------------------------

def work(case):
    size = _size(case)
    if case["op"].startswith("norm"):
        rows, width = case["rows"], case["width"]
        n = rows * width
        if case["op"] == "norm_forward":
            planes = 2 + case["skip"] + case["keep_sum"]
            vectors = 2 + case["bias"]
            flops = 8 * n
        elif case["keep_sum"]:
            planes, vectors, flops = 4, 3, 15 * n
        else:
            planes = 3 + case["skip"]
            vectors = 3 + 2 * case["bias"]
            flops = 14 * n
        return {"bytes": planes * n * size + vectors * width * 4 + rows * 8, "flops": flops}
    tokens, width, out = case["tokens"], case["width"], case["out"]
    if case["op"] == "linear":
        elements = tokens * width + out * width + tokens * out * (1 + case["residual"] + case["keep_z"])
        return {"bytes": elements * size + 4 * out * case["bias"], "flops": 2 * tokens * width * out}
    elements = 2 * tokens * width + 2 * out * width + tokens * out * (1 + (case["act"] != "none"))
    return {"bytes": elements * size + 4 * out * case["bias"], "flops": 4 * tokens * width * out}


def exact(case, seed):
    s = {k: v.double() if isinstance(v, torch.Tensor) else v for k, v in prepare(case, seed).items()}
    zero = torch.zeros((), dtype=torch.float64, device="cuda")
    some = lambda t: zero if t is None else t
    if case["op"].startswith("norm"):
        h = s["x"] + some(s["skip"]) + some(s["bias"])
        if case["op"] == "norm_forward":
            var, mean = torch.var_mean(h, 1, correction=0)
            rstd = (var + s["eps"]) ** -0.5
            y = torch.addcmul(s["beta"], (h - mean.unsqueeze(1)) * rstd.unsqueeze(1), s["gamma"])
            return (y, mean, rstd, h) if case["keep_sum"] else (y, mean, rstd)
        r = s["rstd"].unsqueeze(1)
        xhat = (h - s["mean"].unsqueeze(1)) * r
        g = s["dy"] * s["gamma"]
        dots = torch.stack([g.sum(1), (g * xhat).sum(1)]) / case["width"]
        dh = r * (g - dots[0].unsqueeze(1) - dots[1].unsqueeze(1) * xhat)
        ones = torch.ones(case["rows"], dtype=torch.float64, device="cuda")
        out = (dh + some(s["dsum"]), ones @ (s["dy"] * xhat), ones @ s["dy"])
        return out if s["bias"] is None else out + (ones @ dh,)
    if case["op"] == "linear":
        z = s["x"] @ s["w"].T + some(s["b"])
        y = _exact_act(z, case["act"])[0] + some(s["residual"])
        return (y, z) if case["keep_z"] else y
    dz = s["dy"] if s["z"] is None else s["dy"] * _exact_act(s["z"], case["act"])[1]
    out = (dz @ s["w"], dz.T @ s["x"])
    return out + (torch.ones(case["tokens"], dtype=torch.float64, device="cuda") @ dz,) if case["bias"] else out


def _exact_act(z, name):
    """The activation and its slope in fp64."""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        return z.relu(), torch.heaviside(z, torch.zeros((), dtype=z.dtype, device=z.device))
    if name == "gelu":
        phi = torch.special.ndtr(z)
        return z * phi, phi + z * torch.exp(-z * z / 2) * (2 * math.pi) ** -0.5
    if name == "gelu_tanh":
        # (1 + tanh(u)) / 2 is the logistic function of 2 u
        p = torch.sigmoid(2 * _SQRT_2_OVER_PI * (z + 0.044715 * z ** 3))
        return z * p, p + z * p * (1 - p) * 2 * _SQRT_2_OVER_PI * (1 + 0.134145 * z ** 2)
    p = torch.sigmoid(z)
    return z * p, p + z * p * (1 - p)
