"""PyTorch adapter: the kernels as ``torch.ops.fwdmi.*`` custom ops plus drop-in modules.

Counterpart of the reference's torch-side glue (``TorchEngine::ParseInput`` / ``CopyFromBuffers``,
source/fwd_torch/torch_engine/torch_engine.cpp:134-174): there, int64 ids are copied to int32 and
outputs are copied out of engine buffers; here the bag ops consume int32 or int64 ids as they are and
write straight into the tensors they return, or, in their ``*_out`` forms, into tensors the caller
supplies (declared to PyTorch as mutated arguments), so that a serving loop reuses its buffers.
``linear`` and ``layer_norm_train`` (with their ``*_preact`` / ``*_sum`` forms) are differentiable and back the modules
``Linear``, ``LayerNorm`` and ``FeedForward``, which train as well as serve.
The BERT ops (``emb_layer_norm``, ``emb_skip_layer_norm``) take the ``[B, S]`` tensors a PyTorch model
holds (``batch_major``) or the plugin's ``[S, B]``.  ``nn.EmbeddingBag`` / ``nn.Embedding`` modules of an
inference model can be swapped for the HIP path with ``replace_embedding_modules``.
"""
from typing import List, Optional, Tuple

import torch

from . import ops

_MODE = {"sum": 0, "mean": 1, "max": 2}


@torch.library.custom_op("fwdmi::embedding_bag", mutates_args=())
def embedding_bag(weight: torch.Tensor, indices: torch.Tensor, offsets: torch.Tensor, mode: int,
                  per_sample_weights: Optional[torch.Tensor], include_last_offset: bool) -> torch.Tensor:
    return ops.embedding_bag(weight, indices.contiguous(), offsets.contiguous().to(indices.dtype), mode,
                             per_sample_weights=per_sample_weights, include_last_offset=include_last_offset)


@embedding_bag.register_fake
def _(weight, indices, offsets, mode, per_sample_weights, include_last_offset):
    n = offsets.numel() - (1 if include_last_offset else 0)
    return weight.new_empty((n, weight.shape[1]))


@torch.library.custom_op("fwdmi::embedding_bag_group", mutates_args=())
def embedding_bag_group(weights: List[torch.Tensor], indices: List[torch.Tensor], offsets: List[torch.Tensor],
                        mode: int, include_last_offset: bool,
                        per_sample_weights: List[Optional[torch.Tensor]]) -> torch.Tensor:
    """The embedding bags of a sparse stage and their concatenation: ``[B, T*dim]`` from one launch.
    ``per_sample_weights``: one entry per table, ``None`` for a table without weights (sum only)."""
    idt = indices[0].dtype
    psw = [None if w is None else w.to(weights[0].dtype).contiguous() for w in per_sample_weights]
    if all(w is None for w in psw):
        psw = None
    return ops.embedding_bag_group(weights, [i.contiguous() for i in indices],
                                   [o.contiguous().to(idt) for o in offsets], mode,
                                   include_last_offset=include_last_offset, per_sample_weights=psw)


@embedding_bag_group.register_fake
def _(weights, indices, offsets, mode, include_last_offset, per_sample_weights):
    n = offsets[0].numel() - (1 if include_last_offset else 0)
    return weights[0].new_empty((n, len(weights) * weights[0].shape[1]))


@torch.library.custom_op("fwdmi::embedding_bag_fixed", mutates_args=())
def embedding_bag_fixed(weight: torch.Tensor, indices: torch.Tensor, mode: int) -> torch.Tensor:
    return ops.embedding_bag_fixed(weight, indices.contiguous(), mode)


@embedding_bag_fixed.register_fake
def _(weight, indices, mode):
    return weight.new_empty((indices.shape[0], weight.shape[1]))


@torch.library.custom_op("fwdmi::embedding", mutates_args=())
def embedding(weight: torch.Tensor, indices: torch.Tensor) -> torch.Tensor:
    """``aten::embedding`` as the plain row gather (op 999); out-of-range ids give zero rows."""
    flat = indices.contiguous().reshape(1, -1)
    return ops.gather(weight, flat).reshape(tuple(indices.shape) + (weight.shape[1],))


@embedding.register_fake
def _(weight, indices):
    return weight.new_empty(tuple(indices.shape) + (weight.shape[1],))


@torch.library.custom_op("fwdmi::skip_layer_norm", mutates_args=())
def skip_layer_norm(x: torch.Tensor, skip: Optional[torch.Tensor], gamma: torch.Tensor, beta: torch.Tensor,
                    bias: Optional[torch.Tensor], eps: float) -> torch.Tensor:
    f = lambda t: None if t is None else t.float().contiguous()
    return ops.skip_layer_norm(x.contiguous(), f(gamma), f(beta), skip=None if skip is None else skip.contiguous(),
                               bias=f(bias), eps=eps)


@skip_layer_norm.register_fake
def _(x, skip, gamma, beta, bias, eps):
    return torch.empty_like(x)


def _i32(t):
    """ids of the BERT ops: the launchers read int32 (int64 ids are narrowed, as the reference's
    ParseInput does for every integer input, torch_engine.cpp:134-140)."""
    return None if t is None else t.to(torch.int32).contiguous()


def _f32(t):
    return None if t is None else t.float().contiguous()


@torch.library.custom_op("fwdmi::emb_layer_norm", mutates_args=())
def emb_layer_norm(input_ids: torch.Tensor, segment_ids: torch.Tensor, input_mask: Optional[torch.Tensor],
                   word: torch.Tensor, pos: torch.Tensor, tok: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor,
                   eps: float, batch_major: bool) -> List[torch.Tensor]:
    """BERT embedding + LayerNorm: ``[out, mask_idx]``.  ids / mask are ``[B, S]`` with ``batch_major``
    (out ``[B, S, H]``), else the plugin's ``[S, B]`` (out ``[S, B, H]``); ``mask_idx`` is int32 ``[B]``
    (empty without a mask)."""
    out, midx = ops.emb_layer_norm(_i32(input_ids), _i32(segment_ids), _i32(input_mask), word, pos, tok, _f32(gamma),
                                   _f32(beta), eps=eps, batch_major=batch_major)
    return [out, midx if midx is not None else torch.empty((0,), dtype=torch.int32, device=out.device)]


@emb_layer_norm.register_fake
def _(input_ids, segment_ids, input_mask, word, pos, tok, gamma, beta, eps, batch_major):
    b = input_ids.shape[0] if batch_major else input_ids.shape[1]
    return [word.new_empty(tuple(input_ids.shape) + (word.shape[1],)),
            input_ids.new_empty((b if input_mask is not None else 0,), dtype=torch.int32)]


@torch.library.custom_op("fwdmi::emb_skip_layer_norm", mutates_args=())
def emb_skip_layer_norm(input_ids: torch.Tensor, segment_ids: torch.Tensor, input_mask: Optional[torch.Tensor],
                        word: torch.Tensor, pos: torch.Tensor, tok: torch.Tensor, gamma: torch.Tensor,
                        beta: torch.Tensor, eps: float, skip: torch.Tensor, gamma2: torch.Tensor, beta2: torch.Tensor,
                        bias2: Optional[torch.Tensor], eps2: float, batch_major: bool) -> List[torch.Tensor]:
    """The embedding stage and the SkipLayerNorm that consumes it in one launch:
    ``out = LN2(LN(word + pos + tok) + skip (+ bias2))``, equal bit for bit to the two ops in a row."""
    out, midx = ops.emb_layer_norm(_i32(input_ids), _i32(segment_ids), _i32(input_mask), word, pos, tok, _f32(gamma),
                                   _f32(beta), eps=eps, batch_major=batch_major, skip=skip.contiguous(),
                                   gamma2=_f32(gamma2), beta2=_f32(beta2), bias2=_f32(bias2), eps2=eps2)
    return [out, midx if midx is not None else torch.empty((0,), dtype=torch.int32, device=out.device)]


@emb_skip_layer_norm.register_fake
def _(input_ids, segment_ids, input_mask, word, pos, tok, gamma, beta, eps, skip, gamma2, beta2, bias2, eps2, batch_major):
    b = input_ids.shape[0] if batch_major else input_ids.shape[1]
    return [word.new_empty(tuple(input_ids.shape) + (word.shape[1],)),
            input_ids.new_empty((b if input_mask is not None else 0,), dtype=torch.int32)]


# ---- forms that write into the caller's tensors ------------------------------------------------
# Where the reference copies every output out of an engine buffer into a fresh tensor
# (TorchEngine::CopyFromBuffers, torch_engine.cpp:150-174), these write the result where the caller
# wants it; PyTorch is told which argument is written (mutates_args), nothing is returned.

@torch.library.custom_op("fwdmi::embedding_bag_out", mutates_args=("out",))
def embedding_bag_out(out: torch.Tensor, weight: torch.Tensor, indices: torch.Tensor, offsets: torch.Tensor, mode: int,
                      per_sample_weights: Optional[torch.Tensor], include_last_offset: bool, out_col: int) -> None:
    """``out[:, out_col : out_col + dim]`` = the bags; ``out`` is ``[n_bags, W]`` of the table's dtype."""
    ops.embedding_bag(weight, indices.contiguous(), offsets.contiguous().to(indices.dtype), mode,
                      per_sample_weights=per_sample_weights, include_last_offset=include_last_offset, out=out,
                      out_col=out_col, out_dtype=out.dtype)


@torch.library.custom_op("fwdmi::embedding_bag_group_out", mutates_args=("out",))
def embedding_bag_group_out(out: torch.Tensor, weights: List[torch.Tensor], indices: List[torch.Tensor],
                            offsets: List[torch.Tensor], mode: int, include_last_offset: bool,
                            per_sample_weights: List[Optional[torch.Tensor]]) -> None:
    idt = indices[0].dtype
    psw = [None if w is None else w.to(weights[0].dtype).contiguous() for w in per_sample_weights]
    if all(w is None for w in psw):
        psw = None
    ops.embedding_bag_group(weights, [i.contiguous() for i in indices], [o.contiguous().to(idt) for o in offsets], mode,
                            include_last_offset=include_last_offset, per_sample_weights=psw, out=out, out_dtype=out.dtype)


@torch.library.custom_op("fwdmi::skip_layer_norm_out", mutates_args=("out",))
def skip_layer_norm_out(out: torch.Tensor, x: torch.Tensor, skip: Optional[torch.Tensor], gamma: torch.Tensor,
                        beta: torch.Tensor, bias: Optional[torch.Tensor], eps: float) -> None:
    """``out``: a tensor of ``x``'s shape and dtype (not ``x`` or ``skip`` themselves)."""
    ops.skip_layer_norm(x.contiguous(), _f32(gamma), _f32(beta), skip=None if skip is None else skip.contiguous(),
                        bias=_f32(bias), eps=eps, out=out)


@torch.library.custom_op("fwdmi::emb_layer_norm_out", mutates_args=("out", "mask_idx"))
def emb_layer_norm_out(out: torch.Tensor, mask_idx: Optional[torch.Tensor], input_ids: torch.Tensor,
                       segment_ids: torch.Tensor, input_mask: Optional[torch.Tensor], word: torch.Tensor,
                       pos: torch.Tensor, tok: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor, eps: float,
                       skip: Optional[torch.Tensor], gamma2: Optional[torch.Tensor], beta2: Optional[torch.Tensor],
                       bias2: Optional[torch.Tensor], eps2: float, batch_major: bool) -> None:
    """Both BERT forms (``skip`` given: the fused embedding + SkipLayerNorm) into ``out`` / ``mask_idx``."""
    ops.emb_layer_norm(_i32(input_ids), _i32(segment_ids), _i32(input_mask), word, pos, tok, _f32(gamma), _f32(beta),
                       eps=eps, batch_major=batch_major, out=out, mask_idx=mask_idx,
                       skip=None if skip is None else skip.contiguous(), gamma2=_f32(gamma2), beta2=_f32(beta2),
                       bias2=_f32(bias2), eps2=eps2)


# ---- the dense half of a layer: differentiable ---------------------------------------------------
# Each forward op keeps what its backward op reads.  Parameters may have any floating type: the launchers take biases and
# norm parameters as float32, and gradients go back in the parameter's own type.

def _opt(t):
    return None if t is None else t.contiguous()


def _like_param(grad, p):
    return None if p is None else grad.to(p.dtype)


@torch.library.custom_op("fwdmi::linear", mutates_args=())
def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor], residual: Optional[torch.Tensor],
           activation: str) -> torch.Tensor:
    """``act(x weight^T + bias) + residual``.  Under autograd with an activation use ``linear_preact``, whose backward pass
    reads what it kept."""
    return ops.linear(x.contiguous(), weight.contiguous(), bias=_f32(bias), activation=activation, residual=_opt(residual))


@linear.register_fake
def _(x, weight, bias, residual, activation):
    return x.new_empty(tuple(x.shape[:-1]) + (weight.shape[0],))


@torch.library.custom_op("fwdmi::linear_preact", mutates_args=())
def linear_preact(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor], residual: Optional[torch.Tensor],
                  activation: str) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(act(z) + residual, z)`` with ``z = x weight^T + bias``; no gradient flows into ``z``."""
    return ops.linear(x.contiguous(), weight.contiguous(), bias=_f32(bias), activation=activation, residual=_opt(residual),
                      want_preact=True)


@linear_preact.register_fake
def _(x, weight, bias, residual, activation):
    y = x.new_empty(tuple(x.shape[:-1]) + (weight.shape[0],))
    return y, torch.empty_like(y)


@torch.library.custom_op("fwdmi::linear_backward", mutates_args=())
def linear_backward(dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, preact: Optional[torch.Tensor],
                    activation: str, want_dx: bool, want_dweight: bool, want_dbias: bool) -> List[torch.Tensor]:
    """Those of ``[dx, dweight, dbias (float32)]`` that are wanted."""
    return list(ops.linear_backward(dy.contiguous(), x.contiguous(), weight.contiguous(), preact=_opt(preact),
                                    activation=activation, want_dx=want_dx, want_dweight=want_dweight,
                                    want_dbias=want_dbias))


@linear_backward.register_fake
def _(dy, x, weight, preact, activation, want_dx, want_dweight, want_dbias):
    out = [torch.empty(x.shape, dtype=x.dtype, device=x.device)] if want_dx else []
    if want_dweight:
        out.append(torch.empty(weight.shape, dtype=weight.dtype, device=weight.device))
    if want_dbias:
        out.append(x.new_empty((weight.shape[0],), dtype=torch.float32))
    return out


def _linear_setup(ctx, inputs, output):
    x, weight, bias, residual, activation = inputs
    z = None
    if isinstance(output, tuple):
        z = output[1]
        ctx.mark_non_differentiable(z)
    elif activation != "none" and any(ctx.needs_input_grad):
        raise RuntimeError("fwdmi::linear keeps no pre-activation for the gradient of %r: use fwdmi::linear_preact" % activation)
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(x, weight, bias, z)
    ctx.activation = activation


def _linear_grad(ctx, dy, *_):
    if dy is None:
        return None, None, None, None, None
    x, weight, bias, z = ctx.saved_tensors
    need = list(ctx.needs_input_grad[:3])
    got = iter(torch.ops.fwdmi.linear_backward(dy, x, weight, z if ctx.activation != "none" else None, ctx.activation,
                                               *need) if any(need) else ())
    dx, dw, db = (next(got) if n else None for n in need)
    return dx, dw, None if db is None else _like_param(db, bias), dy if ctx.needs_input_grad[3] else None, None


linear.register_autograd(_linear_grad, setup_context=_linear_setup)
linear_preact.register_autograd(_linear_grad, setup_context=_linear_setup)


@torch.library.custom_op("fwdmi::layer_norm_train", mutates_args=())
def layer_norm_train(x: torch.Tensor, skip: Optional[torch.Tensor], gamma: torch.Tensor, beta: torch.Tensor,
                     bias: Optional[torch.Tensor], eps: float) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(LN(x + skip + bias), mean, rstd)``; no gradient flows into the statistics."""
    return ops.layer_norm_forward(x.contiguous(), _f32(gamma), _f32(beta), skip=_opt(skip), bias=_f32(bias), eps=eps)


@layer_norm_train.register_fake
def _(x, skip, gamma, beta, bias, eps):
    mean = x.new_empty(x.shape[:-1], dtype=torch.float32)
    return torch.empty(x.shape, dtype=x.dtype, device=x.device), mean, torch.empty_like(mean)


@torch.library.custom_op("fwdmi::layer_norm_train_sum", mutates_args=())
def layer_norm_train_sum(x: torch.Tensor, skip: Optional[torch.Tensor], gamma: torch.Tensor, beta: torch.Tensor,
                         bias: Optional[torch.Tensor], eps: float
                         ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(LN(h), h, mean, rstd)`` with ``h = x + skip + bias``, the residual stream of a pre-norm layer."""
    y, mean, rstd, h = ops.layer_norm_forward(x.contiguous(), _f32(gamma), _f32(beta), skip=_opt(skip), bias=_f32(bias),
                                              eps=eps, want_sum=True)
    return y, h, mean, rstd


@layer_norm_train_sum.register_fake
def _(x, skip, gamma, beta, bias, eps):
    mean = x.new_empty(x.shape[:-1], dtype=torch.float32)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    return y, torch.empty_like(y), mean, torch.empty_like(mean)


@torch.library.custom_op("fwdmi::layer_norm_backward", mutates_args=())
def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, skip: Optional[torch.Tensor], gamma: torch.Tensor,
                        bias: Optional[torch.Tensor], mean: torch.Tensor, rstd: torch.Tensor,
                        dsum: Optional[torch.Tensor]) -> List[torch.Tensor]:
    """``[dx, dgamma, dbeta]``, with a bias ``[dx, dgamma, dbeta, dbias]``; all but dx float32."""
    return list(ops.layer_norm_backward(dy.contiguous(), x.contiguous(), _f32(gamma), mean, rstd, skip=_opt(skip),
                                        bias=_f32(bias), dsum=_opt(dsum)))


@layer_norm_backward.register_fake
def _(dy, x, skip, gamma, bias, mean, rstd, dsum):
    out = [torch.empty(x.shape, dtype=x.dtype, device=x.device)]
    return out + [gamma.new_empty(gamma.shape, dtype=torch.float32) for _ in range(2 if bias is None else 3)]


def _norm_setup(ctx, inputs, output):
    x, skip, gamma, beta, bias, _ = inputs
    mean, rstd = output[-2:]
    ctx.mark_non_differentiable(mean, rstd)
    ctx.set_materialize_grads(False)
    ctx.has_sum = len(output) == 4
    ctx.types = (skip is not None, gamma.dtype, beta.dtype, None if bias is None else bias.dtype)
    # The kept sum stands for x and skip, which then need not be: one tensor that the next layer holds anyhow.  It is rounded,
    # the statistics are of the unrounded sum: xhat is off by half a step of h times rstd.  (A bias needs its own sum of dx.)
    if ctx.has_sum and bias is None:
        x, skip = output[1], None
    ctx.save_for_backward(x, skip, gamma, bias, mean, rstd)


def _norm_grad(ctx, dy, *rest):
    x, skip, gamma, bias, mean, rstd = ctx.saved_tensors
    dsum = rest[0] if ctx.has_sum else None
    had_skip, gamma_t, beta_t, bias_t = ctx.types
    if dy is None:
        if dsum is None:
            return None, None, None, None, None, None
        dy = torch.zeros_like(x)
    got = torch.ops.fwdmi.layer_norm_backward(dy, x, skip, gamma, bias, mean, rstd, dsum)
    dx = got[0]
    return (dx, dx if had_skip else None, got[1].to(gamma_t), got[2].to(beta_t), got[3].to(bias_t) if bias is not None else None,
            None)


layer_norm_train.register_autograd(_norm_grad, setup_context=_norm_setup)
layer_norm_train_sum.register_autograd(_norm_grad, setup_context=_norm_setup)


_HOOKS = ("_forward_hooks", "_forward_pre_hooks", "_backward_hooks", "_backward_pre_hooks", "_state_dict_hooks",
          "_state_dict_pre_hooks", "_load_state_dict_pre_hooks", "_load_state_dict_post_hooks")


def _is_plain(m):
    """Whether layer ``m`` is its weight and its bias and nothing else, so that a module which shares them can stand in its
    place.  A weight that a hook or a parametrization computes from others (weight_norm, spectral_norm, pruning) is no
    parameter of the layer; hooks, buffers and a ``forward`` of its own would be lost."""
    return (set(m._parameters) == {"weight", "bias"} and m.weight is not None and not m._buffers and not m._modules
            and "forward" not in m.__dict__ and not any(getattr(m, h, None) for h in _HOOKS))


def _stand_in(cls, m, what):
    """A module of ``cls`` that shares the parameters of ``m`` and its training flag."""
    if not _is_plain(m):
        raise NotImplementedError("%s with weight and bias of its own and without hooks" % what)
    out = cls.__new__(cls)
    torch.nn.Module.__init__(out)
    out.weight, out.bias, out.training = m.weight, m.bias, m.training
    return out


class Linear(torch.nn.Module):
    """``nn.Linear`` with its activation and a residual in the product's epilogue: ``act(x W^T + b) (+ residual)``.
    Trains and serves; ``activation`` is a key of ``ops.ACTIVATIONS``.  ``forward(x, residual, add_bias=False)`` leaves the
    bias to a norm that follows (``LayerNorm.forward``'s ``bias``)."""

    def __init__(self, in_features, out_features, bias=True, activation="none", device=None, dtype=None):
        super().__init__()
        m = torch.nn.Linear(in_features, out_features, bias=bias, device=device, dtype=dtype)
        self.weight, self.bias = m.weight, m.bias
        self.activation = activation

    @classmethod
    def from_torch(cls, m, activation="none"):
        """Shares the parameters of an ``nn.Linear``.  One whose weight is recomputed (weight_norm and its like) or that has
        hooks is refused."""
        out = _stand_in(cls, m, "a linear layer")
        out.activation = activation
        return out

    in_features = property(lambda self: self.weight.shape[1])
    out_features = property(lambda self: self.weight.shape[0])

    def extra_repr(self):
        return "in_features=%d, out_features=%d, bias=%s%s" % (
            self.in_features, self.out_features, self.bias is not None,
            "" if self.activation == "none" else ", activation=%r" % self.activation)

    def forward(self, x, residual=None, add_bias=True):
        bias = self.bias if add_bias else None
        keep = self.activation != "none" and torch.is_grad_enabled() and (
            x.requires_grad or self.weight.requires_grad or (bias is not None and bias.requires_grad)
            or (residual is not None and residual.requires_grad))
        if keep:
            return torch.ops.fwdmi.linear_preact(x, self.weight, bias, residual, self.activation)[0]
        return torch.ops.fwdmi.linear(x, self.weight, bias, residual, self.activation)


class LayerNorm(torch.nn.Module):
    """``nn.LayerNorm`` over the last axis of ``x (+ skip) (+ bias)``, for training and serving.  ``forward(x, skip, bias)``
    returns the normalised rows, with ``keep_sum`` ``(rows, sum)``: the residual stream of a pre-norm layer.  The parameters
    have ``nn.LayerNorm``'s names."""

    def __init__(self, size, eps=1e-5, keep_sum=False, device=None, dtype=None):
        super().__init__()
        self.weight = torch.nn.Parameter(torch.ones(size, device=device, dtype=dtype))
        self.bias = torch.nn.Parameter(torch.zeros(size, device=device, dtype=dtype))
        self.eps, self.keep_sum = float(eps), keep_sum

    @classmethod
    def from_torch(cls, m, keep_sum=False):
        """Shares the parameters of an ``nn.LayerNorm`` over one axis with weight and bias.  One whose parameters are
        recomputed or that has hooks is refused."""
        if len(m.normalized_shape) != 1 or m.weight is None or m.bias is None:
            raise NotImplementedError("layer norm over one axis, with weight and bias")
        out = _stand_in(cls, m, "a layer norm")
        out.eps, out.keep_sum = float(m.eps), keep_sum
        return out

    gamma = property(lambda self: self.weight)
    beta = property(lambda self: self.bias)
    normalized_shape = property(lambda self: tuple(self.weight.shape))

    def extra_repr(self):
        return "%s, eps=%s%s" % (self.normalized_shape, self.eps, ", keep_sum=True" if self.keep_sum else "")

    def forward(self, x, skip=None, bias=None):
        op = torch.ops.fwdmi.layer_norm_train_sum if self.keep_sum else torch.ops.fwdmi.layer_norm_train
        got = op(x, skip, self.weight, self.bias, bias, self.eps)
        return got[:2] if self.keep_sum else got[0]


class FeedForward(torch.nn.Module):
    """The feed-forward half of a BERT layer, post-norm: ``LN(x + W2 act(W1 x + b1) + b2)``: two products and one norm, the
    second product's bias and the residual joined in the norm."""

    def __init__(self, hidden, inner, activation="gelu", eps=1e-12, device=None, dtype=None):
        super().__init__()
        self.up = Linear(hidden, inner, activation=activation, device=device, dtype=dtype)
        self.down = Linear(inner, hidden, device=device, dtype=dtype)
        self.norm = LayerNorm(hidden, eps=eps, device=device, dtype=dtype)

    def forward(self, x):
        f = self.down(self.up(x), add_bias=False)      # (a call of the module: its hooks run)
        return self.norm(f, skip=x, bias=self.down.bias)


class BertEmbeddings(torch.nn.Module):
    """Inference replacement of a BERT embedding block (word + position + token-type lookup, then
    LayerNorm) on ``[B, S]`` tensors: ``forward(input_ids, token_type_ids, attention_mask)`` returns
    ``(embeddings [B, S, H], valid_length int32 [B])``, the two outputs of the embedding plugin the
    reference wires in (trt_bert_creator.h:113-155), without its transposes to and from ``[S, B]``."""

    def __init__(self, word, pos, tok, gamma, beta, eps=1e-12):
        super().__init__()
        p = lambda t: torch.nn.Parameter(t.detach().contiguous(), requires_grad=False)
        self.word, self.pos, self.tok = p(word), p(pos), p(tok)
        self.gamma, self.beta, self.eps = p(gamma.float()), p(beta.float()), float(eps)

    def forward(self, input_ids, token_type_ids=None, attention_mask=None):
        if token_type_ids is None:
            token_type_ids = torch.zeros_like(input_ids)
        out, midx = torch.ops.fwdmi.emb_layer_norm(input_ids, token_type_ids, attention_mask, self.word, self.pos,
                                                   self.tok, self.gamma, self.beta, self.eps, True)
        return out, midx


class EmbeddingBag(torch.nn.Module):
    """Inference replacement of ``torch.nn.EmbeddingBag`` (1-D ids + offsets, or 2-D ids)."""

    def __init__(self, weight, mode="sum", include_last_offset=False):
        super().__init__()
        self.weight = torch.nn.Parameter(weight.detach().contiguous(), requires_grad=False)
        self.mode, self.include_last_offset = mode, include_last_offset

    @classmethod
    def from_torch(cls, m):
        if m.padding_idx is not None or m.max_norm is not None:
            raise NotImplementedError("padding_idx / max_norm are not part of the plugin path")
        return cls(m.weight, m.mode, m.include_last_offset)

    def forward(self, input, offsets=None, per_sample_weights=None):
        if input.dim() == 2:
            if per_sample_weights is not None:
                raise NotImplementedError("per_sample_weights with 2-D ids")
            return torch.ops.fwdmi.embedding_bag_fixed(self.weight, input, _MODE[self.mode])
        psw = None if per_sample_weights is None else per_sample_weights.to(self.weight.dtype).contiguous()
        return torch.ops.fwdmi.embedding_bag(self.weight, input, offsets, _MODE[self.mode], psw,
                                             self.include_last_offset)


class EmbeddingBagCollection(torch.nn.Module):
    """The ``nn.EmbeddingBag`` list of a DLRM-style model (equal dim, mode and dtype) as one module:
    ``forward(indices_list, offsets_list)`` returns what ``torch.cat([bag_t(ids_t, offsets_t)], dim=1)``
    returns, from one launch."""

    def __init__(self, weights, mode="sum", include_last_offset=False):
        super().__init__()
        self.weights = torch.nn.ParameterList(
            [torch.nn.Parameter(w.detach().contiguous(), requires_grad=False) for w in weights])
        self.mode, self.include_last_offset = mode, include_last_offset

    @classmethod
    def from_torch(cls, bags):
        bags = list(bags)
        first = bags[0]
        for m in bags:
            if m.padding_idx is not None or m.max_norm is not None:
                raise NotImplementedError("padding_idx / max_norm are not part of the plugin path")
            if (m.mode, m.include_last_offset, m.embedding_dim, m.weight.dtype) != \
                    (first.mode, first.include_last_offset, first.embedding_dim, first.weight.dtype):
                raise ValueError("the bags of a collection share mode, include_last_offset, dim and dtype")
        return cls([m.weight for m in bags], first.mode, first.include_last_offset)

    def forward(self, indices, offsets, per_sample_weights=None):
        psw = [None] * len(self.weights) if per_sample_weights is None else list(per_sample_weights)
        return torch.ops.fwdmi.embedding_bag_group(list(self.weights), list(indices), list(offsets),
                                                   _MODE[self.mode], self.include_last_offset, psw)


class Embedding(torch.nn.Module):
    """Inference replacement of ``torch.nn.Embedding`` (plain gather)."""

    def __init__(self, weight):
        super().__init__()
        self.weight = torch.nn.Parameter(weight.detach().contiguous(), requires_grad=False)

    def forward(self, input):
        return torch.ops.fwdmi.embedding(self.weight, input)


def replace_embedding_modules(model):
    """Swaps every ``nn.EmbeddingBag`` / ``nn.Embedding`` (without padding_idx / max_norm) in place."""
    for name, child in list(model.named_children()):
        if isinstance(child, torch.nn.EmbeddingBag) and child.padding_idx is None and child.max_norm is None:
            setattr(model, name, EmbeddingBag.from_torch(child))
        elif isinstance(child, torch.nn.Embedding) and child.padding_idx is None and child.max_norm is None:
            setattr(model, name, Embedding(child.weight))
        else:
            replace_embedding_modules(child)
    return model


def replace_dense_modules(model):
    """Swaps the ``nn.Linear`` and the ``nn.LayerNorm`` over one axis (with weight and bias) below ``model`` in place; the
    parameters are shared and keep their names, so an optimizer that holds them and checkpoints of the model keep working.

    Layers that are more than their parameters stay as they are: a weight that is recomputed from others (weight_norm,
    spectral_norm, pruning, parametrizations), hooks, a ``forward`` of the instance's own.  So does ``model`` itself
    (``Linear.from_torch`` takes a layer that stands alone)."""
    _swap_dense(model, {})
    return model


def _swap_dense(model, seen):
    for name, child in list(model._modules.items()):
        if child is None:
            continue
        if id(child) not in seen:              # (a layer that stands in two places stays one layer)
            new = child
            if type(child) is torch.nn.Linear:
                if _is_plain(child):
                    new = Linear.from_torch(child)
            elif type(child) is torch.nn.LayerNorm:
                if _is_plain(child) and len(child.normalized_shape) == 1 and child.bias is not None:
                    new = LayerNorm.from_torch(child)
            seen[id(child)] = (child, new)     # (the layer too, so that no other one gets its id)
            if new is child:
                _swap_dense(child, seen)
        new = seen[id(child)][1]
        if new is not child:
            setattr(model, name, new)
