"""The vocabulary's ends of a training step on gfx950 kernels.

    embed_tokens         rows of the embedding times a factor; its gradient groups the positions by token
    top_logits           a teacher's k largest logits of every position and their tokens
    distillation_loss    a student's loss on them (and on labels), one pass over the logits a direction

Kernels: ``dh_embed_fwd`` / ``dh_embed_bwd``, ``dh_top_logits``, ``dh_distill_fwd`` / ``dh_distill_bwd``. The model runs them
under ``model.enable_fused_vocab()``; ``distillation.py`` has the formulas as torch operations. fp32 and bf16; sums are fp32
or wider, in an order that does not change from call to call.

Each is one registered operation (``dispatcher::embed_tokens``, ...) for compilers, which torch.func's transforms refuse. In
plain eager execution the launches and the autograd nodes are C++ (``csrc/host/vocab_nodes.cpp``): a backward pass runs on
autograd's thread for the device, and a node in Python costs it several times the small kernels' own time.

Importing this module loads the kernel library and that extension, and raises ImportError if one is missing.
"""

from typing import List, Optional

import torch
import torch.nn as nn

from . import _hip, _nodes
from . import distillation as plain
from .fused_gates import _function_mode, _has_any_global_hook, plain_eager

_PLAIN = (torch.Tensor, nn.Parameter)
_INTS = (torch.int32, torch.int64)
_REDUCTION = {"none": 0, "mean": 1, "sum": 2}


def _again(logits, teacher_logits, teacher_tokens, labels, temperature, weight, ignore_index, reduction, g):
    """The loss's gradient in the logits from the formula as torch operations, differentiable itself (create_graph)."""
    z = logits.view_as(logits)
    loss = plain.distillation_loss(z, teacher_logits, teacher_tokens, labels, temperature, weight, ignore_index,
                                   plain.REDUCTIONS[reduction])
    return torch.autograd.grad(loss, z, g, create_graph=True)[0]


_native = _nodes.load(_again)
_lookup, _lookup_grad = _native.lookup, _native.lookup_grad


# ---------------------------------------------------------------------------------------------
# embedding
# ---------------------------------------------------------------------------------------------
@torch.library.custom_op("dispatcher::embed_tokens", mutates_args=(), device_types="cuda")
def _embed_op(weight: torch.Tensor, tokens: torch.Tensor, scale: float, zero_token: int, skip_token: int) -> torch.Tensor:
    return _lookup(weight, tokens, scale, zero_token)


@_embed_op.register_fake
def _(weight, tokens, scale, zero_token, skip_token):
    return weight.new_empty(*tokens.shape, weight.shape[1])


@torch.library.custom_op("dispatcher::embed_tokens_grad", mutates_args=(), device_types="cuda")
def _embed_grad_op(dy: torch.Tensor, tokens: torch.Tensor, rows: int, scale: float, skip_token: int) -> torch.Tensor:
    return _lookup_grad(dy, tokens, rows, scale, skip_token)


@_embed_grad_op.register_fake
def _(dy, tokens, rows, scale, skip_token):
    return dy.new_empty(rows, dy.shape[-1])


def _embed_setup(ctx, inputs, output):
    weight, tokens, scale, _, skip_token = inputs
    ctx.save_for_backward(tokens)
    ctx.args = (weight.shape[0], scale, skip_token)


def _embed_backward(ctx, dy):
    tokens, = ctx.saved_tensors
    return torch.ops.dispatcher.embed_tokens_grad(dy, tokens, *ctx.args), None, None, None, None


def _embed_grad_setup(ctx, inputs, output):
    _, tokens, _, scale, skip_token = inputs
    ctx.save_for_backward(tokens)
    ctx.args = (scale, skip_token)


def _zero_token(g, skip_token):
    """zero_token of the lookup that undoes a gradient by tokens: the left-out token, or one past the vocabulary (none)."""
    return skip_token if skip_token >= 0 else g.shape[0]


def _embed_grad_backward(ctx, g):
    # the gradient is linear in dy: its own gradient looks the rows of g up, zeros where positions were left out
    tokens, = ctx.saved_tensors
    scale, skip_token = ctx.args
    return torch.ops.dispatcher.embed_tokens(g, tokens, scale, _zero_token(g, skip_token), skip_token), None, None, None, None


torch.library.register_autograd("dispatcher::embed_tokens", _embed_backward, setup_context=_embed_setup)
torch.library.register_autograd("dispatcher::embed_tokens_grad", _embed_grad_backward, setup_context=_embed_grad_setup)


def embed_tokens(tokens, weight, scale=1.0, padding_idx=None):
    """weight[tokens] * scale, (*tokens.shape, d), differentiable in weight; rounded once.

    tokens: int32 or int64 of any shape; weight (V, d) fp32 or bf16 of any width. A token outside [0, V) gives a row of NaN
    (it is neither read nor reported) and no gradient. padding_idx: this token's row gets no gradient, as nn.Embedding's. The
    gradient is dense: (V, d) in weight's dtype, every token's positions summed in fp32, by stretches joined in an order
    that the tokens and sizes fix, and rounded once: the same bits on every call."""
    if tokens.dtype not in _INTS:
        raise TypeError(f"embed_tokens: tokens must be int32 or int64, got {tokens.dtype}")
    if weight.dim() != 2 or weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError(f"embed_tokens: weight (V, d) expected, got {tuple(weight.shape)}")
    skip = -1
    if padding_idx is not None:
        V = weight.shape[0]
        if not -V <= padding_idx < V:
            raise ValueError(f"embed_tokens: padding_idx {padding_idx} outside a vocabulary of {V}")
        skip = padding_idx % V
    if type(weight) in _PLAIN and weight.is_cuda and plain_eager():
        return _native.embed_tokens(weight, tokens, scale, -1, skip)
    _hip.require_gpu(weight, "embed_tokens")
    return torch.ops.dispatcher.embed_tokens(weight, tokens, float(scale), -1, skip)


def embedding_fits(module):
    """Whether embed_tokens is all that calling this module does: an nn.Embedding itself with a plain weight of the kernels'
    dtypes on the GPU, no renormalisation, sparse or frequency-scaled gradient, hook or replaced forward."""
    return (type(module) is nn.Embedding and type(module.weight) in _PLAIN and module.weight.is_cuda
            and module.weight.dtype in (torch.float32, torch.bfloat16) and module.max_norm is None and not module.sparse
            and not module.scale_grad_by_freq and "forward" not in module.__dict__
            and not (module._forward_hooks or module._forward_pre_hooks or module._backward_hooks
                     or module._backward_pre_hooks) and not _has_any_global_hook() and not _function_mode())


# ---------------------------------------------------------------------------------------------
# a teacher's targets
# ---------------------------------------------------------------------------------------------
@torch.library.custom_op("dispatcher::top_logits", mutates_args=(), device_types="cuda")
def _top_op(logits: torch.Tensor, k: int) -> List[torch.Tensor]:
    return list(_native.top_logits(logits, k))


@_top_op.register_fake
def _(logits, k):
    shape = (*logits.shape[:-1], k)
    return [logits.new_empty(shape), logits.new_empty(shape, dtype=torch.int64)]


def top_logits(logits, k):
    """(values, tokens), each (..., k): the k largest of logits (..., V) and where they stand, falling; equal values (0.0 and
    -0.0 are) by the lower token, NaN above every number. k up to 256. values keep the dtype; constants: no gradient flows to
    `logits`."""
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"top_logits: logits (..., vocabulary) expected, got {tuple(logits.shape)}")
    if not 1 <= k <= min(plain.MAX_TARGETS, logits.shape[-1]):
        raise ValueError(f"top_logits: k={k} must be in [1, min({plain.MAX_TARGETS}, vocabulary {logits.shape[-1]})]")
    if type(logits) in _PLAIN and logits.is_cuda and plain_eager():
        return _native.top_logits(logits, k)
    _hip.require_gpu(logits, "top_logits")
    values, tokens = torch.ops.dispatcher.top_logits(logits.detach(), k)
    return values, tokens


# ---------------------------------------------------------------------------------------------
# distillation loss
# ---------------------------------------------------------------------------------------------
def _kept_numel(n):
    """fp32 numbers of what a backward pass keeps of n rows: four a row and, behind them, the divisor (and to 16 bytes)."""
    return 4 * n + 4


@torch.library.custom_op("dispatcher::distillation_loss", mutates_args=(), device_types="cuda")
def _distill_op(logits: torch.Tensor, teacher_logits: torch.Tensor, teacher_tokens: torch.Tensor,
                labels: Optional[torch.Tensor], temperature: float, weight: float, ignore_index: int,
                reduction: int) -> List[torch.Tensor]:
    out, kept = _native.distill(logits, teacher_logits, teacher_tokens, labels, temperature, weight, ignore_index, reduction)
    return [out, kept[:_kept_numel(logits.shape[:-1].numel())].clone()]        # (a size that its fake form can say)


@_distill_op.register_fake
def _(logits, teacher_logits, teacher_tokens, labels, temperature, weight, ignore_index, reduction):
    f32 = torch.float32
    lead = logits.shape[:-1]
    n = 1
    for s in lead:
        n = n * s
    return [logits.new_empty(() if reduction else lead, dtype=f32), logits.new_empty((_kept_numel(n),), dtype=f32)]


@torch.library.custom_op("dispatcher::distillation_loss_grad", mutates_args=(), device_types="cuda")
def _distill_grad_op(g: torch.Tensor, logits: torch.Tensor, teacher_logits: torch.Tensor, teacher_tokens: torch.Tensor,
                     labels: Optional[torch.Tensor], kept: torch.Tensor, temperature: float, weight: float, ignore_index: int,
                     reduction: int) -> torch.Tensor:
    return _native.distill_grad(g, logits, teacher_logits, teacher_tokens, labels, kept, temperature, weight, ignore_index, reduction)


@_distill_grad_op.register_fake
def _(g, logits, teacher_logits, teacher_tokens, labels, kept, temperature, weight, ignore_index, reduction):
    return logits.new_empty(logits.shape)


def _distill_setup(ctx, inputs, output):
    logits, *constants = inputs[:4]
    ctx.set_materialize_grads(False)
    # (what was made under inference mode, as a teacher's targets may be, cannot be saved: a copy can)
    ctx.save_for_backward(logits, *(t.clone() if t is not None and t.is_inference() else t for t in constants), output[1])
    ctx.args = tuple(inputs[4:])


def _distill_backward(ctx, grads):
    if grads[0] is None:
        return (None,) * 8
    if torch.is_grad_enabled():
        return (_again(*ctx.saved_tensors[:4], *ctx.args, grads[0]), *(None,) * 7)
    return (torch.ops.dispatcher.distillation_loss_grad(grads[0], *ctx.saved_tensors, *ctx.args), *(None,) * 7)


torch.library.register_autograd("dispatcher::distillation_loss", _distill_backward, setup_context=_distill_setup)


def distillation_loss(logits, teacher_logits, teacher_tokens, labels=None, temperature=1.0, weight=1.0, ignore_index=-100,
                      reduction="mean"):
    """Distillation from a teacher's top logits, differentiable in `logits`; a scalar, or (reduction="none") the positions'
    losses, fp32.

    logits (..., V) fp32 or bf16; teacher_logits, teacher_tokens (..., k) as top_logits gives them (fp32 or bf16, int32 or
    int64; k up to 256), a slot with a token below 0 or a logit of -inf being empty; labels (...) int32 or int64, or None.
    Per position, with p the softmax of the teacher's live logits over the temperature and q that of `logits`,

        weight * temperature^2 * sum_j p_j (log p_j - log q_j)  +  (1 - weight) * cross-entropy of the label

    without the first term where every slot is empty. weight < 1 needs labels. A position whose label is ignore_index counts
    for nothing: no loss, a gradient of zeros, whatever its logits hold. reduction: "mean" over the other positions (NaN when
    there is none, as the cross-entropy's mean), "sum" or "none". A teacher token past the vocabulary or a live teacher logit
    of NaN or +inf (with weight > 0; the teacher is not read otherwise), or a label outside the vocabulary, makes its position's
    loss and all of its gradient NaN. The teacher's logits are constants."""
    plain.check_targets(logits, teacher_logits, teacher_tokens, labels, temperature, weight, reduction)
    args = (logits, teacher_logits, teacher_tokens, labels, float(temperature), float(weight), int(ignore_index),
            _REDUCTION[reduction])
    if type(logits) in _PLAIN and logits.is_cuda and plain_eager():
        return _native.distillation_loss(*args)
    _hip.require_gpu(logits, "distillation_loss")
    return torch.ops.dispatcher.distillation_loss(*args)[0]
