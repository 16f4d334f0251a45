"""Post-training at the vocabulary's end on gfx950 kernels.

    token_logprobs     log-probabilities of given tokens, and entropies, of logits; one pass over them a direction
    head_logprobs      the same from hidden states and the head's weight: the logits are not stored (no gradient)
    preference_loss    a loss on pairs of sequences, one preferred
    policy_loss        the clipped policy loss with a KL term and an entropy bonus

Kernels: ``dh_logprob_fwd`` / ``dh_logprob_bwd``, ``dh_preference_fwd``, ``dh_policy_fwd``, ``dh_head_logprob``. The model runs
them under ``model.enable_fused_vocab()``; ``logprobs.py`` has the formulas as torch operations. fp32 and bf16; sums over the
vocabulary are fp32, what is made of them fp64, in an order that does not change from call to call.

Each is one registered operation (``dispatcher::token_logprobs``, ...) for compilers, which torch.func's transforms refuse. In
plain eager execution the launches and the autograd nodes are C++ (``csrc/host/logprob_nodes.cpp``).

Importing this module loads the kernel library and the extension, and raises ImportError if one is missing.
"""

from typing import List, Optional

import torch
import torch.nn as nn

from . import _hip
from . import logprobs as plain
from .fused_gates import plain_eager
from .fused_vocab import _native

_PLAIN = (torch.Tensor, nn.Parameter)
_f32 = torch.float32


# ---- the gradients as torch operations, differentiable themselves (create_graph) ----------------------------------------
def _again_logprobs(logits, tokens, temperature, ignore_index, g_lp, g_ent):
    z = logits.view_as(logits)
    out = plain.token_logprobs(z, tokens, temperature, ignore_index, g_ent is not None)
    pairs = [(o, g) for o, g in zip(out if g_ent is not None else (out,), (g_lp, g_ent)) if g is not None]
    return torch.autograd.grad([o for o, _ in pairs], z, [g.to(o.dtype) for o, g in pairs], create_graph=True)[0]


def _again_preference(logits, tokens, reference, kind, average, beta, margin, smoothing, ignore_index, reduction, g):
    z = logits.view_as(logits)
    loss, _ = plain.preference_loss(z, tokens, reference, beta, plain.KINDS[kind], average, margin, smoothing, ignore_index,
                                    plain.PAIR_REDUCTIONS[reduction])
    return torch.autograd.grad(loss, z, g, create_graph=True)[0]


def _again_policy(logits, tokens, old, advantages, reference, clip, clip_high, kl, entropy, temperature, ignore_index, reduction,
                  g):
    z = logits.view_as(logits)
    loss, _ = plain.policy_loss(z, tokens, old, advantages, reference, clip, clip_high, kl, entropy, temperature, ignore_index,
                                plain.TOKEN_REDUCTIONS[reduction])
    return torch.autograd.grad(loss, z, g, create_graph=True)[0]


_native.bind_logprobs(_again_logprobs, _again_preference, _again_policy)


def _savable(t):
    """(what was made under inference mode cannot be saved: a copy can)"""
    return t.clone() if t is not None and t.is_inference() else t


def _count(shape):
    n = 1
    for s in shape:
        n = n * s
    return n


# ---- log-probabilities ----------------------------------------------------------------------------------------------
@torch.library.custom_op("dispatcher::token_logprobs", mutates_args=(), device_types="cuda")
def _logprobs_op(logits: torch.Tensor, tokens: torch.Tensor, temperature: float, ignore_index: int,
                 entropy: bool) -> List[torch.Tensor]:
    out, kept = _native.logprobs(logits, tokens, temperature, ignore_index, entropy)
    return [*out, kept]


@_logprobs_op.register_fake
def _(logits, tokens, temperature, ignore_index, entropy):
    lead = logits.shape[:-1]
    out = [logits.new_empty(lead, dtype=_f32) for _ in range(2 if entropy else 1)]
    return [*out, logits.new_empty((4 * _count(lead),), dtype=_f32)]


@torch.library.custom_op("dispatcher::token_logprobs_grad", mutates_args=(), device_types="cuda")
def _logprobs_grad_op(g_logprobs: Optional[torch.Tensor], g_entropy: Optional[torch.Tensor], logits: torch.Tensor,
                      tokens: torch.Tensor, kept: torch.Tensor, temperature: float, ignore_index: int) -> torch.Tensor:
    return _native.logprobs_grad(g_logprobs, g_entropy, logits, tokens, kept, temperature, ignore_index)


@_logprobs_grad_op.register_fake
def _(g_logprobs, g_entropy, logits, tokens, kept, temperature, ignore_index):
    return logits.new_empty(logits.shape)


def _logprobs_setup(ctx, inputs, output):
    logits, tokens, *ctx.args, _ = inputs
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(logits, _savable(tokens), output[-1])


def _logprobs_backward(ctx, grads):
    g_lp, g_ent = grads[0], grads[1] if len(grads) > 2 else None
    if g_lp is None and g_ent is None:
        return (None,) * 5
    logits, tokens, kept = ctx.saved_tensors
    if torch.is_grad_enabled():
        dz = _again_logprobs(logits, tokens, *ctx.args, g_lp, g_ent)
    else:
        dz = torch.ops.dispatcher.token_logprobs_grad(g_lp, g_ent, logits, tokens, kept, *ctx.args)
    return (dz, *(None,) * 4)


torch.library.register_autograd("dispatcher::token_logprobs", _logprobs_backward, setup_context=_logprobs_setup)


def token_logprobs(logits, tokens, temperature=1.0, ignore_index=-100, entropy=False):
    """Log-probabilities of the tokens under softmax(logits / temperature), fp32, and with `entropy` the entropies of those
    distributions too, (logprobs, entropies); both differentiable in `logits`.

    logits (..., V) fp32 or bf16, entries of -inf allowed; tokens (...) int32 or int64. A position whose token is ignore_index
    counts for nothing: zeros, a gradient of zeros, whatever its logits hold. Another token outside the vocabulary makes its
    position's values and all of its gradient NaN. Fewer than 2^22 positions, up to 2^24 logits each (as for the losses)."""
    plain.check_tokens("token_logprobs", logits, tokens, temperature)
    args = (logits, tokens, float(temperature), int(ignore_index), bool(entropy))
    if type(logits) in _PLAIN and logits.is_cuda and plain_eager():
        out = _native.token_logprobs(*args)
    else:
        _hip.require_gpu(logits, "token_logprobs")
        out = torch.ops.dispatcher.token_logprobs(*args)
    return (out[0], out[1]) if entropy else out[0]


@torch.library.custom_op("dispatcher::head_logprobs", mutates_args=(), device_types="cuda")
def _head_op(hidden: torch.Tensor, weight: torch.Tensor, tokens: torch.Tensor, temperature: float, ignore_index: int, entropy: bool,
             round_logits: bool) -> List[torch.Tensor]:
    return _native.head_logprobs(hidden, weight, tokens, temperature, ignore_index, entropy, round_logits)


@_head_op.register_fake
def _(hidden, weight, tokens, temperature, ignore_index, entropy, round_logits):
    return [hidden.new_empty(hidden.shape[:-1], dtype=_f32) for _ in range(2 if entropy else 1)]


def head_logprobs(hidden, weight, tokens, temperature=1.0, ignore_index=-100, entropy=False, round_logits=False):
    """token_logprobs of the logits hidden . weight^T without those logits in memory; no gradient (raises where one is wanted of
    `hidden` or `weight`).

    hidden (..., d) and weight (V, d) of one type, fp32 or bf16; tokens (...) int32 or int64. The logits are fp32 sums; with
    round_logits they are rounded to the operands' type first, as a head that stores them does. Positions whose token is
    ignore_index cost nothing where there are many (zeros); another token outside the vocabulary gives NaN."""
    plain.check_head(hidden, weight, tokens, temperature)
    args = (hidden, weight, tokens, float(temperature), int(ignore_index), bool(entropy), bool(round_logits))
    if type(hidden) in _PLAIN and type(weight) in _PLAIN and hidden.is_cuda and plain_eager():
        out = _native.head_logprobs(*args)
    else:
        _hip.require_gpu(hidden, "head_logprobs")
        out = torch.ops.dispatcher.head_logprobs(hidden.detach(), weight.detach(), *args[2:])
    return (out[0], out[1]) if entropy else out[0]


# ---- preference loss --------------------------------------------------------------------------------------------------
@torch.library.custom_op("dispatcher::preference_loss", mutates_args=(), device_types="cuda")
def _preference_op(logits: torch.Tensor, tokens: torch.Tensor, reference: Optional[torch.Tensor], kind: int, average: bool,
                   beta: float, margin: float, label_smoothing: float, ignore_index: int, reduction: int) -> List[torch.Tensor]:
    loss, sums, kept = _native.preference(logits, tokens, reference, kind, average, beta, margin, label_smoothing, ignore_index,
                                          reduction)
    n, T = logits.shape[0], logits.shape[1]
    return [loss, sums, kept[:4 * n * T + 2 * (n // 2) + 1].clone()]           # (a size that its fake form can say)


@_preference_op.register_fake
def _(logits, tokens, reference, kind, average, beta, margin, label_smoothing, ignore_index, reduction):
    n, T = logits.shape[0], logits.shape[1]
    return [logits.new_empty(() if reduction else (n // 2,), dtype=_f32), logits.new_empty((n,), dtype=_f32),
            logits.new_empty((4 * n * T + 2 * (n // 2) + 1,), dtype=_f32)]


@torch.library.custom_op("dispatcher::preference_loss_grad", mutates_args=(), device_types="cuda")
def _preference_grad_op(g: torch.Tensor, logits: torch.Tensor, tokens: torch.Tensor, kept: torch.Tensor, ignore_index: int,
                        reduction: int) -> torch.Tensor:
    return _native.preference_grad(g, logits, tokens, kept, ignore_index, reduction)


@_preference_grad_op.register_fake
def _(g, logits, tokens, kept, ignore_index, reduction):
    return logits.new_empty(logits.shape)


def _preference_setup(ctx, inputs, output):
    logits, tokens, reference, *ctx.args = inputs
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(logits, _savable(tokens), _savable(reference), output[2])


def _preference_backward(ctx, grads):
    if grads[0] is None:
        return (None,) * 10
    logits, tokens, reference, kept = ctx.saved_tensors
    if torch.is_grad_enabled():
        dz = _again_preference(logits, tokens, reference, *ctx.args, grads[0])
    else:
        dz = torch.ops.dispatcher.preference_loss_grad(grads[0], logits, tokens, kept, *ctx.args[-2:])
    return (dz, *(None,) * 9)


torch.library.register_autograd("dispatcher::preference_loss", _preference_backward, setup_context=_preference_setup)


def preference_loss(logits, tokens, reference=None, beta=0.1, loss="sigmoid", average=False, margin=0.0, label_smoothing=0.0,
                    ignore_index=-100, reduction="mean"):
    """A loss on pairs of sequences, one of each preferred: (loss, logprobs), fp32. The loss is differentiable in `logits`;
    logprobs (2 n), constants, are what it is made of.

    logits (2 n, T, V) fp32 or bf16: sequence i is preferred to sequence n + i. tokens (2 n, T) int32 or int64: the token that
    each position is scored on, ignore_index where it is no part of an answer (not read, a gradient of zeros). A sequence's
    logprob S is the sum of its tokens' log-probabilities or, with `average`, their mean (0 of none); reference (2 n) any
    floating type, or None for zeros: the same of a reference model. With D = (S - reference)_i - (S - reference)_{n+i} and
    x = beta D - margin, a pair's loss is

        "sigmoid"   -(1 - label_smoothing) log sigma(x) - label_smoothing log sigma(-x)
        "hinge"     max(0, 1 - x)
        "squared"   (D - 1 / (2 beta))^2             (no margin)

    reduction: "mean" over the pairs (NaN when there is none), "sum" or "none" (n losses). A token outside the vocabulary makes
    its sequence's logprob, its pair's loss and the gradient of the pair's answers NaN. A token of probability 0 (its logit -inf)
    makes its sequence's logprob -inf: the squared loss is inf and its pair's gradients infinite or NaN, those of the others are
    numbers."""
    plain.check_preference(logits, tokens, reference, beta, loss, margin, label_smoothing, reduction)
    args = (logits, tokens, reference, plain.KINDS.index(loss), bool(average), float(beta), float(margin), float(label_smoothing),
            int(ignore_index), plain.PAIR_REDUCTIONS.index(reduction))
    if type(logits) in _PLAIN and logits.is_cuda and plain_eager():
        return tuple(_native.preference_loss(*args))
    _hip.require_gpu(logits, "preference_loss")
    out = torch.ops.dispatcher.preference_loss(*args)
    return out[0], out[1].detach()


# ---- policy loss --------------------------------------------------------------------------------------------------------
@torch.library.custom_op("dispatcher::policy_loss", mutates_args=(), device_types="cuda")
def _policy_op(logits: torch.Tensor, tokens: torch.Tensor, old_logprobs: torch.Tensor, advantages: torch.Tensor,
               reference_logprobs: Optional[torch.Tensor], clip: float, clip_high: float, kl_weight: float,
               entropy_weight: float, temperature: float, ignore_index: int, reduction: int) -> List[torch.Tensor]:
    loss, scores, kept = _native.policy(logits, tokens, old_logprobs, advantages, reference_logprobs, clip, clip_high, kl_weight,
                                        entropy_weight, temperature, ignore_index, reduction)
    return [loss, scores, kept[:(6 if entropy_weight != 0.0 else 5) * _count(logits.shape[:-1]) + 1].clone()]


@_policy_op.register_fake
def _(logits, tokens, old_logprobs, advantages, reference_logprobs, clip, clip_high, kl_weight, entropy_weight, temperature,
      ignore_index, reduction):
    lead = logits.shape[:-1]
    return [logits.new_empty(() if reduction else lead, dtype=_f32), logits.new_empty(lead, dtype=_f32),
            logits.new_empty(((6 if entropy_weight != 0.0 else 5) * _count(lead) + 1,), dtype=_f32)]


@torch.library.custom_op("dispatcher::policy_loss_grad", mutates_args=(), device_types="cuda")
def _policy_grad_op(g: torch.Tensor, logits: torch.Tensor, tokens: torch.Tensor, kept: torch.Tensor, entropy_weight: float,
                    temperature: float, ignore_index: int, reduction: int) -> torch.Tensor:
    return _native.policy_grad(g, logits, tokens, kept, entropy_weight, temperature, ignore_index, reduction)


@_policy_grad_op.register_fake
def _(g, logits, tokens, kept, entropy_weight, temperature, ignore_index, reduction):
    return logits.new_empty(logits.shape)


def _policy_setup(ctx, inputs, output):
    ctx.args = inputs[5:]
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(inputs[0], *(_savable(t) for t in inputs[1:5]), output[2])


def _policy_backward(ctx, grads):
    if grads[0] is None:
        return (None,) * 12
    *saved, kept = ctx.saved_tensors
    if torch.is_grad_enabled():
        dz = _again_policy(*saved, *ctx.args, grads[0])
    else:
        dz = torch.ops.dispatcher.policy_loss_grad(grads[0], saved[0], saved[1], kept, *ctx.args[3:])
    return (dz, *(None,) * 11)


torch.library.register_autograd("dispatcher::policy_loss", _policy_backward, setup_context=_policy_setup)


def policy_loss(logits, tokens, old_logprobs, advantages, reference_logprobs=None, clip=0.2, clip_high=None, kl_weight=0.0,
                entropy_weight=0.0, temperature=1.0, ignore_index=-100, reduction="mean"):
    """The clipped policy loss: (loss, logprobs), fp32. The loss is differentiable in `logits`; logprobs (...), constants, are
    the tokens' log-probabilities under softmax(logits / temperature).

    logits (..., T, V) fp32 or bf16; tokens (..., T) int32 or int64: the sampled token of each position, ignore_index where there
    is none (nothing of the position is read, a gradient of zeros). old_logprobs (..., T): of the policy that sampled them;
    advantages (..., T), or (...) one a sequence; reference_logprobs (..., T): of a reference model, needed for kl_weight > 0.
    Floating types, taken as fp32; constants. With r = exp(logprob - old), A the advantage, d = reference - logprob, a position's
    loss is

        -min(r A, clip(r, 1 - clip, 1 + clip_high) A) + kl_weight (exp(d) - d - 1) - entropy_weight entropy

    clip_high: clip when None. reduction: "mean" over the positions (NaN when there is none), "sequence": the mean over the
    sequences that have a position of each one's mean, "sum" or "none". A token outside the vocabulary makes its position's loss
    and all of its gradient NaN. A token of probability 0 (its logit -inf) has a ratio of 0; with a KL term its position's loss is
    NaN and its gradient infinite or NaN. So is the gradient, and inf the loss, of a ratio times its advantage that is past fp32 and
    not clipped."""
    clip_high = clip if clip_high is None else clip_high
    plain.check_policy(logits, tokens, old_logprobs, advantages, reference_logprobs, clip, clip_high, kl_weight, entropy_weight,
                       temperature, reduction)
    args = (logits, tokens, old_logprobs, advantages, reference_logprobs if kl_weight else None, float(clip), float(clip_high),
            float(kl_weight), float(entropy_weight), float(temperature), int(ignore_index),
            plain.TOKEN_REDUCTIONS.index(reduction))
    if type(logits) in _PLAIN and logits.is_cuda and plain_eager():
        return tuple(_native.policy_loss(*args))
    _hip.require_gpu(logits, "policy_loss")
    out = torch.ops.dispatcher.policy_loss(*args)
    return out[0], out[1].detach()
