"""Distillation from a teacher's top logits as torch operations: the formulas of the kernels in ``fused_vocab``, on any device.

A teacher's targets for a position are its k largest logits and their tokens (top_logits). With z the student's logits, t_j
the teacher's at tokens k_j, temperature tau and weight w:

    p = softmax(t / tau) over the live slots (k_j >= 0 and t_j > -inf),  q = softmax(z / tau),  P = softmax(z)
    row = w tau^2 sum_j p_j (log p_j - log q_{k_j}) + (1 - w) (-log P_label)

The reference trains on token labels alone (reference dispatcher_hybrid/modeling_dispatcher.py:352-356); it has no counterpart
of this.
"""

import math

import torch

MAX_TARGETS = 256              # targets a position: the kernels' limit, kept by both forms

REDUCTIONS = ("none", "mean", "sum")


def check_targets(logits, teacher_logits, teacher_tokens, labels, temperature, weight, reduction):
    """Raise unless these are a distillation_loss call."""
    shape, targets = logits.shape, teacher_logits.shape
    if not shape or not logits.is_floating_point():
        raise ValueError(f"distillation_loss: logits (..., vocabulary) expected, got {tuple(shape)} {logits.dtype}")
    lead = shape[:-1]
    if targets != teacher_tokens.shape or targets[:-1] != lead or len(targets) != len(shape):
        raise ValueError(f"distillation_loss: teacher logits {tuple(targets)} and tokens {tuple(teacher_tokens.shape)} must both "
                         f"be {(*lead, 'k')}, for logits {tuple(shape)}")
    if not 1 <= targets[-1] <= MAX_TARGETS:
        raise ValueError(f"distillation_loss: {targets[-1]} targets a position, 1 to {MAX_TARGETS} possible")
    if shape[-1] < 1:
        raise ValueError("distillation_loss: empty vocabulary")
    if teacher_logits.requires_grad:
        raise ValueError("distillation_loss: the teacher's logits are constants; detach them")
    if not teacher_logits.is_floating_point():
        raise TypeError(f"distillation_loss: teacher logits of {teacher_logits.dtype}")
    if teacher_tokens.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"distillation_loss: teacher tokens must be int32 or int64, got {teacher_tokens.dtype}")
    if labels is not None:
        if labels.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"distillation_loss: labels must be int32 or int64, got {labels.dtype}")
        if labels.shape != lead:
            raise ValueError(f"distillation_loss: labels {tuple(labels.shape)} for logits {tuple(shape)}")
    if not (0.0 < temperature < math.inf):
        raise ValueError(f"distillation_loss: temperature {temperature} must be positive and finite")
    if not 0.0 <= weight <= 1.0:
        raise ValueError(f"distillation_loss: weight {weight} must be in [0, 1]")
    if labels is None and weight != 1.0:
        raise ValueError(f"distillation_loss: weight {weight} leaves a part to labels, and there are none")
    if reduction not in REDUCTIONS:
        raise ValueError(f"distillation_loss: reduction {reduction!r}; use one of {', '.join(REDUCTIONS)}")


def distillation_loss(logits, teacher_logits, teacher_tokens, labels=None, temperature=1.0, weight=1.0, ignore_index=-100,
                      reduction="mean"):
    """fused_vocab.distillation_loss as torch operations (fp32, or fp64 for fp64 logits), differentiable in `logits`."""
    check_targets(logits, teacher_logits, teacher_tokens, labels, temperature, weight, reduction)
    wide = torch.float64 if logits.dtype == torch.float64 else torch.float32
    V = logits.shape[-1]
    z = logits.to(wide)
    kept = torch.ones(z.shape[:-1], dtype=torch.bool, device=z.device) if labels is None else labels != ignore_index
    z = torch.where(kept.unsqueeze(-1), z, torch.zeros((), dtype=wide, device=z.device))
    zero = torch.zeros((), dtype=wide, device=z.device)
    rows = torch.zeros(z.shape[:-1], dtype=wide, device=z.device)
    bad = torch.zeros_like(kept) if labels is None else (labels < 0) | (labels >= V)
    if weight > 0.0:
        t = teacher_logits.to(wide)
        bad = bad | (teacher_tokens >= V).any(-1)
        live = (teacher_tokens >= 0) & (teacher_tokens < V) & (t != -math.inf)
        # (an all-dead row goes through the softmax as zeros, and is masked behind it)
        t = torch.where(live, t / temperature, torch.where(live.any(-1, keepdim=True), -math.inf, 0.0).to(wide))
        p, log_p = torch.softmax(t, -1), torch.log_softmax(t, -1)
        use = live & (p != 0)
        log_q = torch.log_softmax(z / temperature, -1).gather(-1, teacher_tokens.long().clamp(0, V - 1))
        terms = torch.where(use, p, zero) * (torch.where(use, log_p, zero) - torch.where(use, log_q, zero))
        # (a bad row without a live slot: a term for the factor of NaN below to reach the gradient through)
        rows = rows + weight * temperature ** 2 * terms.sum(-1) + torch.where(bad, log_q[..., 0], zero)
    if labels is not None and weight < 1.0:
        picked = torch.log_softmax(z, -1).gather(-1, labels.long().clamp(0, V - 1).unsqueeze(-1)).squeeze(-1)
        rows = rows - (1.0 - weight) * picked
    # (a factor of NaN: the row's gradient is NaN too)
    rows = rows * torch.where(bad, math.nan, 1.0).to(wide)
    rows = torch.where(kept, rows, zero)
    if reduction == "none":
        return rows
    return rows.sum() / kept.sum() if reduction == "mean" else rows.sum()


def top_logits(logits, k):
    """fused_vocab.top_logits as a stable sort."""
    if not 1 <= k <= min(MAX_TARGETS, logits.shape[-1]):
        raise ValueError(f"top_logits: k={k} must be in [1, min({MAX_TARGETS}, vocabulary {logits.shape[-1]})]")
    logits = logits.detach()
    # (NaN of one sign: the GPU's sort puts one whose sign bit is set below every number)
    order = torch.where(logits.isnan(), math.nan, logits)
    tokens = torch.sort(order, dim=-1, descending=True, stable=True).indices[..., :k].contiguous()
    return logits.gather(-1, tokens), tokens
