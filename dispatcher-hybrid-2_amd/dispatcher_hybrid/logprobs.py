"""Log-probabilities of given tokens and the post-training losses on them as torch operations: the formulas of the kernels in
``fused_logprobs``, on any device, each differentiable in the logits.

With z a position's logits, y its token and tau a temperature, p = softmax(z / tau):

    token_logprobs    log p_y and, wanted, the entropy  - sum_v p_v log p_v
    preference_loss   sequences i and n + i are a pair, i preferred. S = sum (or mean) of a sequence's log-probabilities, R the same
                      of a reference model, D = (S - R)_i - (S - R)_{n+i}, x = beta D - margin:
                        "sigmoid"  - (1 - s) log sigma(x) - s log sigma(-x)        s: label_smoothing
                        "hinge"    max(0, 1 - x)
                        "squared"  (D - 1 / (2 beta))^2
    policy_loss       r = exp(log p_y - old), advantage A, d = reference - log p_y:
                        - min(r A, clip(r, 1 - clip, 1 + clip_high) A) + kl_weight (exp(d) - d - 1) - entropy_weight entropy

The reference trains on token labels alone (reference dispatcher_hybrid/modeling_dispatcher.py:352-356); it has no counterpart
of these.
"""

import math

import torch

KINDS = ("sigmoid", "hinge", "squared")
PAIR_REDUCTIONS = ("none", "mean", "sum")
TOKEN_REDUCTIONS = ("none", "mean", "sum", "sequence")
_INTS = (torch.int32, torch.int64)


def check_tokens(what, logits, tokens, temperature=1.0):
    """Raise unless these are logits (..., V), the tokens (...) of them and a temperature."""
    if not logits.dim() or not logits.is_floating_point():
        raise ValueError(f"{what}: logits (..., vocabulary) expected, got {tuple(logits.shape)} {logits.dtype}")
    if logits.shape[-1] < 1:
        raise ValueError(f"{what}: empty vocabulary")
    if tokens.dtype not in _INTS:
        raise TypeError(f"{what}: tokens must be int32 or int64, got {tokens.dtype}")
    if tokens.shape != logits.shape[:-1]:
        raise ValueError(f"{what}: tokens {tuple(tokens.shape)} for logits {tuple(logits.shape)}")
    if not 2.0 ** -126 <= temperature <= 2.0 ** 126:
        raise ValueError(f"{what}: temperature {temperature} must be positive and finite (2^-126 to 2^126)")


def _constant(what, name, t, shape):
    if not t.is_floating_point():
        raise TypeError(f"{what}: {name} of {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{what}: {name} {tuple(t.shape)}, {tuple(shape)} needed")
    if t.requires_grad:
        raise ValueError(f"{what}: {name} are constants; detach them")


def check_preference(logits, tokens, reference, beta, loss, margin, label_smoothing, reduction):
    """Raise unless these are a preference_loss call."""
    what = "preference_loss"
    check_tokens(what, logits, tokens)
    if logits.dim() != 3 or logits.shape[0] % 2:
        raise ValueError(f"{what}: logits (2 n, T, vocabulary) expected, the preferred sequences before the others, got "
                         f"{tuple(logits.shape)}")
    if reference is not None:
        _constant(what, "the reference's log-probabilities", reference, logits.shape[:1])
    if loss not in KINDS:
        raise ValueError(f"{what}: loss {loss!r}; use one of {', '.join(KINDS)}")
    if not 0.0 < beta < math.inf:
        raise ValueError(f"{what}: beta {beta} must be positive and finite")
    if not math.isfinite(margin):
        raise ValueError(f"{what}: margin {margin} must be finite")
    if not 0.0 <= label_smoothing <= 0.5:
        raise ValueError(f"{what}: label_smoothing {label_smoothing} must be in [0, 1/2]")
    if loss == "squared" and margin or loss != "sigmoid" and label_smoothing:
        raise ValueError(f"{what}: the {loss} loss has no {'margin' if margin and loss == 'squared' else 'label_smoothing'}")
    if reduction not in PAIR_REDUCTIONS:
        raise ValueError(f"{what}: reduction {reduction!r}; use one of {', '.join(PAIR_REDUCTIONS)}")


def check_policy(logits, tokens, old_logprobs, advantages, reference_logprobs, clip, clip_high, kl_weight, entropy_weight,
                 temperature, reduction):
    """Raise unless these are a policy_loss call (clip_high a number)."""
    what = "policy_loss"
    check_tokens(what, logits, tokens, temperature)
    if logits.dim() < 2:
        raise ValueError(f"{what}: logits (..., T, vocabulary) expected, got {tuple(logits.shape)}")
    _constant(what, "the old log-probabilities", old_logprobs, tokens.shape)
    _constant(what, "the advantages", advantages, tokens.shape[:-1] if advantages.dim() < tokens.dim() else tokens.shape)
    if reference_logprobs is not None:
        _constant(what, "the reference's log-probabilities", reference_logprobs, tokens.shape)
    if not (0.0 <= clip <= 1.0 and 0.0 <= clip_high < math.inf):
        raise ValueError(f"{what}: clip {clip} must be in [0, 1], clip_high {clip_high} not negative and finite")
    if not (0.0 <= kl_weight < math.inf and math.isfinite(entropy_weight)):
        raise ValueError(f"{what}: kl_weight {kl_weight} must not be negative, entropy_weight {entropy_weight} finite")
    if kl_weight and reference_logprobs is None:
        raise ValueError(f"{what}: a KL term of weight {kl_weight} needs reference_logprobs")
    if reduction not in TOKEN_REDUCTIONS:
        raise ValueError(f"{what}: reduction {reduction!r}; use one of {', '.join(TOKEN_REDUCTIONS)}")


def _wide(t):
    return torch.float64 if t.dtype == torch.float64 else torch.float32


def _values(logits, tokens, temperature, ignore_index, entropy):
    """(live, log-probabilities, entropies or None), zeros where ignored and NaN where a token is outside the vocabulary."""
    wide = _wide(logits)
    zero, nan = torch.zeros((), dtype=wide, device=logits.device), torch.full((), math.nan, dtype=wide, device=logits.device)
    live = tokens != ignore_index
    bad = live & ((tokens < 0) | (tokens >= logits.shape[-1]))
    z = torch.where(live.unsqueeze(-1), logits.to(wide), zero)
    # (a factor of NaN: the row's gradient is NaN too)
    factor = torch.where(bad, nan, torch.ones_like(zero))
    if temperature < 1.0:                  # (of differences: a logit over the temperature may be past the type where they are not)
        most = z.detach().amax(-1, keepdim=True)
        z = z - torch.where(most.isfinite(), most, zero)
    log_p = torch.log_softmax(z / temperature, -1)
    lp = log_p.gather(-1, torch.where(live & ~bad, tokens, torch.zeros_like(tokens)).long().unsqueeze(-1)).squeeze(-1)
    lp = torch.where(live, lp * factor, zero)
    if not entropy:
        return live, lp, None
    closed = log_p == -math.inf
    p = torch.where(closed, zero, log_p.exp())
    ent = -(p * torch.where(closed, zero, log_p)).sum(-1)
    return live, lp, torch.where(live, ent * factor, zero)


def token_logprobs(logits, tokens, temperature=1.0, ignore_index=-100, entropy=False):
    """fused_logprobs.token_logprobs as torch operations (fp32, or fp64 for fp64 logits)."""
    check_tokens("token_logprobs", logits, tokens, temperature)
    _, lp, ent = _values(logits, tokens, temperature, ignore_index, entropy)
    return (lp, ent) if entropy else lp


def head_logprobs(hidden, weight, tokens, temperature=1.0, ignore_index=-100, entropy=False, round_logits=False):
    """fused_logprobs.head_logprobs as torch operations; the logits are stored."""
    check_head(hidden, weight, tokens, temperature)
    wide = _wide(hidden)
    if round_logits:
        logits = torch.nn.functional.linear(hidden.detach(), weight.detach())
    else:
        logits = torch.nn.functional.linear(hidden.detach().to(wide), weight.detach().to(wide))
    return token_logprobs(logits, tokens, temperature, ignore_index, entropy)


def check_head(hidden, weight, tokens, temperature):
    """Raise unless these are a head_logprobs call."""
    what = "head_logprobs"
    if not hidden.dim() or not hidden.is_floating_point() or hidden.shape[-1] < 1:
        raise ValueError(f"{what}: hidden states (..., d) expected, got {tuple(hidden.shape)} {hidden.dtype}")
    if weight.dim() != 2 or weight.shape[0] < 1 or weight.shape[1] != hidden.shape[-1]:
        raise ValueError(f"{what}: weight (V, {hidden.shape[-1]}) expected, got {tuple(weight.shape)}")
    if weight.dtype != hidden.dtype:
        raise TypeError(f"{what}: weight of {weight.dtype} for hidden states of {hidden.dtype}")
    if tokens.dtype not in _INTS:
        raise TypeError(f"{what}: tokens must be int32 or int64, got {tokens.dtype}")
    if tokens.shape != hidden.shape[:-1]:
        raise ValueError(f"{what}: tokens {tuple(tokens.shape)} for hidden states {tuple(hidden.shape)}")
    if not 2.0 ** -126 <= temperature <= 2.0 ** 126:
        raise ValueError(f"{what}: temperature {temperature} must be positive and finite (2^-126 to 2^126)")
    if torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad):
        raise RuntimeError(f"{what}: no gradient flows to the hidden states or the weight; call it under torch.no_grad(), or "
                           "token_logprobs on the logits")


def preference_loss(logits, tokens, reference=None, beta=0.1, loss="sigmoid", average=False, margin=0.0, label_smoothing=0.0,
                    ignore_index=-100, reduction="mean"):
    """fused_logprobs.preference_loss as torch operations."""
    check_preference(logits, tokens, reference, beta, loss, margin, label_smoothing, reduction)
    live, lp, _ = _values(logits, tokens, 1.0, ignore_index, False)
    n = logits.shape[0] // 2
    # (a sum of thousands, differences of which count)
    sums = lp.double().sum(1)
    if average:
        sums = sums / live.sum(1).clamp(min=1)
    gain = sums if reference is None else sums - reference.double()
    d = gain[:n] - gain[n:]
    x = beta * d - margin
    if loss == "sigmoid":
        pairs = -(1.0 - label_smoothing) * torch.nn.functional.logsigmoid(x)
        if label_smoothing:
            pairs = pairs - label_smoothing * torch.nn.functional.logsigmoid(-x)
    elif loss == "hinge":
        # (a factor of NaN: a broken pair's gradient is NaN too)
        pairs = torch.where(x >= 1.0, torch.zeros_like(x), 1.0 - x) * torch.where(x.isnan(), math.nan, 1.0)
    else:
        pairs = (d - 0.5 / beta) ** 2
    out = pairs if reduction == "none" else pairs.sum() / n if reduction == "mean" and n else \
        pairs.sum() * math.nan if reduction == "mean" else pairs.sum()
    return out.to(lp.dtype), sums.detach().to(lp.dtype)


def policy_loss(logits, tokens, old_logprobs, advantages, reference_logprobs=None, clip=0.2, clip_high=None, kl_weight=0.0,
                entropy_weight=0.0, temperature=1.0, ignore_index=-100, reduction="mean"):
    """fused_logprobs.policy_loss as torch operations."""
    clip_high = clip if clip_high is None else clip_high
    check_policy(logits, tokens, old_logprobs, advantages, reference_logprobs, clip, clip_high, kl_weight, entropy_weight,
                 temperature, reduction)
    live, lp, ent = _values(logits, tokens, temperature, ignore_index, entropy_weight != 0.0)
    zero = torch.zeros((), dtype=lp.dtype, device=lp.device)

    def known(t):                          # (what stands at ignored positions reaches nothing)
        return torch.where(live, t.to(lp.dtype), zero)
    A = known(advantages.unsqueeze(-1).expand(tokens.shape) if advantages.dim() < tokens.dim() else advantages)
    moved = lp - known(old_logprobs)
    ratio, low, high = moved.detach().exp(), 1.0 - clip, 1.0 + clip_high
    off = ((A > 0) & (ratio > high)) | ((A < 0) & (ratio < low))
    clipped = -torch.where(A > 0, torch.full_like(A, high), torch.full_like(A, low)) * A
    # (a clipped ratio may be infinite: no 0 * inf in its gradient)
    rows = torch.where(off, clipped, -torch.exp(torch.where(off, zero, moved)) * A)
    if kl_weight:
        d = known(reference_logprobs) - lp
        rows = rows + kl_weight * (torch.expm1(d) - d)
    if entropy_weight:
        rows = rows - entropy_weight * ent
    rows = torch.where(live, rows, zero)
    if reduction == "none":
        out = rows
    elif reduction == "sequence":
        count = live.sum(-1)
        out = (rows.sum(-1) / count.clamp(min=1)).sum() / (count > 0).sum()
    else:
        out = rows.sum() / live.sum() if reduction == "mean" else rows.sum()
    return out, lp.detach()
