"""The post-training operators without a GPU: the formulas against a row-by-row computation in float64 and against differences,
what the entry points refuse (before any device work), and the model's losses on log-probabilities."""

import math

import numpy as np
import pytest
import torch

from dispatcher_hybrid import logprobs as plain
from helpers import product_model, tiny

IGNORE = -100


def rows_of(z, tokens, tau):
    """(log-probabilities, entropies), numpy float64, from the definition."""
    z = np.asarray(z, np.float64)
    lp, ent = np.zeros(len(z)), np.zeros(len(z))
    for n, y in enumerate(tokens):
        if y == IGNORE:
            continue
        p = np.exp(z[n] / tau - (z[n] / tau).max())
        p /= p.sum()
        lp[n] = math.log(p[y]) if p[y] else -math.inf
        ent[n] = -sum(q * math.log(q) for q in p if q > 0)
    return lp, ent


def case(lead, V, seed, ignored=0.25):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(*lead, V, generator=g, dtype=torch.float64) * 2
    tokens = torch.randint(0, V, lead, generator=g)
    tokens[torch.rand(lead, generator=g) < ignored] = IGNORE
    return z, tokens, g


@pytest.mark.parametrize("tau", [1.0, 0.6, 2.5])
def test_logprobs_against_rows(tau):
    z, tokens, _ = case((9,), 17, 1)
    z[2, :9] = -math.inf
    tokens[2] = 12
    lp, ent = plain.token_logprobs(z, tokens, tau, entropy=True)
    ref = rows_of(z.numpy(), tokens.tolist(), tau)
    # float64, 17 terms
    assert np.abs(lp.numpy() - ref[0]).max() < 1e-12 and np.abs(ent.numpy() - ref[1]).max() < 1e-12
    zz = z[3:].clone().requires_grad_()
    f = lambda x: plain.token_logprobs(x, tokens[3:], tau, entropy=True)
    assert torch.autograd.gradcheck(f, zz) and torch.autograd.gradgradcheck(f, zz)


def test_masked_and_broken_positions():
    z, tokens, _ = case((6,), 11, 2, ignored=0.0)
    tokens[1], tokens[2], tokens[3] = IGNORE, 11, -3
    z[1] = math.nan
    z[4, tokens[4]] = -math.inf
    z[5, :] = torch.finfo(torch.float64).min / 4
    zz = z.clone().requires_grad_()
    lp, ent = plain.token_logprobs(zz, tokens, entropy=True)
    assert lp.isnan().tolist() == ent.isnan().tolist() == [False, False, True, True, False, False]
    assert lp[1] == 0 and ent[1] == 0 and lp[4] == -math.inf and abs(ent[5].item() - math.log(11)) < 1e-12
    dz, = torch.autograd.grad(lp[:4].sum() + ent.sum(), zz)
    assert not dz[1].any() and dz[2].isnan().all() and dz[3].isnan().all() and dz[[0, 4, 5]].isfinite().all()


KINDS = [("sigmoid", 0.1, False, 0.0, 0.0), ("sigmoid", 0.7, True, 0.4, 0.2), ("hinge", 0.3, False, 0.2, 0.0), ("squared", 0.2, True, 0.0, 0.0)]


@pytest.mark.parametrize("kind,beta,average,margin,eps", KINDS)
def test_preference_against_pairs(kind, beta, average, margin, eps):
    n, T, V = 3, 5, 13
    z, tokens, g = case((2 * n, T), V, 3)
    tokens[4] = IGNORE
    reference = torch.randn(2 * n, generator=g, dtype=torch.float64) * 3 - 9
    lp = rows_of(z.reshape(-1, V).numpy(), tokens.flatten().tolist(), 1.0)[0].reshape(2 * n, T)
    count = (tokens != IGNORE).sum(1).numpy()
    S = lp.sum(1) / (np.maximum(count, 1) if average else 1)
    for ref in (reference, None):
        gain = S - (0 if ref is None else ref.numpy())
        want = []
        for i in range(n):
            d = gain[i] - gain[n + i]
            x = beta * d - margin
            want.append({"sigmoid": lambda: (1 - eps) * math.log1p(math.exp(-x)) + eps * math.log1p(math.exp(x)),
                         "hinge": lambda: max(0.0, 1 - x), "squared": lambda: (d - 0.5 / beta) ** 2}[kind]())
        args = dict(beta=beta, loss=kind, average=average, margin=margin, label_smoothing=eps)
        pairs, sums = plain.preference_loss(z, tokens, ref, reduction="none", **args)
        assert np.abs(sums.numpy() - S).max() < 1e-11 and np.abs(pairs.numpy() - want).max() < 1e-11
        assert abs(plain.preference_loss(z, tokens, ref, **args)[0].item() - np.mean(want)) < 1e-11
        assert abs(plain.preference_loss(z, tokens, ref, reduction="sum", **args)[0].item() - np.sum(want)) < 1e-11
        f = lambda x: plain.preference_loss(x, tokens, ref, **args)[0]
        assert torch.autograd.gradcheck(f, z.clone().requires_grad_())


@pytest.mark.parametrize("kind,beta,average,margin,eps", KINDS)
def test_a_broken_pair_is_nan_throughout(kind, beta, average, margin, eps):
    z, tokens, _ = case((4, 3), 7, 8, ignored=0.0)
    tokens[2, 1], tokens[0, 2] = 7, IGNORE                     # outside the vocabulary; no part of an answer
    zz = z.clone().requires_grad_()
    pairs, sums = plain.preference_loss(zz, tokens, beta=beta, loss=kind, average=average, margin=margin, label_smoothing=eps,
                                        reduction="none")
    dz, = torch.autograd.grad(pairs.sum(), zz)
    assert pairs.isnan().tolist() == [True, False] and sums.isnan().tolist() == [False, False, True, False]
    live = tokens != IGNORE
    assert dz[[0, 2]][live[[0, 2]]].isnan().all() and not dz[0, 2].any() and dz[[1, 3]].isfinite().all()


@pytest.mark.parametrize("clip,high,kl,w,per_sequence", [(0.2, None, 0.0, 0.0, False), (0.1, 0.4, 0.3, 0.02, True), (1.0, 0.5, 0.0, 0.1, True)])
def test_policy_against_rows(clip, high, kl, w, per_sequence):
    B, T, V, tau = 3, 6, 13, 0.8
    z, tokens, g = case((B, T), V, 4)
    tokens[1] = IGNORE
    lp, ent = (x.reshape(B, T) for x in rows_of(z.reshape(-1, V).numpy(), tokens.flatten().tolist(), tau))
    old = torch.tensor(lp) + 0.3 * torch.randn(B, T, generator=g, dtype=torch.float64)
    ref = torch.tensor(lp) + 0.3 * torch.randn(B, T, generator=g, dtype=torch.float64)
    adv = torch.randn((B,) if per_sequence else (B, T), generator=g, dtype=torch.float64)
    old[tokens == IGNORE] = math.nan                           # nothing of an ignored position is looked at
    lo, hi = 1 - clip, 1 + (clip if high is None else high)
    rows = np.zeros((B, T))
    for b in range(B):
        for t in range(T):
            if tokens[b, t] == IGNORE:
                continue
            A, r = (adv[b] if per_sequence else adv[b, t]).item(), math.exp(lp[b, t] - old[b, t])
            d = ref[b, t].item() - lp[b, t]
            rows[b, t] = -min(r * A, min(max(r, lo), hi) * A) + kl * (math.exp(d) - d - 1) - w * ent[b, t]
    args = dict(reference_logprobs=ref if kl else None, clip=clip, clip_high=high, kl_weight=kl, entropy_weight=w, temperature=tau)
    live = (tokens != IGNORE).numpy()
    got = {r: plain.policy_loss(z, tokens, old, adv, reduction=r, **args)[0] for r in plain.TOKEN_REDUCTIONS}
    assert np.abs(got["none"].numpy() - rows).max() < 1e-11
    assert abs(got["sum"].item() - rows.sum()) < 1e-11 and abs(got["mean"].item() - rows.sum() / live.sum()) < 1e-11
    means = [rows[b].sum() / live[b].sum() for b in range(B) if live[b].any()]
    assert abs(got["sequence"].item() - np.mean(means)) < 1e-11
    for r in ("mean", "sequence"):
        f = lambda x: plain.policy_loss(x, tokens, old, adv, reduction=r, **args)[0]
        assert torch.autograd.gradcheck(f, z.clone().requires_grad_())


def test_nothing_to_average():
    z = torch.randn(2, 3, 7, requires_grad=True)
    none = torch.full((2, 3), IGNORE)
    old = torch.zeros(2, 3)
    for reduction in ("mean", "sequence"):
        loss, _ = plain.policy_loss(z, none, old, old, reduction=reduction)
        assert math.isnan(loss.item()) and not torch.autograd.grad(loss, z)[0].nan_to_num().any()
    loss, sums = plain.preference_loss(z, none)
    assert abs(loss.item() - math.log(2)) < 1e-6 and not sums.any()
    loss, _ = plain.preference_loss(z[:0], none[:0])
    assert math.isnan(loss.item())


def refused():
    z, tok = torch.randn(2, 3, 8), torch.zeros(2, 3, dtype=torch.long)
    h, w = torch.randn(2, 3, 4), torch.randn(8, 4)
    old, adv, ref = torch.zeros(2, 3), torch.zeros(2), torch.zeros(2)
    grad = lambda t: t.clone().requires_grad_()
    return [
        ("token_logprobs", ValueError, "vocabulary", (z.long(), tok), {}),
        ("token_logprobs", ValueError, "empty", (z[..., :0], tok), {}),
        ("token_logprobs", ValueError, "tokens", (z, tok[0]), {}),
        ("token_logprobs", TypeError, "tokens", (z, tok.float()), {}),
        ("token_logprobs", TypeError, "tokens", (z, tok.short()), {}),
        ("token_logprobs", ValueError, "temperature", (z, tok), dict(temperature=0.0)),
        ("token_logprobs", ValueError, "temperature", (z, tok), dict(temperature=math.nan)),
        ("token_logprobs", ValueError, "temperature", (z, tok), dict(temperature=-1.0)),
        ("head_logprobs", ValueError, "weight", (h, w[:, :3], tok), {}),
        ("head_logprobs", ValueError, "weight", (h, w[0], tok), {}),
        ("head_logprobs", TypeError, "weight", (h, w.bfloat16(), tok), {}),
        ("head_logprobs", ValueError, "tokens", (h, w, tok[:1]), {}),
        ("head_logprobs", TypeError, "tokens", (h, w, tok.float()), {}),
        ("head_logprobs", ValueError, "hidden", (h[..., :0], w[:, :0], tok), {}),
        ("head_logprobs", ValueError, "temperature", (h, w, tok), dict(temperature=math.inf)),
        ("head_logprobs", RuntimeError, "no gradient", (grad(h), w, tok), {}),
        ("head_logprobs", RuntimeError, "no gradient", (h, grad(w), tok), {}),
        ("preference_loss", ValueError, "2 n", (z[0], tok[0]), {}),
        ("preference_loss", ValueError, "2 n", (torch.randn(3, 3, 8), torch.zeros(3, 3, dtype=torch.long)), {}),
        ("preference_loss", ValueError, "reference", (z, tok, torch.zeros(3)), {}),
        ("preference_loss", ValueError, "constants", (z, tok, grad(ref)), {}),
        ("preference_loss", TypeError, "reference", (z, tok, ref.long()), {}),
        ("preference_loss", ValueError, "loss", (z, tok), dict(loss="dpo")),
        ("preference_loss", ValueError, "beta", (z, tok), dict(beta=0.0)),
        ("preference_loss", ValueError, "margin", (z, tok), dict(margin=math.inf)),
        ("preference_loss", ValueError, "label_smoothing", (z, tok), dict(label_smoothing=0.6)),
        ("preference_loss", ValueError, "no margin", (z, tok), dict(loss="squared", margin=1.0)),
        ("preference_loss", ValueError, "no label_smoothing", (z, tok), dict(loss="hinge", label_smoothing=0.1)),
        ("preference_loss", ValueError, "reduction", (z, tok), dict(reduction="sequence")),
        ("policy_loss", ValueError, "T, vocabulary", (z[0, 0], tok[0, 0], old[0, 0], old[0, 0]), {}),
        ("policy_loss", ValueError, "old", (z, tok, old[:1], adv), {}),
        ("policy_loss", TypeError, "old", (z, tok, tok, adv), {}),
        ("policy_loss", ValueError, "constants", (z, tok, grad(old), adv), {}),
        ("policy_loss", ValueError, "advantages", (z, tok, old, adv[:1]), {}),
        ("policy_loss", ValueError, "advantages", (z, tok, old, old.t()), {}),
        ("policy_loss", ValueError, "reference", (z, tok, old, adv, old[:1]), {}),
        ("policy_loss", ValueError, "reference_logprobs", (z, tok, old, adv), dict(kl_weight=0.1)),
        ("policy_loss", ValueError, "clip", (z, tok, old, adv), dict(clip=1.5)),
        ("policy_loss", ValueError, "clip", (z, tok, old, adv), dict(clip_high=math.nan)),
        ("policy_loss", ValueError, "kl_weight", (z, tok, old, adv, old), dict(kl_weight=-1.0)),
        ("policy_loss", ValueError, "entropy_weight", (z, tok, old, adv), dict(entropy_weight=math.inf)),
        ("policy_loss", ValueError, "reduction", (z, tok, old, adv), dict(reduction="avg")),
    ]


@pytest.mark.parametrize("i", range(42))
def test_refusals(i):
    from dispatcher_hybrid import fused_logprobs as fl
    assert len(refused()) == 42
    name, exc, match, args, kw = refused()[i]
    for module in (plain, fl):
        with pytest.raises(exc, match=match):
            getattr(module, name)(*args, **kw)


def test_kernel_entry_points_refuse_cpu_tensors():
    from dispatcher_hybrid import fused_logprobs as fl
    z, tok, old = torch.randn(2, 3, 8), torch.zeros(2, 3, dtype=torch.long), torch.zeros(2, 3)
    for call in (lambda: fl.token_logprobs(z, tok), lambda: fl.head_logprobs(z, torch.randn(5, 8), tok),
                 lambda: fl.preference_loss(z, tok), lambda: fl.policy_loss(z, tok, old, old)):
        with pytest.raises(RuntimeError, match="on the GPU"):
            call()


def test_c_entry_points_refuse_before_any_launch():
    from dispatcher_hybrid import _hip
    lib, N, one = _hip.lib, None, 256                          # never dereferenced: every call is refused

    def fwd(**kw):
        a = dict(dtype=1, z=one, sb=8, st=8, B=1, T=2, V=8, tok=one, bits=64, ignore=-100, tau=1.0, lp=one, ent=one, kept=one, ws=N, nb=0)
        a.update(kw)
        return lib.dh_logprob_fwd(*a.values(), N)
    for kw, code in ((dict(dtype=5), 3), (dict(bits=16), 3), (dict(V=0), 2), (dict(V=(1 << 24) + 1), 2), (dict(B=1 << 22), 2),
                     (dict(B=-1), 2), (dict(T=0), 2), (dict(tau=0.0), 1), (dict(tau=1e-40), 1), (dict(tau=math.nan), 1), (dict(tau=1e39), 1),
                     (dict(z=N), 1), (dict(tok=N), 1), (dict(lp=N), 1), (dict(z=one + 1), 1), (dict(tok=one + 4), 1), (dict(lp=one + 2), 1),
                     (dict(ent=one + 1), 1), (dict(kept=one + 8), 1), (dict(V=1 << 20, ws=N), 1), (dict(dtype=0, z=one + 2), 1)):
        assert fwd(**kw) == code, kw
    assert lib.dh_logprob_workspace_bytes(1, 1, 1 << 20) > 0 and lib.dh_logprob_workspace_bytes(1, 1 << 20, 1 << 20) == 0
    assert lib.dh_logprob_workspace_bytes(1, -1, 8) == lib.dh_logprob_workspace_bytes(1, 8, 0) == -1

    def bwd(**kw):
        a = dict(dtype=1, z=one, sb=8, st=8, B=1, T=2, V=8, tok=one, bits=64, ignore=-100, tau=1.0, kept=one, lp=one, div=1, ls=1,
                 ent=N, es=0, g=N, gd=1, gm=1, gs=0, divisor=N, dz=one)
        a.update(kw)
        return lib.dh_logprob_bwd(*a.values(), N)
    for kw in (dict(kept=N), dict(kept=one + 4), dict(lp=N), dict(dz=N), dict(dz=one + 1), dict(div=0), dict(ls=-1), dict(ent=one + 2),
               dict(g=one, gd=0), dict(g=one, gm=0), dict(g=one, gs=-1), dict(g=one + 2), dict(divisor=one + 1)):
        assert bwd(**kw) == 1, kw

    def pref(**kw):
        a = dict(dtype=1, z=one, sb=8, st=8, pairs=2, T=2, V=8, tok=one, bits=64, ignore=-100, ref=N, rbits=32, kind=0, average=0,
                 beta=0.1, margin=0.0, eps=0.0, red=1, pl=one, sums=one, coef=one, kept=one, loss=one, div=one, ws=one, nb=1 << 20)
        a.update(kw)
        return lib.dh_preference_fwd(*a.values(), N)
    for kw, code in ((dict(pairs=-1), 2), (dict(T=-1), 2), (dict(pairs=1 << 21), 2), (dict(pairs=1 << 11, T=1 << 11), 2), (dict(kind=3), 1),
                     (dict(red=3), 1), (dict(beta=0.0), 1), (dict(beta=math.nan), 1), (dict(margin=math.nan), 1), (dict(eps=0.7), 1),
                     (dict(ref=one, rbits=16), 3), (dict(ref=one + 4, rbits=64), 1), (dict(sums=N), 1), (dict(coef=N), 1), (dict(kept=N), 1),
                     (dict(loss=N), 1), (dict(red=0, pl=N), 1), (dict(ws=N), 1), (dict(nb=8), 1), (dict(ws=one + 4), 1), (dict(dtype=9), 3)):
        assert pref(**kw) == code, kw

    def policy(**kw):
        a = dict(dtype=1, z=one, sb=8, st=8, B=2, T=2, V=8, tok=one, bits=64, ignore=-100, tau=1.0, old=one, adv=one, per=0, ref=N,
                 clip=0.2, high=0.2, kl=0.0, w=0.0, red=1, rl=one, lp=one, by=one, be=N, kept=one, loss=one, div=one, ws=one, nb=1 << 20)
        a.update(kw)
        return lib.dh_policy_fwd(*a.values(), N)
    for kw, code in ((dict(B=-1), 2), (dict(B=1 << 22), 2), (dict(V=0), 2), (dict(red=4), 1), (dict(clip=-0.1), 1), (dict(clip=1.1), 1),
                     (dict(high=math.inf), 1), (dict(kl=0.1), 1), (dict(w=0.1), 1), (dict(be=one, w=math.nan), 1), (dict(old=N), 1),
                     (dict(adv=N), 1), (dict(by=N), 1), (dict(kept=N), 1), (dict(loss=N), 1), (dict(red=0, rl=N), 1), (dict(nb=0), 1),
                     (dict(lp=one + 2), 1), (dict(tau=0.0), 1)):
        assert policy(**kw) == code, kw

    def head(**kw):
        a = dict(dtype=1, h=one, hs=64, rows=4, d=64, w=one, wsr=64, V=8, tok=one, bits=64, ignore=-100, tau=1.0, rnd=0, lp=one, ent=N,
                 ws=one, nb=1 << 30)
        a.update(kw)
        return lib.dh_head_logprob(*a.values(), N)
    for kw, code in ((dict(dtype=2), 3), (dict(bits=8), 3), (dict(rows=-1), 2), (dict(rows=1 << 22), 2), (dict(d=0), 2), (dict(d=(1 << 20) + 1), 2),
                     (dict(V=0), 2), (dict(tau=0.0), 1), (dict(h=N), 1), (dict(w=N), 1), (dict(tok=N), 1), (dict(lp=N), 1), (dict(hs=-1), 1),
                     (dict(wsr=-64), 1), (dict(h=one + 1), 1), (dict(ent=one + 2), 1), (dict(nb=0), 1), (dict(ws=one + 8), 1)):
        assert head(**kw) == code, kw
    assert lib.dh_head_logprob_workspace_bytes(1, 1 << 22, 8) == lib.dh_head_logprob_workspace_bytes(3, 1, 8) == -1


def test_model_scores_and_trains_on_the_cpu():
    cfgd, sd = tiny("tiny_a")
    m = product_model(cfgd, sd).train()
    g = torch.Generator().manual_seed(1)
    ids = torch.randint(0, 255, (4, 20), generator=g)
    labels = ids.clone()
    labels[:, :6] = IGNORE
    labels[1, 15:] = IGNORE
    logits = m(ids).logits
    moved = torch.cat([labels[:, 1:], torch.full((4, 1), IGNORE)], 1)
    lp, ent = m.token_logprobs(ids, labels, temperature=0.7, entropy=True)
    want = plain.token_logprobs(logits.double(), moved, 0.7, entropy=True)
    assert lp.shape == (4, 20) and not lp.requires_grad and (lp - want[0]).abs().max() < 1e-5 and (ent - want[1]).abs().max() < 1e-5
    assert not m.token_logprobs(ids)[:, -1].any() and (m.token_logprobs(ids)[:, :-1] < 0).all()
    reference = m.token_logprobs(ids, labels).sum(1) + torch.randn(4, generator=g)
    out = m(ids, labels=labels, preference=dict(reference=reference, beta=0.3))
    ref = plain.preference_loss(logits.double(), moved, reference, beta=0.3)
    assert abs(out.loss.item() - ref[0].item()) < 1e-5 and (out.logprobs - ref[1]).abs().max() < 1e-4
    out.loss.backward()
    assert all(p.grad is not None and bool(p.grad.isfinite().all()) for p in m.parameters())
    old = m.token_logprobs(ids, labels) + 0.1 * torch.randn(4, 20, generator=g)
    policy = dict(old_logprobs=old, advantages=torch.randn(4, generator=g), reference_logprobs=old, kl_weight=0.1, entropy_weight=0.01,
                  reduction="sequence")
    out = m(ids, labels=labels, policy=policy)
    ref = plain.policy_loss(logits.double(), moved, **policy)
    assert abs(out.loss.item() - ref[0].item()) < 1e-5 and (out.logprobs - ref[1]).abs().max() < 1e-5
    out.loss.backward()
    loss, z, scores = m(ids, labels=labels, policy=policy, return_dict=False)
    assert torch.equal(scores, out.logprobs) and z.shape == logits.shape
    with pytest.raises(ValueError, match="labels"):
        m(ids, policy=policy)
    with pytest.raises(ValueError, match="one of"):
        m(ids, labels=labels, policy=policy, preference={})
    with pytest.raises(TypeError):
        m(ids, labels=labels, preference=dict(betta=1.0))
    m.enable_fused_vocab()
    for call in (lambda: m(ids, labels=labels, preference={}), lambda: m(ids, labels=labels, policy=policy), lambda: m.token_logprobs(ids)):
        with pytest.raises(RuntimeError, match="CPU"):
            call()


@pytest.mark.parametrize("name", ["preference", "policy"])
def test_model_losses_ignore_what_labels_ignore(name):
    """(the last position has no next token: with another ignore_index it would count as a token outside the vocabulary)"""
    cfgd, sd = tiny("tiny_a")
    m = product_model(cfgd, sd)
    ids = torch.randint(0, 255, (2, 8), generator=torch.Generator().manual_seed(2))
    args = dict(old_logprobs=torch.zeros(2, 8), advantages=torch.ones(2)) if name == "policy" else {}
    with pytest.raises(ValueError, match="-100"):
        m(ids, labels=ids, **{name: dict(args, ignore_index=0)})
    out = m(ids, labels=ids, **{name: dict(args, ignore_index=IGNORE)})
    assert bool(out.loss.isfinite())
