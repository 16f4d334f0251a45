"""The vocabulary-end operators without a GPU: the distillation formulas against a row-by-row computation in float64, what
the entry points refuse (before any device work), and the model's loss from a teacher's targets."""

import math

import numpy as np
import pytest
import torch
import torch.nn.functional as F

from dispatcher_hybrid import distillation as plain
from helpers import product_model, tiny


def row_by_row(z, t, k, labels, tau, w, ignore=-100):
    """Losses of the rows and d(sum of losses)/dz, numpy float64, from the definition."""
    z = np.asarray(z, np.float64)
    N, V = z.shape
    loss, grad = np.zeros(N), np.zeros((N, V))
    for n in range(N):
        if labels is not None and labels[n] == ignore:
            continue
        live = [j for j in range(len(k[n])) if k[n][j] >= 0 and t[n][j] != -math.inf]
        q = np.exp(z[n] / tau - (z[n] / tau).max())
        q /= q.sum()
        if live and w > 0:
            e = np.exp(np.array([t[n][j] for j in live]) / tau - max(t[n][j] for j in live) / tau)
            p = e / e.sum()
            for pj, j in zip(p, live):
                if pj > 0:
                    loss[n] += w * tau * tau * pj * (math.log(pj) - math.log(q[k[n][j]]))
                grad[n, k[n][j]] -= w * tau * pj
            grad[n] += w * tau * q
        if labels is not None:
            P = np.exp(z[n] - z[n].max())
            P /= P.sum()
            loss[n] -= (1 - w) * math.log(P[labels[n]])
            grad[n] += (1 - w) * P
            grad[n, labels[n]] -= 1 - w
    return loss, grad


def case(N, V, k, seed, empties=True, repeats=False):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(N, V, generator=g, dtype=torch.float64) * 2
    t = torch.randn(N, k, generator=g, dtype=torch.float64) * 3
    tok = torch.stack([torch.randperm(V, generator=g)[:k] for _ in range(N)])
    if empties:
        tok[torch.rand(N, k, generator=g) < 0.3] = -1
        t[torch.rand(N, k, generator=g) < 0.1] = -math.inf
        tok[0] = -1
    if repeats and k > 2:
        tok[:, 2] = tok[:, 0]
    labels = torch.randint(0, V, (N,), generator=g)
    labels[1 % N] = -100
    return z, t, tok, labels


@pytest.mark.parametrize("tau,w,with_labels", [(1.0, 1.0, False), (2.0, 0.5, True), (0.7, 0.9, True), (3.0, 0.0, True),
                                               (1.0, 0.25, True), (2.0, 1.0, True)])
@pytest.mark.parametrize("repeats", [False, True])
def test_formula_against_rows(tau, w, with_labels, repeats):
    z, t, tok, labels = case(7, 19, 5, 3, repeats=repeats)
    labels = labels if with_labels else None
    ref, grad = row_by_row(z, t.tolist(), tok.tolist(), None if labels is None else labels.tolist(), tau, w)
    zz = z.clone().requires_grad_()
    rows = plain.distillation_loss(zz, t, tok, labels, tau, w, reduction="none")
    rows.sum().backward()
    # float64 throughout, 19 terms of magnitude < 100 a sum
    assert np.abs(rows.detach().numpy() - ref).max() < 1e-12
    assert np.abs(zz.grad.numpy() - grad).max() < 1e-12
    count = 7 if labels is None else int((labels != -100).sum())
    assert abs(plain.distillation_loss(z, t, tok, labels, tau, w).item() - ref.sum() / count) < 1e-12
    assert abs(plain.distillation_loss(z, t, tok, labels, tau, w, reduction="sum").item() - ref.sum()) < 1e-11


def test_formula_is_the_cross_entropy_without_a_teacher_and_the_divergence_with_all_of_it():
    z, t, tok, labels = case(6, 11, 11, 5, empties=False)
    ce = F.cross_entropy(z, labels)
    assert abs(plain.distillation_loss(z, t, tok, labels, 2.0, 0.0).item() - ce.item()) < 1e-12
    full = torch.zeros(6, 11, dtype=torch.float64).scatter(1, tok, t)
    kl = F.kl_div(F.log_softmax(z / 2, 1), F.softmax(full / 2, 1), reduction="none").sum(1).mean() * 4
    assert abs(plain.distillation_loss(z, t, tok, None, 2.0).item() - kl.item()) < 1e-12


def test_masked_places_do_not_reach_the_loss():
    z, t, tok, labels = case(5, 13, 4, 7, empties=False)
    tok[2] = -1
    t[2] = math.nan                                            # empty slots may hold anything
    z[1] = math.nan                                            # labels[1] is ignored
    zz = z.clone().requires_grad_()
    rows = plain.distillation_loss(zz, t, tok, labels, 2.0, 0.5, reduction="none")
    rows.sum().backward()
    assert bool(rows.isfinite().all()) and rows[1] == 0 and bool((zz.grad[1] == 0).all())
    assert bool(zz.grad.isfinite().all())
    # every row ignored: the mean of none, and no gradient
    zz.grad = None
    none = plain.distillation_loss(zz, t, tok, torch.full((5,), -100), 2.0, 0.5)
    none.backward()
    assert math.isnan(none.item()) and not bool(zz.grad[2:].isnan().any())
    # a token or label outside the vocabulary: its row alone is NaN
    z, t, tok, labels = case(5, 13, 4, 7, empties=False)
    tok[3, 1], labels[4] = 13, 99
    zz = z.clone().requires_grad_()
    rows = plain.distillation_loss(zz, t, tok, labels, 2.0, 0.5, reduction="none")
    rows.sum().backward()
    assert rows.isnan().tolist() == [False, False, False, True, True]
    assert zz.grad.isnan().all(1).tolist() == [False, False, False, True, True]


def test_formula_gradient_against_differences():
    z, t, tok, labels = case(4, 9, 3, 11)
    fn = lambda x: plain.distillation_loss(x, t, tok, labels, 1.7, 0.6)
    assert torch.autograd.gradcheck(fn, z.clone().requires_grad_())
    assert torch.autograd.gradgradcheck(fn, z.clone().requires_grad_())


def test_top_logits_formula():
    x = torch.tensor([[1.0, 3.0, -0.0, 3.0, 0.0, math.nan, -math.inf]])
    v, i = plain.top_logits(x, 5)
    assert i.tolist() == [[5, 1, 3, 0, 2]] and math.isnan(v[0, 0]) and v[0, 1:].tolist() == [3.0, 3.0, 1.0, 0.0]
    for k in (0, 8, 257):
        with pytest.raises(ValueError, match="k="):
            plain.top_logits(x, k)


def refused():
    z, t, tok, lb = torch.randn(2, 3, 8), torch.randn(2, 3, 4), torch.zeros(2, 3, 4, dtype=torch.long), torch.zeros(2, 3).long()
    return [
        (ValueError, "must both be", (z, t[:, :2], tok[:, :2]), {}),
        (ValueError, "must both be", (z, t, tok[..., :2]), {}),
        (ValueError, "must both be", (z, t[0], tok[0]), {}),
        (ValueError, "0 targets", (z, t[..., :0], tok[..., :0]), {}),
        (ValueError, "257 targets", (z, torch.zeros(2, 3, 257), torch.zeros(2, 3, 257).long()), {}),
        (ValueError, "vocabulary", (z[..., :0], t, tok), {}),
        (ValueError, "constants", (z, t.clone().requires_grad_(), tok), {}),
        (TypeError, "teacher tokens", (z, t, tok.to(torch.int16)), {}),
        (TypeError, "teacher logits", (z, t.long(), tok), {}),
        (TypeError, "labels", (z, t, tok), dict(labels=lb.float(), weight=0.5)),
        (ValueError, "labels", (z, t, tok), dict(labels=lb[0], weight=0.5)),
        (ValueError, "temperature", (z, t, tok), dict(temperature=0.0)),
        (ValueError, "temperature", (z, t, tok), dict(temperature=math.inf)),
        (ValueError, "temperature", (z, t, tok), dict(temperature=math.nan)),
        (ValueError, "weight", (z, t, tok), dict(labels=lb, weight=1.5)),
        (ValueError, "weight", (z, t, tok), dict(labels=lb, weight=math.nan)),
        (ValueError, "none", (z, t, tok), dict(weight=0.5)),
        (ValueError, "reduction", (z, t, tok), dict(reduction="avg")),
    ]


@pytest.mark.parametrize("i", range(18))
def test_loss_refusals(i):
    from dispatcher_hybrid import fused_vocab as fv
    exc, match, args, kw = refused()[i]
    for fn in (plain.distillation_loss, fv.distillation_loss):
        with pytest.raises(exc, match=match):
            fn(*args, **kw)


def test_kernel_entry_points_refuse_cpu_tensors_and_bad_arguments():
    from dispatcher_hybrid import fused_vocab as fv
    W, ids = torch.randn(6, 4), torch.zeros(3, dtype=torch.long)
    for call in (lambda: fv.embed_tokens(ids, W), lambda: fv.top_logits(W, 2),
                 lambda: fv.distillation_loss(W, W[:, :2], ids.new_zeros(6, 2))):
        with pytest.raises(RuntimeError, match="on the GPU"):
            call()
    with pytest.raises(TypeError, match="tokens"):
        fv.embed_tokens(ids.float(), W)
    with pytest.raises(ValueError, match="weight"):
        fv.embed_tokens(ids, W[0])
    for bad in (6, -7):
        with pytest.raises(ValueError, match="padding_idx"):
            fv.embed_tokens(ids, W, padding_idx=bad)
    for k in (0, 5, -1):
        with pytest.raises(ValueError, match="k="):
            fv.top_logits(W, k)


def test_c_entry_points_refuse_before_any_launch():
    from dispatcher_hybrid import _hip
    lib, N = _hip.lib, None
    one = 256                                                  # never dereferenced: every call is refused
    assert lib.dh_embed_fwd(7, one, 8, 8, 8, one, 64, 1, 1.0, -1, one, 8, N) == 3
    assert lib.dh_embed_fwd(1, one, 8, 8, 8, one, 16, 1, 1.0, -1, one, 8, N) == 3
    assert lib.dh_embed_fwd(1, one, 8, 8, 8, one, 64, 1 << 24, 1.0, -1, one, 8, N) == 2
    assert lib.dh_embed_fwd(1, one, 7, 8, 8, one, 64, 1, 1.0, -1, one, 8, N) == 1
    assert lib.dh_embed_fwd(1, N, 8, 8, 8, one, 64, 1, 1.0, -1, one, 8, N) == 1
    for zero in (-2, 9, 1 << 40):                                # -1, a token, or one past them
        assert lib.dh_embed_fwd(1, one, 8, 8, 8, one, 64, 1, 1.0, zero, one, 8, N) == 1 and b"zero_token" in lib.dh_last_error()
    for skip in (-2, 8, (1 << 32) + 3):
        assert lib.dh_embed_bwd(1, one, 8, one, 64, 100, 8, 8, 1.0, skip, one, N, 0, N) == 1 and b"skip_token" in lib.dh_last_error()
    assert lib.dh_embed_bwd_workspace_bytes(1 << 24, 8, 8) == -1
    assert lib.dh_embed_bwd_workspace_bytes(100, 50, 8) == 0     # few positions: one launch
    need = lib.dh_embed_bwd_workspace_bytes(1000, 50, 8)
    assert need > 0
    assert lib.dh_embed_bwd(1, one, 8, one, 64, 1000, 50, 8, 1.0, -1, one, one, need - 1, N) == 1
    assert b"workspace" in lib.dh_last_error()
    assert lib.dh_embed_bwd(1, one + 1, 8, one, 64, 100, 50, 8, 1.0, -1, one, N, 0, N) == 1
    assert b"aligned" in lib.dh_last_error()
    assert lib.dh_embed_bwd(1, one, 8, one, 64, 100, 0, 8, 1.0, -1, one, one, need, N) == 2
    assert lib.dh_top_logits(1, one, 8, 1, 8, 9, one, one, N) == 2 and b"K=9" in lib.dh_last_error()
    assert lib.dh_top_logits(1, one, 8, 1, 8, 0, one, one, N) == 2
    assert lib.dh_top_logits(1, one + 1, 8, 1, 8, 2, one, one, N) == 1
    assert lib.dh_top_logits(1, N, 8, 1, 8, 2, one, one, N) == 1

    def fwd(**kw):
        a = dict(dtype=1, z=one, sb=8, st=8, B=1, T=2, V=8, td=1, tl=one, tt=one, bits=64, K=2, lb=N, lbits=64, ignore=-100,
                 tau=1.0, w=1.0, red=1, rows=one, kept=one, loss=one, div=one, ws=N, nb=0)
        a.update(kw)
        return lib.dh_distill_fwd(*a.values(), N)
    for kw, code in ((dict(dtype=5), 3), (dict(td=5), 3), (dict(bits=8), 3), (dict(lb=one, lbits=8), 3), (dict(K=0), 2),
                     (dict(K=257), 2), (dict(V=0), 2), (dict(B=1 << 22), 2), (dict(tau=0.0), 1), (dict(tau=1e-40), 1), (dict(tau=math.nan), 1),
                     (dict(w=0.5), 1), (dict(w=-1.0), 1), (dict(red=3), 1), (dict(rows=N), 1), (dict(kept=one + 4), 1),
                     (dict(loss=N), 1), (dict(z=N), 1), (dict(V=1 << 20, ws=N), 1)):
        assert fwd(**kw) == code, kw
    assert lib.dh_distill_workspace_bytes(1, 1, 1 << 20) > 0 and lib.dh_distill_workspace_bytes(1, 1 << 20, 1 << 20) == 0


def test_model_trains_on_a_teachers_targets_on_the_cpu():
    cfgd, sd = tiny("tiny_a")
    m = product_model(cfgd, sd).train()
    g = torch.Generator().manual_seed(1)
    ids = torch.randint(0, 255, (2, 20), generator=g)
    values, tokens = m.teacher_targets(ids, 6)
    assert values.shape == tokens.shape == (2, 20, 6) and not values.requires_grad
    logits = m(ids).logits
    assert torch.equal(values, torch.gather(logits.detach(), -1, tokens))
    labels = ids.clone()
    labels[0, 5] = -100
    out = m(ids, labels=labels, teacher_logits=values, teacher_tokens=tokens, distill_temperature=2.0, distill_weight=0.5)
    moved = torch.cat([labels[:, 1:], torch.full((2, 1), -100)], 1)
    ref = plain.distillation_loss(logits.double(), values, tokens, moved, 2.0, 0.5)
    assert abs(out.loss.item() - ref.item()) < 1e-5
    out.loss.backward()
    assert all(p.grad is not None and bool(p.grad.isfinite().all()) for p in m.parameters())
    assert torch.equal(m(ids, labels=labels).loss, F.cross_entropy(logits[:, :-1].reshape(-1, 256), labels[:, 1:].reshape(-1)))
    with pytest.raises(ValueError, match="together"):
        m(ids, teacher_logits=values)
    with pytest.raises(ValueError, match="none"):
        m(ids, teacher_logits=values, teacher_tokens=tokens, distill_weight=0.5)
    m.enable_fused_vocab()
    with pytest.raises(RuntimeError, match="CPU"):
        m(ids, teacher_logits=values, teacher_tokens=tokens)
    m.enable_fused_vocab(False)
    assert m(ids, teacher_logits=values, teacher_tokens=tokens).loss.isfinite()
