"""The post-training formulas as torch operations where numbers end: what the kernels are held to there (test_gpu_logprobs_limits)."""

import math

import pytest
import torch

from dispatcher_hybrid import logprobs as plain

LEAST = 2.0 ** -126


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_least_temperature(dtype):
    """Probabilities of 0 and 1, though a logit of 4 or more over the temperature is past fp32: log-probabilities of 0 and of differences
    over the temperature, entropies of 0, gradients (a ([v = y] - p_v)) / tau."""
    z = torch.tensor([[9.0, 1.0, -3.0], [9.0, 8.5, -math.inf], [2.0, 9.0, 9.0], [-5.0, -9.0, -5.5]], dtype=dtype)
    tokens = torch.tensor([0, 1, 1, 2])
    leaf = z.clone().requires_grad_()
    lp, ent = plain.token_logprobs(leaf, tokens, LEAST, entropy=True)
    assert lp.tolist()[:2] == [0.0, -0.5 / LEAST] and lp[3] == -0.5 / LEAST
    assert ent[[0, 1, 3]].tolist() == [0.0] * 3
    assert abs(lp[2] + math.log(2)) < 1e-6 and abs(ent[2] - math.log(2)) < 1e-6
    a, e = torch.tensor([5.0, 1.0, 2.0, -1.0]), torch.tensor([1.0, -2.0, 0.0, 3.0])
    dz, = torch.autograd.grad((lp, ent), leaf, (a, e))
    want = torch.tensor([[0.0, 0.0, 0.0], [-1.0, 1.0, 0.0], [0.0, 1.0, -1.0], [1.0, 0.0, -1.0]], dtype=torch.float64) / LEAST
    assert ((dz.double() - want).abs() <= 1e-6 * want.abs()).all()


def test_small_temperatures_against_float64():
    """Two more roundings than before a softmax of large numbers: the shift's (half a step of the difference) and the quotient's."""
    g = torch.Generator().manual_seed(1)
    z = 3 * torch.randn(40, 300, generator=g)
    z[:, ::7] = -math.inf
    tokens = torch.randint(1, 7, (40,), generator=g) + 7 * torch.randint(0, 42, (40,), generator=g)
    for tau in (0.9, 0.05, 1e-4):
        lp, ent = plain.token_logprobs(z, tokens, tau, entropy=True)
        x = z.double() / tau
        ref = torch.log_softmax(x, -1)
        want = ref.gather(1, tokens.unsqueeze(1)).squeeze(1)
        d = (x - x.max(1, keepdim=True).values).clamp(min=-800)
        p = ref.exp()
        # an exponent is off by 3 half steps of itself, a sum of 300 by as many, a logarithm and the difference by one each
        slack = 2.0 ** -24 * ((p * 3 * d.abs()).sum(1) + 310)
        assert ((lp.double() - want).abs() <= slack + 2.0 ** -24 * 5 * want.abs()).all()
        h = -(p * ref.clamp(min=-800)).sum(1)
        assert ((ent.double() - h).abs() <= 4 * (slack * (1 + h) + 2.0 ** -24 * (p * d * d).sum(1))).all()


def closed_pairs():
    """Two pairs of one token each, the answer of the first pair's preferred sequence of probability 0."""
    z = torch.tensor([[[1.0, -math.inf, 0.0]], [[0.5, 1.0, 2.0]], [[0.0, 1.0, 2.0]], [[2.0, 0.0, 1.0]]])
    return z.requires_grad_(), torch.tensor([[1], [0], [0], [1]])


def test_preference_of_a_closed_token():
    """An answer of probability 0 has a log-probability of -inf. The slopes of the sigmoid and the hinge are bounded, so its pair's
    gradients are numbers; that of the squared loss is infinite, and a probability of 0 times it NaN. The other pair has its own."""
    for first in (True, False):
        for kind in ("sigmoid", "hinge", "squared"):
            z, tokens = closed_pairs()
            if not first:                                        # the closed answer is the one that is not preferred
                z, tokens = z.detach().roll(2, 0).requires_grad_(), tokens.roll(2, 0)
            loss, sums = plain.preference_loss(z, tokens, loss=kind, reduction="none")
            assert sums.isinf().tolist() == [first, False, not first, False]
            dz, = torch.autograd.grad(loss.sum(), z)
            assert loss[1].isfinite() and dz[[1, 3]].isfinite().all()
            if kind == "squared":
                assert loss[0] == math.inf and not dz[[0, 2]].isfinite().any() and dz[[0, 2]].isnan().any()
            else:
                assert loss[0] == (math.inf if first else 0.0) and dz[[0, 2]].isfinite().all()


def test_policy_of_a_closed_token_and_of_a_ratio_past_fp32():
    """A closed token has a ratio of 0, and with a KL term a slope of -inf; a ratio of e^95 that its advantage does not clip is inf."""
    z, tokens = closed_pairs()
    ones, low = torch.ones(4, 1), torch.full((4, 1), -2.0)
    loss, _ = plain.policy_loss(z, tokens, low, ones, reduction="none")
    dz, = torch.autograd.grad(loss.sum(), z)
    assert loss[0] == 0 and loss.isfinite().all() and dz.isfinite().all()
    loss, _ = plain.policy_loss(z, tokens, low, ones, low, kl_weight=0.1, reduction="none")
    dz, = torch.autograd.grad(loss.sum(), z)
    assert loss[0].isnan() and not dz[0].isfinite().any() and loss[1:].isfinite().all() and dz[1:].isfinite().all()
    old = torch.tensor([[-2.0], [-97.0], [-2.0], [-97.0]])
    loss, _ = plain.policy_loss(z, tokens, old, torch.tensor([[1.0], [-1.0], [1.0], [1.0]]), reduction="none")
    dz, = torch.autograd.grad(loss.sum(), z)
    assert loss[1] == math.inf and not dz[1].isfinite().any() and dz[1].isnan().any()
    assert loss[3] == -torch.tensor(1.2) and not dz[3].any()     # clipped
