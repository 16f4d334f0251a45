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
