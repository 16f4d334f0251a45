"""The post-training operators where numbers end: temperatures at the ends of their range with gradients. Bounds: test_gpu_logprobs."""

import pytest
import torch

from test_gpu_logprobs import DEV, TYPES, Rows, gen, inputs, ops, say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,V", [(6, 3001), (6, 50257), (1100, 1003), (1100, 9001)])
def test_gradients_at_extreme_temperatures(rows, V, dtype):
    """The least temperature, 2^-126: a row with one largest logit has probabilities of 0 and 1. dz_v = (a ([v = y] - p_v) - 0) / tau:
    0 throughout where the token is that logit, elsewhere a / tau at the token, -a / tau at the largest and 0 at the others, whatever
    the gradient in the entropy. All of them are numbers of either type."""
    say("extreme", rows, V, dtype)
    z, tokens = inputs((rows,), V, dtype, 31, ignored=0.0)
    most = (z + torch.rand(z.shape, device=DEV, generator=gen(32))).argmax(1)
    z.scatter_(1, most.unsqueeze(1), 16.0)                       # (the others are below 12)
    tokens = torch.where(most == tokens, (tokens + 1) % V, tokens)
    tokens[::2] = most[::2]
    at = torch.arange(rows, device=DEV)
    a = torch.tensor([8.0, 1.0, -5.0, -0.5], device=DEV)[at % 4]  # 8 / tau is past fp32: nothing of it is in a row of zeros
    e = torch.tensor([0.5, -300.0, 1e6], device=DEV)[at % 3]
    tau = 2.0 ** -126
    leaf = z.clone().requires_grad_()
    lp, ent = ops().token_logprobs(leaf, tokens, temperature=tau, entropy=True)
    want = torch.zeros(rows, V, dtype=torch.float64, device=DEV)
    want[at, tokens] = a.double() / tau
    want[at, most] = -a.double() / tau
    want[::2] = 0.0
    assert bool((torch.autograd.grad((lp, ent), leaf, (a, e), retain_graph=True)[0].double() == want).all())
    assert bool((torch.autograd.grad(lp, leaf, a, retain_graph=True)[0].double() == want).all())
    assert not bool(torch.autograd.grad(ent, leaf, e)[0].any())
    for tau in (1e-3, 300.0, 1e30):                              # (times tau: gradients of ordinary size)
        ref = Rows(z, tokens, tau)
        lp, ent = ops().token_logprobs(leaf, tokens, temperature=tau, entropy=True)
        ref.check_grad(torch.autograd.grad((lp, ent), leaf, (a * tau, e.clamp(-1, 1) * tau))[0], a * tau, e.clamp(-1, 1) * tau)


def test_create_graph_at_the_least_temperature():
    """With create_graph a gradient is the torch formula's: the same numbers."""
    z, tokens = inputs((5,), 1003, torch.float32, 33, ignored=0.0)
    z[:, 7] = 16.0
    tokens[1] = 7
    leaf = z.clone().requires_grad_()
    out = ops().token_logprobs(leaf, tokens, temperature=2.0 ** -126, entropy=True)
    by = (torch.ones(5, device=DEV), torch.ones(5, device=DEV))
    first, = torch.autograd.grad(out, leaf, by, retain_graph=True)
    again, = torch.autograd.grad(out, leaf, by, create_graph=True)
    assert bool(first.isfinite().all()) and torch.equal(first, again.detach())
