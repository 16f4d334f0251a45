"""The post-training operators where numbers end, and rows laid out as they seldom are. Bounds: test_gpu_logprobs."""

import pytest
import torch

from dispatcher_hybrid import logprobs as plain
from test_gpu_logprobs import DEV, TYPES, U, Rows, gen, inputs, ops, say

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


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,V", [(40, 50257), (1500, 1003), (1030, 9001)])
def test_gradients_of_broadcast_rows(rows, V, dtype):
    """One row of logits for many positions (stride 0): every position's gradient against float64, and all of them equal. (A gradient
    row's pieces begin at its own 16-byte boundary, but its elements depend on the row's kept numbers alone; the token's own is a sum
    that may be rounded once or twice.)"""
    say("broadcast", rows, V, dtype)
    z = (2 * torch.randn(1, V, device=DEV, generator=gen(34))).to(dtype).expand(rows, V)
    for entropy in (True, False):
        for token in (5, V - 1):
            tokens = torch.full((rows,), token, device=DEV)
            leaf = z.detach().requires_grad_()
            assert leaf.stride(0) == 0
            out = ops().token_logprobs(leaf, tokens, temperature=0.8, entropy=entropy)
            by = (torch.full((rows,), 0.75, device=DEV), torch.full((rows,), -1.5, device=DEV))
            dz, = torch.autograd.grad(out, leaf, by if entropy else by[0])
            Rows(z, tokens, 0.8).check_grad(dz, by[0], by[1] if entropy else None)
            others = torch.arange(V, device=DEV) != token
            assert bool((dz[:, others] == dz[:1, others]).all())
    # gradients that differ from position to position, summed over them
    a = torch.randn(rows, device=DEV, generator=gen(35))
    one = z[0].detach().clone().requires_grad_()
    lp = ops().token_logprobs(one.expand(rows, V), tokens, temperature=0.8)
    got, = torch.autograd.grad(lp, one, a)
    p = torch.softmax(one.detach().double() / 0.8, 0)
    want = -a.double().sum() * p / 0.8
    want[V - 1] += a.double().sum() / 0.8
    # each position's value off by 20 u or a half step of its type, their sum in fp32 by as many u as positions, rounded to the type
    size = a.double().abs().sum() * (p + (torch.arange(V, device=DEV) == V - 1)) / 0.8
    step = torch.finfo(dtype).eps / 2
    assert bool(((got.double() - want).abs() <= size * ((20 + 40 + rows) * 2.0 ** -24 + step) + step * want.abs() + 1e-12).all())


# (the form: few rows; by DMA 64 x 64, 64 x 256, 128 x 256, 256 x 256 tiles, rows sorted out by a launch; staged 64 x 64 and 128 x 128
# tiles, rows that are not aligned)
ROUNDED = [(1, 50257, 1024, 0), (9, 50257, 1024, 0), (32, 1003, 512, 0), (64, 1003, 512, 0), (64, 50257, 1024, 0), (90, 50257, 1024, 0),
           (512, 50257, 1024, 0), (1100, 5003, 320, 0), (5, 5003, 77, 0), (700, 5003, 77, 0), (1100, 5003, 203, 0), (20, 1003, 512, 1)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,V,d,shift", ROUNDED)
def test_head_rounds_its_logits(rows, V, d, shift, dtype):
    """Eighths and whole numbers, whose fp32 sums are exact in any order: with round_logits the logits are those sums rounded to bf16,
    no other numbers. Sums of some tens, so that most change by it; fp32 logits do not."""
    say("rounded", rows, V, d, shift, dtype)
    g = gen(36)
    most = int((3 * 1600 / 0.03125 / d) ** 0.5)                  # sums of d products: a standard deviation of 40
    assert most <= 256 and 3 * most * d < 2 ** 21                # whole numbers of bf16, eighths of fp32
    h = torch.randint(-most, most + 1, (rows, d + shift), device=DEV, generator=g).to(dtype)[:, shift:]
    w = (torch.randint(-2, 3, (V, d + shift), device=DEV, generator=g) / 8).to(dtype)[:, shift:]
    tokens = torch.randint(0, V, (rows,), device=DEV, generator=g)
    tokens[3::7] = -100
    tau = 16.0
    rounded = ops().head_logprobs(h, w, tokens, temperature=tau, entropy=True, round_logits=True)
    whole = ops().head_logprobs(h, w, tokens, temperature=tau, entropy=True)
    if dtype == torch.float32:
        assert all(torch.equal(x, y) for x, y in zip(rounded, whole))
    apart = 0
    for r in range(0, rows, 256):
        part, z = slice(r, r + 256), h[r:r + 256].double() @ w.double().t()
        near = z.to(torch.bfloat16).double() if dtype == torch.bfloat16 else z
        found = []
        for got, logits in ((rounded, near), (whole, z)):
            ref = Rows(logits, tokens[part], tau)
            # fp32 logits with exponents rounded once; 200 additions that a term passes through (lanes, tiles, slots)
            rel = U * (4 * ref.near.abs() + 3)
            rel_s = (ref.p * rel).sum(1) + 200 * U
            err_lp = rel_s + U * (ref.lp.abs() + 30)
            lean = ref.lean.abs()
            err_ent = rel_s * (1 + lean) + (ref.p * ref.near.abs() * (rel + 4 * U)).sum(1) + U * (ref.ent + 30) + 200 * U * lean
            for x, want, err in ((got[0], ref.lp, err_lp), (got[1], ref.ent, err_ent)):
                off = (x[part].double() - want).abs() - torch.where(ref.live, err, 0.0)
                assert bool((off <= 0).all()), off.max()
            found.append((ref.lp, err_lp))
        apart += int(((found[0][0] - found[1][0]).abs() > 10 * (found[0][1] + found[1][1])).sum())
    live = int((tokens != -100).sum())
    assert apart > live // 2 if dtype == torch.bfloat16 else apart == 0                         # (the bounds tell the two apart)


def kinds_of(x):
    """-inf, a number, inf or NaN."""
    return torch.where(x.isnan(), 2, torch.where(x.isinf(), x.sign(), 0))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [3, 1003, 50257])
def test_infinite_slopes_as_in_the_formulas(V, dtype):
    """Tokens of probability 0 and ratios past fp32: the losses and gradients that are no numbers are those of the torch formulas."""
    z = (2 * torch.randn(4, 3, V, device=DEV, generator=gen(37))).to(dtype)
    tokens = torch.randint(0, V - 1, (4, 3), device=DEV, generator=gen(38))
    tokens[:, 2] = -100
    tokens[0, 1], z[0, 1, V - 1] = V - 1, -float("inf")
    z[2, 0, V // 2] = -float("inf")                              # (closed, not the token)
    tokens[2, 0] = 0 if V // 2 else 1
    lp = plain.token_logprobs(z.double(), tokens)
    near = torch.where(lp.isfinite(), lp, -5.0).float()
    far = near - 95.0
    signs = torch.tensor([[1.0], [-1.0], [1.0], [-1.0]], device=DEV).expand(4, 3)
    calls = [lambda f, x, kind=kind, red=red, roll=roll: f.preference_loss(x.roll(roll, 0), tokens.roll(roll, 0), loss=kind, reduction=red)
             for kind in ("sigmoid", "hinge", "squared") for red in ("none", "mean") for roll in (0, 2)]
    calls += [lambda f, x, old=old, kl=kl, red=red: f.policy_loss(x, tokens, old, signs, near, kl_weight=kl, reduction=red)
              for old in (near, far) for kl in (0.0, 0.1) for red in ("none", "sequence")]
    for i, call in enumerate(calls):
        found = []
        for f in (ops(), plain):
            leaf = z.clone().requires_grad_()
            loss, values = call(f, leaf)
            found.append([loss.detach(), values, torch.autograd.grad(loss.sum(), leaf)[0]])
        for j, (x, y) in enumerate(zip(*found)):
            say("call", i, "output", j)
            assert torch.equal(kinds_of(x.float()), kinds_of(y.float()))
            ok = kinds_of(y.float()) == 0
            # (that numbers are right is other tests' matter: here to 1e-4 and a step of the type)
            assert torch.allclose(x.float()[ok], y.float()[ok], rtol=1e-4 + torch.finfo(x.dtype).eps, atol=1e-4)
