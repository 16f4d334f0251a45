"""The post-training operators on the GPU against the formulas in 64 bits: log-probabilities of tokens and entropies with their
gradient, the preference loss and the policy loss with theirs.

Bounds. u = 2^-24, half a step of fp32. With d = (z - max) / tau of a logit and p its probability, an exponential is off by
rel_e = (2.5 |d| + 3) u of itself where the logits are bf16 (the product that makes the exponent, the scale, the hardware's exp)
and 6 u where they are fp32; a row's sum of them by sum p rel_e and one u for each of the additions that a term passes through
(8 + 4 in a thread's pieces, one for each round of the workgroup over the row, 6 in a wave, 4 waves, 32 parts). A result's last
rounding is half a step of its type."""

import math

import pytest
import torch

from dispatcher_hybrid import logprobs as plain
from helpers import product_model, tiny

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
TYPES = [torch.bfloat16, torch.float32]
IGNORE = -100


def half(dtype):
    return torch.finfo(dtype).eps / 2


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def ops():
    from dispatcher_hybrid import fused_logprobs
    return fused_logprobs


def say(*what):
    print(*what, flush=True)


class Rows:
    """The rows' values in float64 and how far the kernels' may be from them."""

    def __init__(self, z, tokens, tau):
        V = z.shape[-1]
        self.shape, self.dtype, self.tau = z.shape, z.dtype, tau
        self.tokens = tokens.reshape(-1)
        self.live = self.tokens != IGNORE
        x = torch.where(self.live.unsqueeze(1), z.reshape(-1, V).double(), torch.zeros((), dtype=torch.float64, device=z.device))
        self.d = (x - x.max(1, keepdim=True).values) / tau
        self.p = torch.softmax(x / tau, 1)
        near = self.d.clamp(min=-800)                            # (p is 0 below)
        self.rel = U * (2.5 * near.abs() + 3) if z.dtype == torch.bfloat16 else torch.full_like(near, 6 * U)
        adds = 12 + V // 512 + 1 + 6 + 4 + 32
        self.at = self.tokens.clamp(min=0).long().unsqueeze(1)
        log_p = torch.log_softmax(x / tau, 1)
        self.lp = torch.where(self.live, log_p.gather(1, self.at).squeeze(1), torch.zeros_like(x[:, 0]))
        mean = (self.p * near).sum(1)                             # the kernel's mean exponent
        self.lean, log_s = mean, -(log_p - self.d).nan_to_num(neginf=0.0).min(1).values
        log_s = torch.logsumexp(x / tau, 1) - x.max(1).values / tau
        self.ent = torch.where(self.live, log_s - mean, torch.zeros_like(mean))
        self.rel_s = (self.p * self.rel).sum(1) + adds * U
        self.err_lp = self.rel_s + U * (self.lp.abs() + log_s) + 1e-12
        # a term of the mean is e times its exponent: that one's rounding (2 u) and the product's
        self.err_lean = (self.p * near.abs() * (self.rel + 4 * U)).sum(1) + mean.abs() * (adds * U + self.rel_s + U)
        self.err_ent = self.rel_s + self.err_lean + U * (self.ent + log_s) + 1e-12
        self.near = near

    def check(self, lp=None, ent=None):
        for got, ref, err in ((lp, self.lp, self.err_lp), (ent, self.ent, self.err_ent)):
            if got is not None:
                assert got.dtype == torch.float32 and got.shape == self.shape[:-1]
                off = (got.double().reshape(-1) - ref).abs() - err
                assert bool((off <= 0).all()), off.max()

    def check_grad(self, dz, a, e=None, err_a=None):
        """dz against the gradient of sum a lp + e ent; err_a: how far the kernel's a may be from this one."""
        assert dz.dtype == self.dtype and dz.shape == self.shape
        a = a.double().reshape(-1, 1)
        e = torch.zeros_like(a) if e is None else e.double().reshape(-1, 1)
        err_a = torch.zeros_like(a) if err_a is None else err_a.reshape(-1, 1)
        inner = self.near - self.lean.unsqueeze(1)
        hot = torch.zeros_like(self.p).scatter_(1, self.at, 1.0)
        ref = (a * (hot - self.p) - e * self.p * inner) / self.tau
        rel = self.rel + self.rel_s.unsqueeze(1) + 8 * U
        err = self.p * (a.abs() * rel + e.abs() * (inner.abs() * rel + self.err_lean.unsqueeze(1)
                                                   + 4 * U * (self.near.abs() + self.lean.abs().unsqueeze(1))))
        err = (err + hot * a.abs() * 4 * U + (hot + self.p) * err_a) / self.tau
        err = err + half(self.dtype) * (ref.abs() + err) + 1e-36
        live = self.live.unsqueeze(1)
        off = (dz.double().reshape(ref.shape) - torch.where(live, ref, torch.zeros_like(ref))).abs()
        assert bool((off <= torch.where(live, err, torch.zeros_like(err))).all()), (off - err).max()


def inputs(lead, V, dtype, seed, ignored=0.2, banned=0.0, scale=2.0):
    g = gen(seed)
    tokens = torch.randint(0, V, lead, device=DEV, generator=g)
    z = torch.randn(*lead, V, device=DEV, generator=g) * scale
    if banned:
        z.masked_fill_(torch.rand(z.shape, device=DEV, generator=g) < banned, -math.inf)
    z.scatter_(-1, tokens.unsqueeze(-1), 3.0 + 4.0 * torch.rand(*lead, 1, device=DEV, generator=g))
    tokens = torch.where(torch.rand(lead, device=DEV, generator=g) < ignored, IGNORE, tokens)
    return z.to(dtype), tokens


SHAPES = [((1,), 1), ((1,), 7), ((1,), 50257), ((3, 5), 257), ((2, 9), 50257), ((70,), 5003), ((2, 1031), 1003), ((1100,), 4097),
          ((1, 2, 3), 8191), ((515,), 16400), ((1500,), 37), ((2, 3), 80001), ((130,), 140001)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lead,V", SHAPES)
def test_logprobs_and_gradient(lead, V, dtype):
    for i, (tau, entropy, banned) in enumerate([(1.0, False, 0.0), (0.7, True, 0.3), (2.5, True, 0.0)]):
        say("logprobs", lead, V, dtype, tau)
        z, tokens = inputs(lead, V, dtype, 10 + i, banned=banned)
        if i == 1:
            tokens = tokens.int()
        ref = Rows(z, tokens, tau)
        leaf = z.clone().requires_grad_()
        out = ops().token_logprobs(leaf, tokens, temperature=tau, entropy=entropy)
        lp, ent = out if entropy else (out, None)
        ref.check(lp, ent)
        a, e = torch.randn(lead, device=DEV, generator=gen(3)), torch.randn(lead, device=DEV, generator=gen(4))
        if entropy:
            ref.check_grad(torch.autograd.grad((lp, ent), leaf, (a, e), retain_graph=True)[0], a, e)
            ref.check_grad(torch.autograd.grad(ent, leaf, e, retain_graph=True)[0], torch.zeros_like(a), e)
        ref.check_grad(torch.autograd.grad(lp, leaf, a)[0], a)
        with torch.no_grad():
            again = ops().token_logprobs(leaf, tokens, temperature=tau, entropy=entropy)
        for x, y in zip(again if entropy else (again,), (lp, ent)):
            assert torch.equal(x, y) and not x.requires_grad


@pytest.mark.parametrize("dtype", TYPES)
def test_layouts(dtype):
    V = 1003
    z, tokens = inputs((4, 6), V, dtype, 5)
    ref = ops().token_logprobs(z, tokens, entropy=True)
    wide = torch.randn(4, 9, V + 5, device=DEV, generator=gen(1)).to(dtype)
    wide[:, 2:8, 3:3 + V] = z
    views = [wide[:, 2:8, 3:3 + V], z.transpose(0, 1).contiguous().transpose(0, 1), z.transpose(1, 2).contiguous().transpose(1, 2),
             z.view(2, 2, 6, V), z[None].expand(1, 4, 6, V), z.flip(0).flip(0)]
    for view in views:
        say("layout", view.shape, view.stride())
        leaf = view.detach().requires_grad_()
        tok = tokens.reshape(view.shape[:-1])
        got = ops().token_logprobs(leaf, tok, entropy=True)
        # (a row's pieces begin at its first 16-byte boundary: elsewhere other sums)
        Rows(z, tokens, 1.0).check(got[0].reshape(4, 6), got[1].reshape(4, 6))
        g = torch.randn(4, 6, device=DEV, generator=gen(2))
        Rows(z, tokens, 1.0).check_grad(torch.autograd.grad(got[0], leaf, g.reshape(tok.shape))[0].reshape(z.shape), g)
    for rows in (z[0, 0].expand(5, V), z[:1, :1].expand(3, 4, V)):             # one row many times
        got = ops().token_logprobs(rows, tokens[0, 1].expand(rows.shape[:-1]))
        assert bool((got == got.flatten()[0]).all()) and bool(got.isfinite().all())
    assert torch.equal(ref[0], ops().token_logprobs(z, tokens.t().contiguous().t()))
    one = ops().token_logprobs(z[0, 0], tokens[0, 1])
    assert one.shape == () and one.isfinite()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,V", [(3, 50257), (700, 50257), (1200, 1003), (300, 1003), (12, 80001), (12, 50257)])
def test_awkward_rows(rows, V, dtype):
    """Rows of -inf, the lowest value, one +inf, one NaN, one value; tokens outside the vocabulary and closed ones; ignored rows
    that hold NaN."""
    lowest = torch.finfo(dtype).min
    z, tokens = inputs((rows,), V, dtype, 6, ignored=0.0)
    kinds = ["plain", "-inf", "lowest", "+inf", "nan", "equal", "past", "below", "closed", "ignored"][:max(3, min(rows, 10))]
    first = rows - len(kinds)
    for i, k in enumerate(kinds):
        r = first + i
        if k == "-inf":
            z[r] = -math.inf
        elif k == "lowest":
            z[r] = lowest
        elif k == "+inf":
            z[r, V // 2] = math.inf
        elif k == "nan":
            z[r, V // 3] = math.nan
        elif k == "equal":
            z[r] = -7.5
        elif k == "past":
            tokens[r] = V
        elif k == "below":
            tokens[r] = -1
        elif k == "closed":
            z[r, tokens[r]] = -math.inf
        elif k == "ignored":
            z[r], tokens[r] = math.nan, IGNORE
    leaf = z.clone().requires_grad_()
    lp, ent = ops().token_logprobs(leaf, tokens, entropy=True)
    a, e = torch.ones(rows, device=DEV), torch.full((rows,), 0.5, device=DEV)
    dz, = torch.autograd.grad((lp, ent), leaf, (a, e), retain_graph=True)
    d1, = torch.autograd.grad(lp, leaf, a)
    for i, k in enumerate(kinds):
        r = first + i
        say("row", k)
        nan_row = k in ("-inf", "+inf", "nan", "past", "below")
        for x in (lp[r], ent[r]):
            assert bool(x.isnan()) == (nan_row), (k, x)
        assert bool(dz[r].isnan().all()) == nan_row and bool(dz[r].isnan().any()) == nan_row, k
        assert bool(d1[r].isnan().all()) == nan_row and bool(d1[r].isnan().any()) == nan_row, k
        if k in ("lowest", "equal"):
            assert abs(lp[r].item() + math.log(V)) < 1e-5 and abs(ent[r].item() - math.log(V)) < 1e-5
        if k == "closed":
            assert lp[r] == -math.inf and ent[r].isfinite() and d1[r, tokens[r]] == 1 and bool(d1[r].isfinite().all())
        if k == "ignored":
            assert lp[r] == 0 and ent[r] == 0 and not bool(dz[r].any()) and not bool(d1[r].any())
    ok = list(range(first + 1))
    Rows(z[ok], tokens[ok], 1.0).check(lp[ok], ent[ok])
    # no gradient wanted of a row: not read, but NaN where its probabilities are
    zero, = torch.autograd.grad(ops().token_logprobs(leaf, tokens), leaf, torch.zeros(rows, device=DEV))
    for i, k in enumerate(kinds):
        assert bool(zero[first + i].isnan().all()) == (k in ("-inf", "+inf", "nan", "past", "below")), k
    assert not bool(zero[:first + 1].any())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tau", [2.0 ** -126, 1e-3, 300.0, 2.0 ** 126])
def test_extreme_temperatures(tau, dtype):
    z, tokens = inputs((5,), 3001, dtype, 8, ignored=0.0)
    tokens[0] = z[0].argmax()
    z[0, :] = torch.where(torch.arange(3001, device=DEV) == tokens[0], z[0], z[0] - 4)        # one largest logit
    lp, ent = ops().token_logprobs(z, tokens, temperature=tau, entropy=True)
    if tau < 1e-30:
        assert lp[0] == 0 and ent[0] == 0 and bool((lp[1:] <= 0).all())
    elif tau > 1e30:
        assert bool(((lp + math.log(3001)).abs() < 1e-5).all()) and bool(((ent - math.log(3001)).abs() < 1e-5).all())
    else:
        Rows(z, tokens, tau).check(lp, ent)


def test_gradient_against_differences():
    z, tokens = inputs((4,), 61, torch.float32, 9, ignored=0.0)
    a, e = torch.tensor([1.0, -2.0, 0.5, 3.0], device=DEV), torch.tensor([0.3, 1.0, -1.0, 0.2], device=DEV)
    leaf = z.clone().requires_grad_()
    lp, ent = ops().token_logprobs(leaf, tokens, 1.3, entropy=True)
    dz, = torch.autograd.grad((lp, ent), leaf, (a, e))

    def f(x):
        lp, ent = plain.token_logprobs(x, tokens, 1.3, entropy=True)
        return (a.double() * lp + e.double() * ent).sum()
    step, x = 1e-5, z.double()
    for v in range(61):
        up, down = x.clone(), x.clone()
        for r in range(4):                 # rows do not meet: one of them at a time
            up, down = x.clone(), x.clone()
            up[r, v] += step
            down[r, v] -= step
            num = (f(up) - f(down)) / (2 * step)
            assert abs(num.item() - dz[r, v].item()) < 2e-6
        if v == 12:
            break


# ---- from the hidden states ---------------------------------------------------------------------------------------------

def head_inputs(lead, V, d, dtype, seed, ignored=0.3):
    g = gen(seed)
    tokens = torch.randint(0, V, lead, device=DEV, generator=g)
    w = torch.randn(V, d, device=DEV, generator=g) * (2.0 / math.sqrt(d))
    h = torch.randn(*lead, d, device=DEV, generator=g) + w[tokens]
    if len(lead):
        tokens = torch.where(torch.rand(lead, device=DEV, generator=g) < ignored, IGNORE, tokens)
    return h.to(dtype), w.to(dtype), tokens


def check_head(got, h, w, tokens, tau, round_logits=False, exact=False):
    """Against the logits in 64 bits. A logit is a sum of d products: off by at most (d + 2) u of the sum of their magnitudes (and
    where it is rounded, by half a step of bf16, or a whole one if that error crosses a rounding border)."""
    V, d = w.shape
    rows = h.reshape(-1, d)
    lp, ent = got if isinstance(got, tuple) else (got, None)
    for r in range(0, rows.shape[0], 256):
        x = rows[r:r + 256].double()
        z, size = x @ w.double().t(), x.abs() @ w.double().abs().t()
        off = (d + 2) * U * size * (0 if exact else 1)
        if round_logits:
            z = z.to(torch.bfloat16).double()
            off = off + 2.0 ** -7 * (z.abs() + off)
        tok = tokens.reshape(-1)[r:r + 256]
        ref = Rows(z, tok, tau)
        ref.rel = U * (4 * ref.near.abs() + 3)                   # (fp32 logits, exponents rounded as bf16 ones' are)
        ref.rel_s = (ref.p * ref.rel).sum(1) + 200 * U           # 128 columns a tile and lane, tiles, lanes, slots
        mean_off = (ref.p * off).sum(1) / tau
        if round_logits:                                         # few logits cross a border, here bounded by all of them
            own = off.gather(1, ref.at).squeeze(1) / tau
        else:
            own = off.gather(1, ref.at).squeeze(1) / tau
        # with every logit off by at most off: log of the sum by mean_off e^most, the mean exponent by off (1 + |d| + mean |d|)
        most = (off / tau).max(1).values.exp()
        err = (ref.rel_s + mean_off + own) * most + U * (ref.lp.abs() + 30) + 1e-12
        bad = (lp.reshape(-1)[r:r + 256].double() - ref.lp).abs() - torch.where(ref.live, err, 0.0)
        assert bool((bad <= 0).all()), bad.max()
        if ent is not None:
            spread = (ref.p * (off / tau) * (1 + ref.near.abs() + ref.lean.abs().unsqueeze(1))).sum(1) * 2 * most
            err = ref.rel_s * (1 + ref.lean.abs()) + spread + (ref.p * ref.near.abs() * (ref.rel + 4 * U)).sum(1) \
                + U * (ref.ent + 30) + 200 * U * ref.lean.abs()
            bad = (ent.reshape(-1)[r:r + 256].double() - ref.ent).abs() - torch.where(ref.live, err, 0.0)
            assert bool((bad <= 0).all()), bad.max()


HEADS = [((), 7, 3), ((1,), 50257, 1024), ((16,), 50257, 1024), ((3, 7), 1003, 64), ((50,), 130, 200), ((64,), 5003, 320),
         ((65,), 5003, 128), ((2, 100), 257, 1), ((300,), 4097, 72), ((700,), 777, 512), ((2, 400), 2049, 1024), ((1030,), 130, 2048),
         ((4500,), 300, 64), ((130,), 50257, 256)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lead,V,d", HEADS)
def test_head_logprobs(lead, V, d, dtype):
    for i, (tau, entropy, rounded) in enumerate([(1.0, False, False), (0.7, True, False), (2.0, True, True)]):
        say("head", lead, V, d, dtype, tau)
        h, w, tokens = head_inputs(lead, V, d, dtype, 60 + i)
        if i == 1:
            tokens = tokens.int()
        got = ops().head_logprobs(h, w, tokens, temperature=tau, entropy=entropy, round_logits=rounded)
        check_head(got, h, w, tokens, tau, rounded and dtype == torch.bfloat16)
        first = got[0] if entropy else got
        assert first.shape == lead and first.dtype == torch.float32
        again = ops().head_logprobs(h, w, tokens, temperature=tau, entropy=entropy, round_logits=rounded)
        assert torch.equal(first, again[0] if entropy else again)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,V,d", [(9, 50257, 1024), (64, 1003, 2048), (90, 5003, 1024), (700, 2049, 320), (700, 2049, 77), (2600, 514, 64)])
def test_head_of_exact_products(rows, V, d, dtype):
    """Eighths and whole numbers: every sum of products is a number of fp32, whatever its order."""
    g = gen(75)
    h = torch.randint(-3, 4, (rows, d), device=DEV, generator=g).to(dtype)
    w = (torch.randint(-2, 3, (V, d), device=DEV, generator=g) / 8).to(dtype)
    tokens = torch.randint(0, V, (rows,), device=DEV, generator=g)
    tokens[::7] = IGNORE
    for tau in (1.0, 2.0):
        check_head(ops().head_logprobs(h, w, tokens, temperature=tau, entropy=True), h, w, tokens, tau, exact=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lead", [(2, 9), (3, 100)])
def test_head_layouts(lead, dtype):
    V, d = 1003, 128
    h, w, tokens = head_inputs(lead, V, d, dtype, 70)
    wide_h, wide_w = torch.randn(*lead, d + 3, device=DEV).to(dtype), torch.randn(V, d + 5, device=DEV).to(dtype)
    wide_h[..., 1:d + 1], wide_w[:, 2:d + 2] = h, w
    for x, y in ((wide_h[..., 1:d + 1], wide_w[:, 2:d + 2]), (h.transpose(0, 1).contiguous().transpose(0, 1), w.t().contiguous().t()),
                 (h.flip(0).flip(0), w), (h, wide_w[:, 2:d + 2])):
        say("head layout", x.stride(), y.stride())
        check_head(ops().head_logprobs(x, y, tokens, entropy=True), h, w, tokens, 1.0)
    one = ops().head_logprobs(h[:1, :1].expand(*lead, d), w, tokens.flatten()[:1].clamp(min=0).expand(lead), entropy=True)
    for x in one:
        assert bool((x == x.flatten()[0]).all())
    none = ops().head_logprobs(h[:0], w, tokens[:0], entropy=True)
    assert none[0].shape == none[1].shape == (0, lead[1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,d", [(20, 128), (400, 128), (400, 100)])
def test_head_of_awkward_rows(rows, d, dtype):
    V = 2100
    h, w, tokens = head_inputs((rows,), V, d, dtype, 71, ignored=0.0)
    h[3], tokens[3] = math.nan, IGNORE
    h[5] = math.nan
    h[6, 0] = math.inf
    tokens[7], tokens[8] = V, -5
    h[9] = 0
    lp, ent = ops().head_logprobs(h, w, tokens, entropy=True)
    assert lp[3] == 0 and ent[3] == 0
    for r in (5, 6, 7, 8):
        assert lp[r].isnan() and ent[r].isnan(), r
    assert abs(lp[9].item() + math.log(V)) < 1e-5 and abs(ent[9].item() - math.log(V)) < 1e-5
    ok = torch.ones(rows, dtype=torch.bool, device=DEV)
    ok[[5, 6, 7, 8]] = False
    check_head((lp[ok], ent[ok]), h[ok].nan_to_num(), w, tokens[ok], 1.0)
    none = torch.full_like(tokens, IGNORE)                       # no row at all
    lp, ent = ops().head_logprobs(h, w, none, entropy=True)
    assert not bool(lp.any()) and not bool(ent.any())
    w[V // 2] = math.inf                                         # a weight without value: no row has one
    h[3] = 1.0
    assert bool(ops().head_logprobs(h, w, tokens).isnan()[[5, 6, 9]].all())


def test_head_agrees_with_stored_logits():
    h, w, tokens = head_inputs((2, 300), 5003, 256, torch.bfloat16, 72)
    z = torch.nn.functional.linear(h, w)
    stored = ops().token_logprobs(z, tokens)
    rounded = ops().head_logprobs(h, w, tokens, round_logits=True)
    # equal but where a rounding of a logit falls the other way (the library sums in another order): at most a step of the largest
    assert (stored - rounded).abs().max() <= 2.0 ** -7 * z.abs().max()
    assert ((stored - rounded).abs() < 1e-4).double().mean() > 0.9


# ---- preference loss --------------------------------------------------------------------------------------------------

def preference_ref(rows, n, T, reference, beta, kind, average, margin, eps):
    """(pair losses, sums, slopes of the sequences, how far off each of the three may be)."""
    live = rows.live.view(2 * n, T)
    count = live.sum(1).clamp(min=1).double() if average else torch.ones(2 * n, dtype=torch.float64, device=DEV)
    sums = rows.lp.view(2 * n, T).sum(1) / count
    err = torch.where(live, rows.err_lp.view(2 * n, T), 0.0).sum(1) / count
    gain = sums if reference is None else sums - reference.double()
    D = (gain[:n] - gain[n:]).requires_grad_()
    x = beta * D - margin
    ls = torch.nn.functional.logsigmoid
    loss = {"sigmoid": lambda: -(1 - eps) * ls(x) - eps * ls(-x), "hinge": lambda: torch.relu(1 - x),
            "squared": lambda: (D - 1 / (2 * beta)) ** 2}[kind]()
    slope, = torch.autograd.grad(loss.sum(), D)
    err_D = err[:n] + err[n:]
    bend = {"sigmoid": beta ** 2 / 4, "hinge": 0.0, "squared": 2.0}[kind]
    err_loss = slope.abs() * err_D + bend * err_D ** 2 + 4 * U * loss.detach() + 1e-12
    err_slope = (bend * err_D + 2 * U * slope.abs()).repeat(2) / count
    return loss.detach(), sums, torch.cat([slope, -slope]) / count, err_loss, err + U * sums.abs() + 1e-12, err_slope


KINDS = [("sigmoid", 0.1, False, 0.0, 0.0, True), ("sigmoid", 0.5, False, 0.3, 0.2, True), ("sigmoid", 2.0, True, 0.5, 0.0, False),
         ("hinge", 0.05, False, 0.0, 0.0, True), ("squared", 0.2, True, 0.0, 0.0, True), ("hinge", 1.0, True, -0.5, 0.0, False)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,T,V", [(1, 1, 50257), (1, 24, 50257), (3, 37, 1003), (70, 9, 257), (2, 300, 5003), (5, 700, 130), (2, 5, 80001), (3, 24, 60007)])
def test_preference_loss(n, T, V, dtype):
    for i, (kind, beta, average, margin, eps, with_ref) in enumerate(KINDS):
        say("preference", n, T, V, dtype, kind)
        z, tokens = inputs((2 * n, T), V, dtype, 20 + i)
        if T > 1:
            tokens[n] = IGNORE                                 # a sequence without a token
        rows = Rows(z, tokens, 1.0)
        sums = rows.lp.view(2 * n, T).sum(1)
        if average:
            sums = sums / rows.live.view(2 * n, T).sum(1).clamp(min=1)
        reference = (sums + torch.randn(2 * n, device=DEV, generator=gen(7)) * 3) if with_ref else None
        if reference is not None and i % 2:
            reference = reference.float()
        loss, s, slope, err, err_s, err_slope = preference_ref(rows, n, T, reference, beta, kind, average, margin, eps)
        args = dict(beta=beta, loss=kind, average=average, margin=margin, label_smoothing=eps)
        leaf = z.clone().requires_grad_()
        got, got_s = ops().preference_loss(leaf, tokens, reference, reduction="none", **args)
        assert got.shape == (n,) and got_s.shape == (2 * n,) and not got_s.requires_grad
        assert bool(((got_s.double() - s).abs() <= err_s).all())
        assert bool(((got.double() - loss).abs() <= err).all())
        g = torch.randn(n, device=DEV, generator=gen(8))
        up = g.double().repeat(2)
        wide = lambda t: t.unsqueeze(1).expand(2 * n, T)
        rows.check_grad(torch.autograd.grad(got, leaf, g)[0], wide(up * slope), err_a=wide(up.abs() * err_slope + 4 * U * (up * slope).abs()))
        for reduction, share in (("mean", 1.0 / n), ("sum", 1.0)):
            got, _ = ops().preference_loss(leaf, tokens, reference, reduction=reduction, **args)
            assert abs(got.item() - loss.sum().item() * share) <= (err.sum().item() + U * loss.sum().item() * 2) * share
            dz, = torch.autograd.grad(got, leaf)
            rows.check_grad(dz, wide(slope * share), err_a=wide((err_slope + 4 * U * slope.abs()) * share))


def test_preference_of_nothing_and_of_broken_rows():
    f = ops().preference_loss
    z = torch.randn(0, 5, 11, device=DEV, requires_grad=True)
    tok = torch.zeros(0, 5, dtype=torch.long, device=DEV)
    loss, sums = f(z, tok)
    assert math.isnan(loss.item()) and sums.shape == (0,) and torch.autograd.grad(loss, z)[0].shape == z.shape
    assert f(z, tok, reduction="sum")[0] == 0 and f(z, tok, reduction="none")[0].shape == (0,)
    z = torch.randn(4, 0, 11, device=DEV, requires_grad=True)
    ref = torch.tensor([1.0, 2.0, 3.0, 5.0], device=DEV)
    loss, sums = f(z, torch.zeros(4, 0, dtype=torch.long, device=DEV), ref, reduction="none")
    want = torch.nn.functional.softplus(0.1 * torch.tensor([-2.0, -3.0], device=DEV))
    assert not sums.any() and (loss - want).abs().max() < 1e-6 and torch.autograd.grad(loss.sum(), z)[0].shape == z.shape
    z, tok = inputs((6, 5), 97, torch.float32, 30, ignored=0.0)
    tok[4, 2], tok[1, 3] = 97, IGNORE                          # a token past the vocabulary in the second pair
    z[1, 3] = math.nan
    leaf = z.clone().requires_grad_()
    loss, sums = f(leaf, tok, reduction="none")
    dz, = torch.autograd.grad(loss, leaf, torch.ones(3, device=DEV))
    assert loss.isnan().tolist() == [False, True, False] and sums.isnan().tolist() == [False] * 4 + [True, False]
    assert not bool(dz[1, 3].any()) and dz[1, 2].isnan().all() and dz[4].isnan().all() and dz[[0, 2, 3, 5]].isfinite().all()
    # behind the hinge: no gradient, and none of a row's logits is read for it
    leaf = z.clone().requires_grad_()
    tok[4, 2] = 5
    far = torch.tensor([0.0] * 3 + [1e4] * 3, device=DEV)
    loss, _ = f(leaf, tok, far, loss="hinge")
    assert loss == 0 and not bool(torch.autograd.grad(loss, leaf)[0].any())


# ---- policy loss --------------------------------------------------------------------------------------------------------

def policy_inputs(lead, V, dtype, seed, tau, clip, clip_high, by_sequence):
    z, tokens = inputs(lead, V, dtype, seed)
    rows = Rows(z, tokens, tau)
    g = gen(seed + 100)
    move = 0.25 * torch.randn(lead, device=DEV, generator=g, dtype=torch.float64)
    for edge in (math.log1p(-clip), math.log1p(clip_high)):   # no ratio so near to the clip that its rounding decides
        move = torch.where((move - edge).abs() < 1e-2, edge + 2e-2, move)
    old = (rows.lp.view(lead) - move).float()
    ref = (rows.lp.view(lead) + 0.3 * torch.randn(lead, device=DEV, generator=g, dtype=torch.float64)).float()
    adv = torch.randn(lead[:-1] if by_sequence else lead, device=DEV, generator=g)
    return z, tokens, rows, old, ref, adv


def policy_ref(rows, lead, old, adv, ref, clip, clip_high, kl, w):
    """(terms, slopes in lp, how far off each may be), all (rows)."""
    A = (adv.unsqueeze(-1).expand(lead) if adv.dim() < len(lead) else adv).double().reshape(-1)
    lp = rows.lp.clone().requires_grad_()
    ratio = torch.exp(lp - old.double().reshape(-1))
    terms = -torch.min(ratio * A, ratio.clamp(1 - clip, 1 + clip_high) * A)
    err = (ratio * A).abs().detach()
    if kl:
        d = ref.double().reshape(-1) - lp
        terms = terms + kl * (torch.expm1(d) - d)
    slope, = torch.autograd.grad(terms.sum(), lp)
    err_slope = err * (rows.err_lp + 2 * U)
    if kl:
        err_slope = err_slope + kl * d.detach().exp() * (rows.err_lp + 2 * U)
    size = terms.detach().abs()
    terms = terms.detach() - w * rows.ent
    err_terms = slope.abs() * rows.err_lp + abs(w) * rows.err_ent + err * rows.err_lp ** 2 + 2 * U * (terms.abs() + size) + 1e-12
    dead = ~rows.live
    return [t.masked_fill(dead, 0.0) for t in (terms, slope, err_terms, err_slope + 2 * U * slope.abs())]


POLICY = [(1.0, 0.2, 0.2, 0.0, 0.0, False), (0.8, 0.2, 0.3, 0.1, 0.01, True), (1.0, 0.1, 0.4, 0.0, 0.05, False),
          (1.5, 1.0, 0.5, 0.2, 0.0, True)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lead,V", [((1, 1), 50257), ((4, 12), 50257), ((3, 37), 1003), ((7,), 257), ((2, 3, 90), 511), ((300, 5), 131),
                                    ((2, 700), 2049), ((2, 5), 80001), ((1, 64), 60007), ((5, 14), 60007)])
def test_policy_loss(lead, V, dtype):
    for i, (tau, clip, high, kl, w, by_sequence) in enumerate(POLICY):
        say("policy", lead, V, dtype, tau)
        z, tokens, rows, old, ref, adv = policy_inputs(lead, V, dtype, 40 + i, tau, min(clip, 0.999), high, by_sequence)
        if len(lead) > 1 and lead[0] > 2:
            tokens[1] = IGNORE                                 # a sequence without a token
            rows = Rows(z, tokens, tau)
        terms, slope, err, err_slope = policy_ref(rows, lead, old, adv, ref, clip, high, kl, w)
        args = dict(reference_logprobs=ref if kl else None, clip=clip, clip_high=high, kl_weight=kl, entropy_weight=w, temperature=tau)
        leaf = z.clone().requires_grad_()
        got, lp = ops().policy_loss(leaf, tokens, old, adv, reduction="none", **args)
        rows.check(lp)
        assert got.shape == lead and not lp.requires_grad
        assert bool(((got.double().reshape(-1) - terms).abs() <= err).all())
        ent = torch.full_like(slope, -w) if w else None
        g = torch.randn(lead, device=DEV, generator=gen(8))
        up = g.double().reshape(-1)
        rows.check_grad(torch.autograd.grad(got, leaf, g)[0], up * slope, up * ent if w else None, up.abs() * (err_slope + 4 * U * slope.abs()))
        live = rows.live.view(-1, lead[-1])
        count = live.sum(1).clamp(min=1)
        for reduction in ("mean", "sum", "sequence"):
            if reduction != "sum" and not bool(live.any()):
                got, _ = ops().policy_loss(leaf, tokens, old, adv, reduction=reduction, **args)
                assert math.isnan(got.item()) and not bool(torch.autograd.grad(got, leaf)[0].any())
                continue
            if reduction == "sequence":
                share = (1.0 / count.double() / (live.any(1).sum())).unsqueeze(1).expand(live.shape).reshape(-1)
            else:
                share = torch.full_like(terms, 1.0 / live.sum().item() if reduction == "mean" else 1.0)
            got, again = ops().policy_loss(leaf, tokens, old, adv, reduction=reduction, **args)
            want = (terms * share).sum()
            assert torch.equal(again, lp)
            assert abs(got.item() - want.item()) <= (err * share).sum().item() + U * abs(want.item())
            dz, = torch.autograd.grad(got, leaf)
            rows.check_grad(dz, slope * share, share * ent if w else None, share * (err_slope + 6 * U * slope.abs()))


def test_policy_of_nothing_and_of_broken_rows():
    f = ops().policy_loss
    zeros = lambda *s: torch.zeros(*s, device=DEV)
    for shape in ((0, 5), (3, 0), (0,)):
        z = torch.randn(*shape, 11, device=DEV, requires_grad=True)
        tok = torch.zeros(shape, dtype=torch.long, device=DEV)
        for reduction in plain.TOKEN_REDUCTIONS:
            loss, lp = f(z, tok, zeros(shape), zeros(shape), reduction=reduction, entropy_weight=0.1)
            assert lp.shape == shape and (loss.shape == shape if reduction == "none" else loss.shape == ())
            if reduction != "none":
                assert loss == 0 if reduction == "sum" else math.isnan(loss.item())
                assert torch.autograd.grad(loss, z)[0].shape == z.shape
    z, tok = inputs((3, 6), 97, torch.bfloat16, 50, ignored=0.0)
    tok[0], tok[1, 2], tok[2, 4] = IGNORE, 97, IGNORE
    z[2, 4] = math.nan
    old, adv = torch.full((3, 6), -4.0, device=DEV), torch.ones(3, 6, device=DEV)
    for t in (old, adv):
        t[2, 4] = math.nan                                     # nothing of an ignored position is looked at
    leaf = z.clone().requires_grad_()
    rows, lp = f(leaf, tok, old, adv, reduction="none")
    assert rows.isnan().nonzero().tolist() == [[1, 2]] and not bool(rows[0].any()) and rows[2, 4] == 0
    dz, = torch.autograd.grad(rows, leaf, torch.ones_like(rows))
    assert dz[1, 2].isnan().all() and not bool(dz[0].any()) and not bool(dz[2, 4].any())
    assert dz[1, [0, 1, 3, 4, 5]].isfinite().all()
    tok[1, 2] = 3
    loss, _ = f(z, tok, old, adv, reduction="sequence")
    a, b = f(z[1:2], tok[1:2], old[1:2], adv[1:2])[0], f(z[2:], tok[2:], old[2:], adv[2:])[0]
    assert abs(loss.item() - (a + b).item() / 2) < 1e-6        # the sequence without positions is none
    # a ratio past every number: clipped for a gain, as the formula for a loss
    far = torch.full((3, 6), -1e4, device=DEV)
    leaf = z.clone().requires_grad_()
    rows, _ = f(leaf, tok, far, adv, reduction="none")
    assert bool((rows[1] == -torch.tensor(1.2, device=DEV)).all())
    assert not bool(torch.autograd.grad(rows[1].sum(), leaf)[0].any())
    assert bool((f(z, tok, far, -adv, reduction="none")[0][1] == math.inf).all())


def test_ratio_of_one_and_of_the_clip_itself():
    """old = the log-probabilities themselves: a ratio within one rounding of 1, the gradient the plain policy gradient's."""
    z, tok = inputs((2, 33), 1003, torch.float32, 51)
    old = ops().token_logprobs(z, tok)
    adv = torch.randn(2, 33, device=DEV, generator=gen(3))
    leaf = z.clone().requires_grad_()
    rows, lp = ops().policy_loss(leaf, tok, old, adv, clip=0.0, reduction="none")
    live = tok != IGNORE
    assert torch.equal(lp, old)
    assert bool(((rows + adv).abs()[live] <= 4e-6 * adv.abs()[live]).all()) and not bool(rows[~live].any())
    rows, _ = ops().policy_loss(leaf, tok, old, adv, reduction="none")
    got, = torch.autograd.grad(rows.sum(), leaf)
    want, = torch.autograd.grad((ops().token_logprobs(leaf, tok) * -adv).sum(), leaf)
    assert (got - want).abs().max() <= 4e-6 * want.abs().max()


@pytest.mark.parametrize("rows", [1024, 1025, 33000, 70001])
def test_head_of_many_rows(rows):
    """Rows sorted out by several workgroups, one and more a thread: the values of the same rows alone."""
    h, w, tokens = head_inputs((rows,), 257, 64, torch.bfloat16, 76, ignored=0.5)
    lp, ent = ops().head_logprobs(h, w, tokens, entropy=True)
    live = tokens != IGNORE
    check_head((lp, ent), h, w, tokens, 1.0)
    a, b = ops().head_logprobs(h[live], w, tokens[live], entropy=True)
    assert (a - lp[live]).abs().max() < 1e-5 and (b - ent[live]).abs().max() < 1e-5
    assert not bool(lp[~live].any()) and not bool(ent[~live].any())
