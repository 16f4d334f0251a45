"""The vocabulary-end operators on the GPU against plain torch in 64 bits: embedding rows and their gradient, a teacher's top
logits, the distillation loss and its gradient, and a training step of all of them together.

Bounds. u = 2^-24, half a step of fp32; half a step of the output's type is eps / 2. A sum of n fp32 numbers in any order is
off by at most n u times the sum of their magnitudes."""

import math

import pytest
import torch

from dispatcher_hybrid import distillation as plain
from helpers import product_model, tiny

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
TYPES = [torch.bfloat16, torch.float32]


def half(dtype):
    return torch.finfo(dtype).eps / 2


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def ops():
    from dispatcher_hybrid import fused_vocab
    return fused_vocab


def say(*what):
    print(*what, flush=True)


# ---- embedding ------------------------------------------------------------------------------------------------------

def grad_ref(dy, ids, V, scale, skip=None):
    """(gradient, bound without the final rounding) in float64."""
    d = dy.shape[-1]
    x, i = dy.reshape(-1, d).double(), ids.reshape(-1).long()
    ok = (i >= 0) & (i < V)
    if skip is not None:
        ok &= i != skip
    x, i = x[ok], i[ok]
    z = lambda: torch.zeros(V, d, dtype=torch.float64, device=x.device)
    ref = z().index_add_(0, i, x) * scale
    mag = z().index_add_(0, i, x.abs()) * abs(scale)
    n = torch.bincount(i, minlength=V).double().unsqueeze(1)
    return ref, (n + 2) * U * mag


def check_grad(got, dy, ids, V, scale, skip=None):
    ref, bound = grad_ref(dy, ids, V, scale, skip)
    bound = bound + half(got.dtype) * (ref.abs() + bound) + 1e-38
    assert bool(((got.double() - ref).abs() <= bound).all())


def tokens_of(kind, n, V, g):
    if kind == "one":
        return torch.full((n,), V // 2, device=DEV)
    if kind == "text":                                         # a few tokens often, most hardly ever
        u = torch.rand(n, device=DEV, dtype=torch.float64, generator=g)
        return (3.0 * ((V + 3.0) / 3.0) ** u - 3.0).long().clamp_(0, V - 1)
    if kind == "padded":
        t = torch.randint(0, V, (n,), device=DEV, generator=g)
        t[n // 3:] = V - 1
        return t
    return torch.randint(0, V, (n,), device=DEV, generator=g)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,V,d,kind", [
    (1, 1, 1, "any"), (1, 50257, 1024, "any"), (63, 7, 8, "any"), (64, 300, 64, "text"), (65, 256, 33, "padded"),
    (1025, 257, 128, "one"), (4097, 50257, 1024, "text"), (9001, 1000, 100, "padded"), (40000, 5, 24, "any"),
    (33000, 70001, 72, "text"), (3000, 50257, 1030, "one"), (2048, 140000, 16, "any"), (3001, 512, 2048, "text"),
    (3000, 120001, 40, "text"), (511, 120001, 40, "text"), (512, 50257, 1024, "one"), (400, 50257, 1024, "padded"), (4096, 300, 128, "text"),
])
def test_embedding_and_gradient(n, V, d, kind, dtype):
    say("embed", n, V, d, kind, dtype)
    g = gen(n + V + d)
    ids = tokens_of(kind, n, V, g)
    W = torch.randn(V, d, device=DEV, generator=g).to(dtype).requires_grad_()
    dy = torch.randn(n, d, device=DEV, generator=g).to(dtype)
    for scale, bits in ((1.0, torch.int64), (math.sqrt(d), torch.int32)):
        y = ops().embed_tokens(ids.to(bits), W, scale)
        assert torch.equal(y, (W.detach()[ids].float() * torch.tensor(scale, device=DEV)).to(dtype))
        dW, = torch.autograd.grad(y, W, dy)
        check_grad(dW, dy, ids, V, scale)
        again, = torch.autograd.grad(ops().embed_tokens(ids.to(bits), W, scale), W, dy)
        assert torch.equal(dW, again)                          # the same bits on every call


@pytest.mark.parametrize("dtype", TYPES)
def test_embedding_layouts_padding_and_strays(dtype):
    g = gen(5)
    V, d = 90, 40
    W = torch.randn(V, d + 3, device=DEV, generator=g).to(dtype)[:, 1:d + 1]      # rows off every 16-byte boundary
    ids = torch.randint(0, V, (6, 50), device=DEV, generator=g)
    ids[2, 7], ids[3, 3] = -1, V
    part = ids.t()[::2]                                                           # strided tokens
    w = W.detach().requires_grad_()
    y = ops().embed_tokens(part, w, 0.5, padding_idx=4 - V)
    ok = (part >= 0) & (part < V)
    assert torch.equal(y[ok], (W[part[ok]].float() * 0.5).to(dtype)) and bool(y[~ok].isnan().all())
    for dy in (torch.randn(25, 6, 2 * d, device=DEV, generator=g).to(dtype)[..., ::2],
               torch.randn(d, device=DEV, generator=g).to(dtype).expand(25, 6, d),
               torch.randn(25, 6, d + 1, device=DEV, generator=g).to(dtype)[..., 1:]):
        dW, = torch.autograd.grad(y, w, dy, retain_graph=True)
        check_grad(dW, dy, part, V, 0.5, skip=4)
        assert bool((dW[4] == 0).all())
    # nothing to look up
    none = torch.zeros(0, 3, dtype=torch.long, device=DEV)
    y = ops().embed_tokens(none, w)
    dW, = torch.autograd.grad(y, w, torch.zeros_like(y))
    assert y.shape == (0, 3, d) and bool((dW == 0).all())
    # a broadcast table
    row = torch.randn(1, d, device=DEV, generator=g).to(dtype).expand(V, d)
    assert torch.equal(ops().embed_tokens(part[ok], row), row[:1].expand(int(ok.sum()), d))


def test_embedding_gradient_of_the_gradient():
    g = gen(6)
    ids = torch.randint(0, 9, (2, 5), device=DEV, generator=g)
    W = torch.randn(9, 6, device=DEV, generator=g).requires_grad_()
    dy = torch.randn(2, 5, 6, device=DEV, generator=g).requires_grad_()
    dW, = torch.autograd.grad(ops().embed_tokens(ids, W, 2.0, padding_idx=3), W, dy, create_graph=True)
    v = torch.randn(9, 6, device=DEV, generator=g)
    got, = torch.autograd.grad(dW, dy, v)
    assert torch.equal(got, (v * 2.0)[ids] * (ids != 3).unsqueeze(-1))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [1, 5, 16])
def test_a_vocabulary_of_one(d, dtype):
    g = gen(9)
    ids = torch.zeros(3, 7, dtype=torch.long, device=DEV)
    for W in (torch.randn(d, device=DEV, generator=g).to(dtype).expand(1, d),     # a row stride of 0
              torch.randn(d, 1, device=DEV, generator=g).to(dtype).t(),
              torch.randn(1, d, device=DEV, generator=g).to(dtype)):
        w = W.detach().requires_grad_()
        y = ops().embed_tokens(ids, w)
        assert torch.equal(y, W.expand(3, 7, d))
        dy = torch.randn(d, device=DEV, generator=g).to(dtype).expand(1, d)
        dW, = torch.autograd.grad(ops().embed_tokens(ids[0, :1], w), w, dy)       # one row, of stride 0 too
        assert torch.equal(dW, dy)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(2, 5), (7, 150), (40, 1001)])                 # one launch, three, four rows a lane
@pytest.mark.parametrize("wide", [False, True])
def test_tokens_outside_the_vocabulary(wide, shape, dtype):
    g = gen(7)
    V, d = 90, 2048 if shape[0] == 40 else 40
    ids = torch.randint(0, V, shape, device=DEV, generator=g)
    strays = [-1, V, -7, -2 ** 31, 2 ** 31 - 1] + ([2 ** 40 + 3, 2 ** 32, -2 ** 32 + 5] if wide else [])
    flat = ids.view(-1)
    for i, s in enumerate(strays[:flat.numel() - 1]):
        flat[(i * 37 + 1) % flat.numel()] = s
    ids = ids if wide else ids.int()
    ok = (ids >= 0) & (ids < V)
    assert int((~ok).sum()) >= min(len(strays), 5)
    for skip in (None, 3):
        W = torch.randn(V, d, device=DEV, generator=g).to(dtype).requires_grad_()
        dy = torch.randn(*shape, d, device=DEV, generator=g).to(dtype).requires_grad_()
        y = ops().embed_tokens(ids, W, 1.0, skip)
        assert torch.equal(y[ok], W[ids[ok].long()]) and bool(y[~ok].isnan().all())
        dW, = torch.autograd.grad(y, W, dy, create_graph=True)
        check_grad(dW.detach(), dy.detach(), ids, V, 1.0, skip)
        v = torch.randn(V, d, device=DEV, generator=g).to(dtype)
        again, = torch.autograd.grad(dW, dy, v)
        used = ok if skip is None else ok & (ids != skip)
        assert torch.equal(again[used], v[ids[used].long()]) and bool((again[~used] == 0).all())
        x = dy.detach().requires_grad_()                                          # the registered forms
        two = torch.ops.dispatcher.embed_tokens_grad(x, ids, V, 1.0, -1 if skip is None else skip)
        assert torch.equal(two, dW) and torch.equal(torch.autograd.grad(two, x, v)[0], again)


# ---- top logits -----------------------------------------------------------------------------------------------------

def check_top(x, k):
    values, tokens = ops().top_logits(x, k)
    # (NaN of one sign: the GPU's sort puts one whose sign bit is set below every number, the CPU's above)
    ref, at = torch.sort(torch.where(x.isnan(), math.nan, x.double()), dim=-1, descending=True, stable=True)
    assert torch.equal(tokens, at[..., :k])
    picked = x.gather(-1, tokens)
    assert values.dtype == x.dtype and bool(((values == picked) | (values.isnan() & picked.isnan())).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,V,k", [
    (1, 1, 1), (1, 50257, 64), (2, 50257, 256), (3, 257, 256), (5, 256, 256), (7, 1000, 1), (2, 130001, 100), (33, 50257, 20),
    (300, 4099, 17), (600, 515, 65), (1100, 2051, 128), (2100, 700, 3), (4500, 1031, 64), (1, 70, 70),
])
def test_top_logits(rows, V, k, dtype):
    say("top", rows, V, k, dtype)
    x = (torch.randn(rows, V, device=DEV, generator=gen(rows + V)) * 3).to(dtype)
    check_top(x, k)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 70, 4200])
@pytest.mark.parametrize("what", ["equal", "rising", "falling", "ends", "two", "inf", "nan", "zeros", "steps"])
def test_top_logits_of_awkward_rows(what, rows, dtype):
    say("top", what, rows, dtype)
    V, g = 5003 if rows < 100 else 1501, gen(rows)
    i = torch.arange(V, device=DEV, dtype=torch.float32)
    x = {"equal": lambda: torch.full((rows, V), -2.5, device=DEV),
         "rising": lambda: (i * 0.5 - 100).expand(rows, V).clone(),
         "falling": lambda: (100 - i * 0.5).expand(rows, V).clone(),
         "ends": lambda: torch.where((i < 40) | (i >= V - 40), 7.0, -1.0).expand(rows, V).clone(),
         "two": lambda: torch.randint(0, 2, (rows, V), device=DEV, generator=g).float(),
         "inf": lambda: torch.where(torch.rand(rows, V, device=DEV, generator=g) < 0.99, -math.inf, 1.0),
         "nan": lambda: torch.where(torch.rand(rows, V, device=DEV, generator=g) < 0.02, math.nan,
                                    torch.randn(rows, V, device=DEV, generator=g)),
         "zeros": lambda: torch.where(torch.rand(rows, V, device=DEV, generator=g) < 0.5, 0.0, -0.0),
         "steps": lambda: (i // 64).expand(rows, V).clone()}[what]().to(dtype)
    if what == "inf":
        x[0] = torch.finfo(dtype).min
        x[-1, 3] = math.inf
    for k in (1, 50, 256):
        check_top(x, k)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("V", [50257, 65536, 70001])
@pytest.mark.parametrize("what", ["few", "masked", "columns", "rising", "equal"])
def test_top_logits_of_long_awkward_rows(what, V, rows, dtype):
    """A peaked row among -inf, a masked vocabulary, large values that only every 1024th 16-byte piece holds, a rising row."""
    say("top long", what, V, rows, dtype)
    g, i, per = gen(V + rows), torch.arange(V, device=DEV), 8 if dtype == torch.bfloat16 else 4
    noise = torch.randn(rows, V, device=DEV, generator=g)
    x = {"few": lambda: torch.where(i % 9001 == 17, noise, -math.inf), "masked": lambda: torch.where(i < 40000, -math.inf, noise),
         "columns": lambda: torch.where((i // per) % 1024 < 90, noise * 0.1 + 50, noise),
         "rising": lambda: (i * 0.01 - 100).expand(rows, V).clone(),
         "equal": lambda: torch.full((rows, V), -math.inf, device=DEV)}[what]().to(dtype)
    for k in (1, 64, 256):
        check_top(x, k)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,V", [(120, 50257), (600, 50257), (600, 1501), (90, 40)])
def test_top_logits_of_rows_with_one_nan(rows, V, dtype):
    """One NaN a row, of either sign, in every stretch of the row and at both ends; a row in eight without."""
    x = torch.randn(rows, V + 3, device=DEV, generator=gen(rows + V)).to(dtype)[:, 3:]      # rows of every alignment
    at = torch.arange(rows, device=DEV) * 7919 % V
    at[:6] = torch.tensor([0, 1, 7, V - 1, V - 2, V - 8], device=DEV)
    bits = torch.tensor([0x7fc00000, -0x400000], dtype=torch.int32, device=DEV).view(torch.float32).to(dtype)
    i = torch.arange(rows, device=DEV)
    has = i % 8 != 7
    x[i[has], at[has]] = bits[i[has] % 2]
    assert int(x.isnan().sum()) == int(has.sum())
    for k in (1, 33):
        check_top(x, k)
    for a, b in zip(plain.top_logits(x, 9), ops().top_logits(x, 9)):              # the formula sorts them as the kernel does
        assert torch.equal(a.nan_to_num(123.0), b.nan_to_num(123.0)) if a.is_floating_point() else torch.equal(a, b)


@pytest.mark.parametrize("dtype", TYPES)
def test_top_logits_layouts(dtype):
    g = gen(8)
    base = torch.randn(4, 6, 999, device=DEV, generator=g).to(dtype)
    for x in (base, base[:, 1:], base[..., 1:], base[..., 5:700], base.transpose(0, 1), base[..., ::2], base[0, 0],
              base[0, 0].expand(3, 999), base[:0], base.transpose(1, 2)[:, :, :3]):
        check_top(x, min(3, x.shape[-1]))
    leaf = base.float().requires_grad_()
    assert not ops().top_logits(leaf, 2)[0].requires_grad


# ---- distillation loss ----------------------------------------------------------------------------------------------

def bounds(z, t, tok, labels, tau, w, count, dtype):
    """(rows, gradient of the mean, bounds of both), float64. Each exp has a relative error of at most (4 + 3 |x|) u for the
    exponent x (two roundings of x, one of the scale, one unit of exp2), a sum of V of them at most 260 + V / 256 roundings
    more (rescaled thread sums of V / 256 terms, joined over lanes, waves and parts)."""
    V = z.shape[-1]
    zz = z.double().requires_grad_()
    rows = plain.distillation_loss(zz, t.double(), tok, labels, tau, w, reduction="none")
    grad, = torch.autograd.grad(rows.sum() / count, zz)
    zd = zz.detach()
    span = lambda s: ((zd - zd.amax(-1, keepdim=True)) / s).clamp_min(-104.0)      # (smaller terms are 0 in fp32)

    def soft(s):
        x = span(s)
        e = x.exp()
        p = e / e.sum(-1, keepdim=True)
        rel = ((4 + 3 * x.abs()) * p).sum(-1) * U + (260 + V / 256) * U            # of the sum
        return p, rel, (4 + 3 * x.abs()) * U + rel.unsqueeze(-1) + 4 * U           # of each probability
    q, rel_q, each_q = soft(tau)
    P, rel_P, each_P = soft(1.0)
    live = (tok >= 0) & (t != -math.inf)
    td = torch.where(live, t.double() / tau, torch.full((), -1e30, dtype=torch.float64, device=z.device))
    tx = (td - td.amax(-1, keepdim=True)).clamp_min(-104.0)
    p = torch.softmax(td, -1) * live
    rel_p = ((4 + 3 * tx.abs()) * U) + ((4 + 3 * tx.abs()) * p).sum(-1, keepdim=True) * U + 260 * U
    log_q = torch.log_softmax(zd / tau, -1).gather(-1, tok.clamp(0, V - 1).long())
    log_p = torch.log_softmax(td, -1)
    gap = torch.where(live & (p > 0), (log_p - log_q).abs(), torch.zeros_like(p))
    row_bound = w * tau ** 2 * ((p * gap * rel_p).sum(-1) + rel_q + rel_p.amax(-1)) + (1 - w) * rel_P + 2 * U * rows.abs()
    named = torch.zeros_like(q).scatter_add_(-1, tok.clamp(0, V - 1).long(), p * (rel_p + 300 * U))
    has = live.any(-1, keepdim=True)
    grad_bound = (w * tau * (q * each_q * has + named) + (1 - w) * P * each_P + 4 * U * (w * tau + (1 - w)) * (named > 0)) / count
    if labels is not None:
        hit = torch.zeros_like(q).scatter_(-1, labels.clamp(0, V - 1).long().unsqueeze(-1), 1.0)
        grad_bound = grad_bound + 4 * U * (w * tau + 1 - w) * hit / count
        kept = (labels != -100)
        row_bound, grad_bound = row_bound * kept, grad_bound * kept.unsqueeze(-1)
    grad_bound = grad_bound + 4 * U * grad.abs()
    grad_bound = grad_bound + half(dtype) * (grad.abs() + grad_bound) + 1e-38
    return rows.detach(), grad, row_bound + 1e-38, grad_bound


def inputs(lead, V, k, dtype, seed, empties=False, repeats=False):
    g = gen(seed)
    z = (torch.randn(*lead, V, device=DEV, generator=g) * 2.5).to(dtype)
    t = (torch.randn(*lead, k, device=DEV, generator=g) * 3).to(dtype)
    tok = torch.randint(0, V, (*lead, k), device=DEV, generator=g)                # the same token twice, now and then
    if repeats:
        tok[..., k // 2:] = tok[..., :1]
    labels = torch.randint(0, V, lead, device=DEV, generator=g)
    labels[torch.rand(lead, device=DEV, generator=g) < 0.2] = -100
    labels.view(-1)[0] = 0
    tok[..., 0] = torch.where(torch.rand(lead, device=DEV, generator=g) < 0.5, labels.clamp(min=0), tok[..., 0])
    if empties:
        tok[torch.rand(*lead, k, device=DEV, generator=g) < 0.4] = -1
        t[torch.rand(*lead, k, device=DEV, generator=g) < 0.1] = -math.inf
        tok.view(-1, k)[0] = -1
    return z, t, tok, labels


def check_distill(z, t, tok, labels, tau, w, **kw):
    count = z[..., 0].numel() if labels is None else int((labels != -100).sum())
    rows, grad, row_bound, grad_bound = bounds(z, t, tok, labels, tau, w, count, z.dtype)
    leaf = z.detach().requires_grad_()
    loss = ops().distillation_loss(leaf, t, tok, labels, tau, w, **kw)
    got, = torch.autograd.grad(loss, leaf)
    assert loss.dtype == torch.float32 and loss.shape == () and got.dtype == z.dtype
    assert abs(loss.item() - rows.sum().item() / count) <= row_bound.sum().item() / count + 2 * U * abs(loss.item())
    worst = ((got.double() - grad).abs() / grad_bound).max().item()
    assert worst <= 1.0, worst
    with torch.no_grad():
        each = ops().distillation_loss(z, t, tok, labels, tau, w, reduction="none")
    assert bool(((each.double() - rows).abs() <= row_bound).all())
    # row factors of their own, and the sum
    f = torch.rand(rows.shape, device=DEV, generator=gen(1)) + 0.5
    each = ops().distillation_loss(leaf, t, tok, labels, tau, w, reduction="none")
    got, = torch.autograd.grad(each, leaf, f)
    scaled = grad * count * f.double().unsqueeze(-1)
    assert bool(((got.double() - scaled).abs() <= (grad_bound * count * f.unsqueeze(-1)) + 4 * U * scaled.abs() + 1e-38).all())
    total = ops().distillation_loss(leaf, t, tok, labels, tau, w, reduction="sum")
    assert abs(total.item() - rows.sum().item()) <= row_bound.sum().item() + 2 * U * abs(total.item())


MODES = [(1.0, 1.0, False), (2.0, 0.5, True), (0.7, 1.0, False), (3.0, 0.0, True), (1.0, 0.25, True), (4.0, 1.0, True), (4.0, 0.3, True),
         (1.3, 0.6, True)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lead,V,k", [((1,), 1, 1), ((1,), 50257, 64), ((3, 5), 257, 7), ((2, 9), 50257, 16), ((70,), 5003, 256),
                                      ((600,), 1001, 20), ((2, 513), 2050, 33), ((4,), 130001, 5)])
def test_distillation(lead, V, k, dtype):
    for i, (tau, w, with_labels) in enumerate(MODES):
        say("distill", lead, V, k, dtype, tau, w, with_labels)
        z, t, tok, labels = inputs(lead, V, k, dtype, 7 * i + V, empties=i % 2 == 1, repeats=i == 4)
        check_distill(z, t, tok, labels if with_labels else None, tau, w)


@pytest.mark.parametrize("dtype", TYPES)
def test_distillation_layouts_and_types(dtype):
    z, t, tok, labels = inputs((4, 6), 999, 5, dtype, 3)
    wide = torch.randn(4, 7, 1003, device=DEV, generator=gen(4)).to(dtype)
    for x in (z, wide[:, :6, :999], wide[:, 1:, 1:1000], wide[:, 1:, 4:1003], wide.transpose(0, 1)[:6].transpose(0, 1)[..., 2:1001],
              wide[..., :999].transpose(1, 2).contiguous().transpose(1, 2)[:, :6], z[:1].expand(4, 6, 999)):
        say("distill layout", x.stride(), x.storage_offset())
        check_distill(x, t, tok, labels, 2.0, 0.5)
    other = torch.float32 if dtype == torch.bfloat16 else torch.bfloat16
    check_distill(z, t.to(other), tok.int(), labels.int(), 2.0, 0.5)
    check_distill(z, t.transpose(0, 1).contiguous().transpose(0, 1), tok.transpose(0, 1).contiguous().transpose(0, 1),
                  labels.t().contiguous().t(), 2.0, 0.5)
    check_distill(z.view(2, 2, 6, 999), t.view(2, 2, 6, 5), tok.view(2, 2, 6, 5), labels.view(2, 2, 6), 2.0, 0.5)
    check_distill(z[0, 0], t[0, 0], tok[0, 0], None, 2.0, 1.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [3, 700])
def test_distillation_of_masked_and_broken_rows(rows, dtype):
    V, k = 4003, 6
    z, t, tok, labels = inputs((rows,), V, k, dtype, 9)
    labels[labels == -100] = 5
    low = torch.finfo(dtype).min
    z[0, 100:] = -math.inf                                     # a masked vocabulary
    z[1, 10:] = low                                            # masked by the type's lowest value
    z[2] = low                                                 # nothing left: a uniform row
    tok[0], tok[1], tok[2] = torch.arange(6), torch.arange(6), torch.arange(6)
    labels[:3] = 3
    for tau in (2.0, 0.5):
        check_distill(z, t, tok, labels, tau, 0.5)
    t[0] = low                                                 # a uniform teacher
    check_distill(z, t, tok, labels, 2.0, 0.5)
    # ignored rows may hold anything, empty slots too
    labels[0], z[0] = -100, math.nan
    tok[1, 2], t[1, 2] = -1, math.nan
    leaf = z.detach().requires_grad_()
    loss = ops().distillation_loss(leaf, t, tok, labels, 2.0, 0.5)
    grad, = torch.autograd.grad(loss, leaf)
    assert math.isfinite(loss.item()) and bool((grad[0] == 0).all()) and bool(grad.isfinite().all())
    # a label or teacher token outside the vocabulary, NaN and +inf logits, NaN of the teacher: that row alone
    for change in ("label", "negative", "token", "nan", "inf", "teacher", "all"):
        zz, tt, kk, ll = z.clone(), t.clone(), tok.clone(), labels.clone()
        zz[0], ll[0] = 0.0, 1
        if change == "label":
            ll[2] = V
        if change == "negative":
            ll[2] = -7
        if change == "token":
            kk[2, 5] = V
        if change == "nan":
            zz[2, V - 1] = math.nan
        if change == "inf":
            zz[2, 77] = math.inf
        if change == "teacher":
            tt[2, 3] = math.nan
        if change == "all":
            zz[2] = -math.inf
        leaf = zz.requires_grad_()
        each = ops().distillation_loss(leaf, tt, kk, ll, 2.0, 0.5, reduction="none")
        grad, = torch.autograd.grad(each.sum(), leaf)
        bad = torch.arange(rows, device=DEV) == 2
        assert torch.equal(each.isnan(), bad), change
        assert not bool(grad[~bad].isnan().any()) and bool(grad[2].isnan().any()), change
    # the teacher's NaN of above in a slot that is live again
    z[1], tok[1], labels[1] = 1.0, 4, 0
    z[1, 4] = -math.inf
    leaf = z.detach().requires_grad_()
    each = ops().distillation_loss(leaf, t, tok, labels, 2.0, 0.5, reduction="none")
    grad, = torch.autograd.grad(each.sum(), leaf)
    assert each[1].isnan() and bool(grad[1, tok[1, 0]].isnan())
    # empty rows beside unusable logits do not matter to the soft term; every row ignored; no rows
    z[1] = math.nan
    tok[1] = -1
    leaf = z.detach().requires_grad_()
    each = ops().distillation_loss(leaf, t, tok, None, 2.0, reduction="none")
    grad, = torch.autograd.grad(each[1], leaf)
    assert each[1] == 0 and bool((grad[1] == 0).all())
    none = ops().distillation_loss(leaf, t, tok, torch.full_like(labels, -100), 2.0, 0.5)
    grad, = torch.autograd.grad(none, leaf)
    assert math.isnan(none.item()) and bool((grad == 0).all())
    empty = ops().distillation_loss(leaf[:0], t[:0], tok[:0], labels[:0], 2.0, 0.5)
    assert math.isnan(empty.item()) and torch.autograd.grad(empty, leaf)[0].abs().nan_to_num().sum() == 0
    assert ops().distillation_loss(leaf[:0], t[:0], tok[:0], reduction="none").shape == (0,)
    assert ops().distillation_loss(leaf[:0], t[:0], tok[:0], reduction="sum").item() == 0.0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [2, 600])
def test_a_masked_vocabulary_under_the_teachers_token(rows, dtype):
    z, t, tok, _ = inputs((rows,), 2003, 6, dtype, 10)
    z[1, tok[1, 0]] = -math.inf
    leaf = z.requires_grad_()
    each = ops().distillation_loss(leaf, t, tok, temperature=2.0, reduction="none")
    grad, = torch.autograd.grad(each.sum(), leaf)
    assert each[1].item() == math.inf and bool(grad.isfinite().all()) and each.isfinite().sum() == rows - 1
    # a teacher whose logit there is -inf as well names nothing
    t[1, tok[1] == tok[1, 0]] = -math.inf
    each = ops().distillation_loss(leaf, t, tok, temperature=2.0, reduction="none")
    assert bool(each.isfinite().all())


def test_distillation_gradient_against_differences():
    z, t, tok, labels = inputs((3,), 40, 6, torch.float32, 12)
    labels[1] = 7
    leaf = z.clone().requires_grad_()
    grad, = torch.autograd.grad(ops().distillation_loss(leaf, t, tok, labels, 1.5, 0.6), leaf)
    h = 2.0 ** -6
    for v in (int(tok[1, 0]), 7, int(tok[1, 3]), 20):
        up, down = z.clone(), z.clone()
        up[1, v] += h
        down[1, v] -= h
        f = lambda x: ops().distillation_loss(x, t, tok, labels, 1.5, 0.6).item()
        # h^2 / 6 times a third derivative below 1, and the losses' own error (under 64 u of a value below 8) over h
        assert abs((f(up) - f(down)) / (2 * h) - grad[1, v].item()) <= h * h / 6 + 64 * U * 8 / h


def test_distillation_gradient_of_the_gradient_and_in_place_use():
    z, t, tok, labels = inputs((3,), 30, 5, torch.float32, 13)
    for fn in (ops().distillation_loss, plain.distillation_loss):
        leaf = z.clone().requires_grad_()
        g, = torch.autograd.grad(fn(leaf, t, tok, labels, 2.0, 0.5), leaf, create_graph=True)
        gg, = torch.autograd.grad(g.square().sum(), leaf)
        if fn is plain.distillation_loss:
            assert torch.allclose(gg, first, rtol=1e-5, atol=1e-8)                # the same torch operations
        first = gg
    leaf = z.clone().requires_grad_()
    loss = ops().distillation_loss(leaf, t, tok, labels, 2.0, 0.5)
    one, = torch.autograd.grad(loss, leaf, retain_graph=True)
    loss /= 4
    quarter, = torch.autograd.grad(loss, leaf)
    assert torch.equal(quarter, one / 4)


# ---- together -------------------------------------------------------------------------------------------------------

def test_registered_operations_agree_with_the_direct_launches():
    z, t, tok, labels = inputs((2, 9), 501, 5, torch.float32, 14)
    W, ids = torch.randn(50, 16, device=DEV, generator=gen(2)), torch.randint(0, 50, (3, 7), device=DEV, generator=gen(3))
    o = torch.ops.dispatcher
    for red in (0, 1, 2):
        a, b = z.clone().requires_grad_(), z.clone().requires_grad_()
        x = ops().distillation_loss(a, t, tok, labels, 2.0, 0.5, reduction=plain.REDUCTIONS[red])
        y = o.distillation_loss(b, t, tok, labels, 2.0, 0.5, -100, red)[0]
        x.sum().backward()
        y.sum().backward()
        assert torch.equal(x, y) and torch.equal(a.grad, b.grad)
    for x, y in zip(ops().top_logits(z, 5), o.top_logits(z, 5)):
        assert torch.equal(x, y)
    a, b = W.clone().requires_grad_(), W.clone().requires_grad_()
    x, y = ops().embed_tokens(ids, a, 3.0, padding_idx=7), o.embed_tokens(b, ids, 3.0, -1, 7)
    x.square().sum().backward()
    y.square().sum().backward()
    assert torch.equal(x, y) and torch.equal(a.grad, b.grad)
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode() as fake:
        f = lambda q: fake.from_tensor(q)
        assert ops().top_logits(f(z), 5)[1].shape == (2, 9, 5)
        assert ops().distillation_loss(f(z), f(t), f(tok), f(labels), 2.0, 0.5).shape == ()
        assert ops().embed_tokens(f(ids), f(W)).shape == (3, 7, 16)


def test_another_stream_and_two_calls_at_once():
    z, t, tok, labels = inputs((5, 33), 5003, 9, torch.bfloat16, 15)
    W, ids = torch.randn(999, 64, device=DEV, generator=gen(2)), torch.randint(0, 999, (700,), device=DEV, generator=gen(3))
    dy = torch.randn(700, 64, device=DEV, generator=gen(4))

    def step(z, W):
        z, W = z.detach().requires_grad_(), W.detach().requires_grad_()
        loss = ops().distillation_loss(z, t, tok, labels, 2.0, 0.5)
        return [*ops().top_logits(z, 9), loss.detach(), *torch.autograd.grad(loss, z),
                *torch.autograd.grad(ops().embed_tokens(ids, W), W, dy)]
    ref, other = step(z, W), step(z.flip(0), W * 2)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    args = [(z, W), (z.flip(0), W * 2)]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for s, a in zip(streams, args):
            with torch.cuda.stream(s):
                got.append(step(*a))
        torch.cuda.synchronize()
        for x, y in ((got[0], ref), (got[1], other)):
            assert all(torch.equal(p, q) for p, q in zip(x, y))


def test_two_captured_steps_replayed_in_turn():
    """A student's vocabulary end as a user runs it: the teacher's targets, embedding, head, loss, both gradients; captured
    twice with inputs of their own and replayed in turn, each replay against the eager result."""
    V, d, B, T, k = 3001, 64, 2, 40, 8
    g = gen(16)
    W = (torch.randn(V, d, device=DEV, generator=g) * 0.3).to(torch.bfloat16)
    data = [dict(ids=torch.randint(0, V, (B, T), device=DEV, generator=g), teacher=torch.randn(B, T, V, device=DEV, generator=g) * 3)
            for _ in range(2)]

    def step(s):
        values, tokens = ops().top_logits(s["teacher"], k)
        w = W.detach().requires_grad_()
        x = ops().embed_tokens(s["ids"], w, 8.0, padding_idx=0)
        labels = torch.roll(s["ids"], -1, 1)
        loss = ops().distillation_loss(x.view(-1, d).mm(w.t()).view(B, T, V), values, tokens, labels, 2.0, 0.5)
        return [values, tokens, x.detach(), loss.detach(), *torch.autograd.grad(loss, w)]
    graphs = []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in data:
            step(s)
    torch.cuda.current_stream().wait_stream(side)
    for s in data:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(s)
        graphs.append((graph, out))
    for turn in range(3):
        for s in data:
            s["ids"].copy_(torch.randint(0, V, (B, T), device=DEV, generator=g))
            s["teacher"].normal_(generator=g)
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for s, (_, out) in zip(data, graphs):
            for a, b in zip(out, step(s)):
                assert torch.equal(a, b), turn


def test_under_a_compiler_and_a_transform():
    z, t, tok, labels = inputs((2, 9), 501, 5, torch.float32, 21)
    W, ids = torch.randn(50, 16, device=DEV, generator=gen(2)), torch.randint(0, 50, (3, 7), device=DEV, generator=gen(3))

    def step(z, W):
        values, tokens = ops().top_logits(z * 2, 5)
        return ops().distillation_loss(z, values, tokens, labels, 2.0, 0.5) + ops().embed_tokens(ids, W, 2.0).square().sum()
    grads = []
    for fn in (step, torch.compile(step, backend="aot_eager", fullgraph=True)):
        a, b = z.clone().requires_grad_(), W.clone().requires_grad_()
        loss = fn(a, b)
        grads.append([loss.detach(), *torch.autograd.grad(loss, (a, b))])
    for x, y in zip(*grads):
        assert torch.equal(x, y)
    # a registered operation has no rule for torch.func's transforms: refused, as the other training operations are
    with pytest.raises(RuntimeError, match="functorch"):
        torch.func.grad(step, argnums=(0, 1))(z, W)


def test_saved_tensors_that_hooks_move():
    z, t, tok, labels = inputs((2, 9), 501, 5, torch.bfloat16, 22)
    W, ids = torch.randn(50, 16, device=DEV, generator=gen(2)), torch.randint(0, 50, (3, 7), device=DEV, generator=gen(3))

    def step():
        a, b = z.clone().requires_grad_(), W.clone().requires_grad_()
        loss = ops().distillation_loss(a, t, tok, labels, 2.0, 0.5) + ops().embed_tokens(ids, b).sum()
        return torch.autograd.grad(loss, (a, b))

    def strided(x):                                            # the same values at odd addresses and strides
        wide = torch.empty(x.numel() * 2 + 1, dtype=x.dtype, device=x.device)[1:].view(*x.shape, 2)[..., 0] if x.dim() else x
        return wide.copy_(x) if x.dim() else x
    ref = step()
    with torch.autograd.graph.save_on_cpu():
        on_cpu = step()
    with torch.autograd.graph.saved_tensors_hooks(lambda x: x, strided):
        moved = step()
    for other in (on_cpu, moved):
        assert all(torch.equal(x, y) for x, y in zip(ref, other))


def test_captured_gradient_of_a_wide_vocabulary():
    """The one-launch gradient with more than 64 KB of LDS, in a graph."""
    V, n, d = 120001, 500, 40
    ids, dy = torch.randint(0, V, (n,), device=DEV, generator=gen(2)), torch.randn(n, d, device=DEV, generator=gen(3))
    from dispatcher_hybrid import fused_vocab
    f = lambda: fused_vocab._lookup_grad(dy, ids, V, 1.0, -1)
    f()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = f()
    for seed in range(3):
        ids.copy_(torch.randint(0, V, (n,), device=DEV, generator=gen(seed)))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, f())


def test_two_host_threads():
    import threading
    z, t, tok, labels = inputs((40,), 5003, 9, torch.bfloat16, 23)

    def step(z):
        leaf = z.detach().requires_grad_()
        loss = ops().distillation_loss(leaf, t, tok, labels, 2.0, 0.5)
        return [*ops().top_logits(z, 9), loss.detach(), torch.autograd.grad(loss, leaf)[0]]
    data = [z, z.flip(0)]
    ref = [step(x) for x in data]
    got = [None, None]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5):
                got[i] = step(data[i])
            torch.cuda.current_stream().synchronize()
    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join(60)
    for x, y in zip(got, ref):
        assert all(torch.equal(p, q) for p, q in zip(x, y))


def test_refusals_on_the_gpu():
    W, ids = torch.randn(6, 4, device=DEV), torch.zeros(3, dtype=torch.long, device=DEV)
    tok = torch.zeros(6, 2, dtype=torch.long, device=DEV)
    for call in (lambda: ops().embed_tokens(ids, W.half()), lambda: ops().top_logits(W.half(), 2),
                 lambda: ops().distillation_loss(W.half(), W[:, :2], tok), lambda: ops().distillation_loss(W, W[:, :2].half(), tok)):
        with pytest.raises(TypeError, match="float32 and bfloat16"):
            call()
    for call in (lambda: ops().embed_tokens(ids.cpu(), W), lambda: ops().distillation_loss(W, W[:, :2], tok.cpu()),
                 lambda: ops().distillation_loss(W, W[:, :2].cpu(), tok),
                 lambda: ops().distillation_loss(W, W[:, :2], tok, labels=torch.zeros(6).long(), weight=0.5)):
        with pytest.raises(RuntimeError, match="one device"):
            call()


def test_launches_refuse_sizes_that_do_not_fit():
    """The registered operations by name, and tensors that a hook hands back smaller: nothing is launched."""
    o, n = torch.ops.dispatcher, fused_native()
    W, ids = torch.randn(6, 4, device=DEV), torch.zeros(3, dtype=torch.long, device=DEV)
    z, t, tok, labels = inputs((4,), 50, 3, torch.float32, 31)
    out, kept = o.distillation_loss(z, t, tok, labels, 2.0, 0.5, -100, 1)
    assert kept.numel() == 4 * 4 + 4
    for exc, call in (
            (TypeError, lambda: o.embed_tokens(W, ids.byte(), 1.0, -1, -1)),
            (TypeError, lambda: o.embed_tokens_grad(W[:3], ids.short(), 6, 1.0, -1)),
            (ValueError, lambda: o.embed_tokens_grad(W[:2], ids, 6, 1.0, -1)),
            (ValueError, lambda: o.embed_tokens_grad(W[:3], ids, 0, 1.0, -1)),
            (ValueError, lambda: o.embed_tokens(W, ids, 1.0, 7, -1)),
            (ValueError, lambda: n.lookup(W[0], ids, 1.0, -1)),
            (TypeError, lambda: o.distillation_loss(z, t, tok.byte(), labels, 2.0, 0.5, -100, 1)),
            (ValueError, lambda: o.distillation_loss(z, t, tok[:3], labels, 2.0, 0.5, -100, 1)),
            (ValueError, lambda: o.distillation_loss(z, t[:, :2], tok, labels, 2.0, 0.5, -100, 1)),
            (ValueError, lambda: o.distillation_loss(z, t, tok, labels[:3], 2.0, 0.5, -100, 1)),
            (ValueError, lambda: o.distillation_loss(z, t, tok, None, 2.0, 0.5, -100, 1)),
            (ValueError, lambda: o.distillation_loss_grad(out, z, t, tok, labels, kept[:19], 2.0, 0.5, -100, 1)),
            (ValueError, lambda: o.distillation_loss_grad(z[:3, 0], z, t, tok, labels, kept, 2.0, 0.5, -100, 0)),
            (ValueError, lambda: o.top_logits(z, 51))):
        with pytest.raises(exc):
            call()
    leaf, w = z.clone().requires_grad_(), W.clone().requires_grad_()
    with torch.autograd.graph.saved_tensors_hooks(lambda x: x, lambda x: x[:2]):
        loss, rows = ops().distillation_loss(leaf, t, tok, labels, 2.0, 0.5), ops().embed_tokens(ids, w)
        with pytest.raises((ValueError, RuntimeError)):
            torch.autograd.grad(loss, leaf)
        with pytest.raises((ValueError, RuntimeError), match="elements"):
            torch.autograd.grad(rows.sum(), w)
    torch.cuda.synchronize()


def fused_native():
    return ops()._native


# ---- the model ------------------------------------------------------------------------------------------------------

def test_model_step_against_torch():
    """A student's training step with the operators against the same step without them (fp32: the same layers, so the
    difference is the fp32 error of loss and embedding alone)."""
    cfgd, sd = tiny("tiny_a")
    teacher = product_model(cfgd, tiny("tiny_a", seed=77)[1], device=DEV)
    ids = torch.randint(0, 255, (2, 40), device=DEV, generator=gen(1))
    labels = ids.clone()
    labels[1, 30:] = -100
    plain_targets = teacher.teacher_targets(ids, 12)
    targets = teacher.enable_fused_vocab().teacher_targets(ids, 12)
    for a, b in zip(targets, plain_targets):
        assert torch.equal(a, b)
    results = []
    for fused in (False, True):
        m = product_model(cfgd, sd, device=DEV).train().enable_fused_vocab(fused)
        out = m(ids, labels=labels, teacher_logits=targets[0], teacher_tokens=targets[1], distill_temperature=2.0,
                distill_weight=0.5)
        out.loss.backward()
        results.append((out.loss.item(), out.logits.detach(), {n: p.grad for n, p in m.named_parameters()}))
    (l0, z0, g0), (l1, z1, g1) = results
    assert torch.equal(z0, z1)                                 # the embedding's rows are copies
    assert abs(l0 - l1) <= 64 * U * abs(l0)
    for n in g0:
        # fp32 products and sums over the network in both: errors of some 2^-16 of the largest entry
        assert (g0[n] - g1[n]).abs().max() <= 2.0 ** -14 * g0[n].abs().max(), n


def test_model_keeps_what_stands_around_the_embedding():
    cfgd, sd = tiny("tiny_a")
    m = product_model(cfgd, sd, device=DEV).enable_fused_vocab()
    ids = torch.randint(0, 255, (1, 9), device=DEV, generator=gen(2))
    seen = []
    h = m.embedding.register_forward_hook(lambda mod, a, y: seen.append(1) or y * 2)
    ref = product_model(cfgd, sd, device=DEV)
    ref.embedding.register_forward_hook(lambda mod, a, y: y * 2)
    with torch.no_grad():
        assert torch.equal(m(ids).logits, ref(ids).logits) and seen
        h.remove()
        assert torch.equal(m(ids).logits, product_model(cfgd, sd, device=DEV)(ids).logits)
