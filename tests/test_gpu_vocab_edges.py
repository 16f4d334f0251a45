"""Corners of the vocabulary-end operators on the GPU: teachers without probabilities, exponents far below the maximum, tied and
masked vocabularies, gradients past the caches, tensors of inference mode, refused sizes and allocations.

u = 2^-24, half a step of fp32."""

import math

import pytest
import torch

from dispatcher_hybrid import distillation as plain

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
TYPES = [torch.bfloat16, torch.float32]


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def ops():
    from dispatcher_hybrid import fused_vocab
    return fused_vocab


def say(*what):
    print(*what, flush=True)


# ---- distillation loss ----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,V", [(3, 50257), (700, 1003)])                     # a row over several workgroups, one each
@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("with_labels", [False, True])
def test_a_teacher_without_probabilities_makes_its_whole_row_nan(with_labels, value, rows, V, dtype):
    say("teacher", value, rows, V, dtype, with_labels)
    g = gen(rows)
    z = torch.randn(rows, V, device=DEV, generator=g).to(dtype)
    t = torch.randn(rows, 5, device=DEV, generator=g).to(dtype)
    tok = torch.randint(0, V, (rows, 5), device=DEV, generator=g)
    labels = torch.randint(0, V, (rows,), device=DEV, generator=g) if with_labels else None
    t[1, 3] = value
    t[2, 3], tok[2, 3] = value, -1                             # an empty slot may hold anything
    for fn in (ops().distillation_loss, plain.distillation_loss):
        leaf = z.clone().requires_grad_()
        each = fn(leaf, t, tok, labels, 2.0, 0.5 if with_labels else 1.0, reduction="none")
        grad, = torch.autograd.grad(each.sum(), leaf)
        bad = torch.arange(rows, device=DEV) == 1
        assert torch.equal(each.isnan(), bad)
        assert torch.equal(grad.isnan(), bad.unsqueeze(1).expand(rows, V))


@pytest.mark.parametrize("rows", [4, 600])
@pytest.mark.parametrize("tau,w", [(1.0, 1.0), (2.0, 0.0), (3.0, 1.0), (4.0, 0.5), (2.0, 0.5), (0.75, 0.5)])
def test_fp32_probabilities_far_below_the_maximum(tau, w, rows):
    """Rows of one logit at 0 and the others at exponents of -20 to -80, all multiples of 2^-10 (their differences are exact).

    Every exp: one unit of exp2 (2 u) and the rounding of its correction, 3 u. The sum is 1 and some 1e-6: at most four roundings
    in the thread that holds the 1, six in its wave, three over the waves, 13 u. Then 1 / sum 1 u, the factor of the term
    (weight, temperature, 1 / sum) 3 u, its product 1 u, the two terms' sum 1 u: 22 u in all."""
    say("far", tau, w, rows)
    V, g = 1000, gen(rows)
    soft = tau if w > 0 else 1.0
    x = (-20 - 60 * torch.rand(rows, V, device=DEV, generator=g)) * soft
    x = (x * 1024).round() / 1024
    x[:, 17] = 0
    t, tok = torch.zeros(rows, 1, device=DEV), torch.full((rows, 1), 17, device=DEV)
    labels = tok[:, 0].clone()
    leaf, wide = x.clone().requires_grad_(), x.double().requires_grad_()
    grad, = torch.autograd.grad(ops().distillation_loss(leaf, t, tok, labels, tau, w, reduction="sum"), leaf)
    ref, = torch.autograd.grad(plain.distillation_loss(wide, t.double(), tok, labels, tau, w, reduction="sum"), wide)
    far = torch.arange(V, device=DEV) != 17
    worst = ((grad.double() - ref).abs() / ref.abs())[:, far].max().item() / U
    assert worst <= 22, worst


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tau,w", [(1.0, 1.0), (2.0, 0.5), (1.0, 0.0)])
def test_many_small_exponentials_beside_a_large_one(tau, w, dtype):
    """A logit of 0 and 400000 of about -15 (times the temperature), each some 2.5 steps of the numbers from 1 on: added to the 1
    one by one, every rounding is off by nearly half a step to the same side.

    Bounds: a thread reads V / 256 logits, 16 fp32 or 32 bf16 between two roundings of its sum, so the one that holds the 1 is
    off by at most V / 4096 (V / 8192) u; 7 u in a wave, 9 over the waves; the other terms, an eighth of the sum, by 11 u in
    their sums and by 3 u (fp32) or 25 u (bf16: an exponent of 22 rounded twice) each: 5 u of the whole. The loss is the log of
    that sum, a term of it the exponent of the hard one at temperature 2, where all of it is smaller; the gradient's factors
    and its exp 9 u, or 31 u and the type's half step."""
    rows, V = 520, 400001
    x0 = -15.03125 if dtype == torch.float32 else -15.0
    say("small", dtype, tau, w)
    z = torch.full((rows, V), x0 * (tau if w > 0 else 1.0), device=DEV, dtype=dtype)
    z[:, 0] = 0
    t, tok = torch.zeros(rows, 1, device=DEV), torch.zeros(rows, 1, dtype=torch.long, device=DEV)
    labels = tok[:, 0].clone()
    leaf = z.clone().requires_grad_()
    each = ops().distillation_loss(leaf, t, tok, labels, tau, w, reduction="none")
    grad, = torch.autograd.grad(each.sum(), leaf)
    at = float(z[0, 1])
    sums = lambda s: 1 + (V - 1) * math.exp(at / s)
    loss = w * tau * tau * math.log(sums(tau)) + (1 - w) * math.log(sums(1.0))
    dz = w * tau * math.exp(at / tau) / sums(tau) + (1 - w) * math.exp(at) / sums(1.0)
    full = dtype == torch.float32
    bound = V / (4096 if full else 8192) + 7 + 9 + 5 + 2
    scale = w * tau * tau + (1 - w)
    worst = (each.double() - loss).abs().max().item() / U
    assert worst <= bound * scale, (worst, bound * scale)
    worst = (grad[:, 1:].double() - dz).abs().max().item() / dz
    assert worst <= (bound + (9 if full else 31)) * U + (0 if full else 2.0 ** -8), (worst / U, bound)


@pytest.mark.parametrize("tau", [1e-30, 0.5, 3.0, 1e30])
@pytest.mark.parametrize("rows", [2, 600])
def test_fp32_infinite_and_lowest_logits_at_any_temperature(rows, tau):
    """What a mask leaves of a vocabulary, at temperatures at both ends: no exponent becomes NaN, masked tokens get zeros."""
    say("masked", rows, tau)
    V, low = 2003, torch.finfo(torch.float32).min
    z = torch.randn(rows, V, device=DEV, generator=gen(rows))
    z[0, 5:], z[1, 5:] = -math.inf, low
    t, tok = torch.zeros(rows, 2, device=DEV), torch.randint(0, 5, (rows, 2), device=DEV, generator=gen(1))
    labels = tok[:, 0].clone()
    for w in (1.0, 0.5):
        leaf = z.clone().requires_grad_()
        each = ops().distillation_loss(leaf, t, tok, labels, tau, w, reduction="none")
        grad, = torch.autograd.grad(each[:2].sum(), leaf)
        assert bool(grad.isfinite().all()) and bool((grad[:2, 5:] == 0).all()) and not bool(each.isnan().any())


@pytest.mark.parametrize("dtype,rows,V", [(torch.bfloat16, 1100, 130001), (torch.float32, 1100, 65001),
                                          (torch.bfloat16, 40, 4000001)])         # odd rows; the last over several workgroups
def test_gradients_past_the_caches(dtype, rows, V):
    """A gradient of more than 256 MiB, stored past the caches with the named tokens written behind, against the same rows in two
    calls of less: the same bits."""
    say("past", dtype, rows, V)
    g, size, K = gen(V), 2 if dtype == torch.bfloat16 else 4, 64
    assert rows * V * size >= 256 << 20 > (rows // 2) * V * size
    z = torch.randn(rows, V, device=DEV, generator=g, dtype=torch.bfloat16).to(dtype)
    t = torch.randn(rows, K, device=DEV, generator=g)
    tok = torch.randint(0, V, (rows, K), device=DEV, generator=g)
    tok[:, :10] = torch.arange(10, device=DEV)                                    # the ends of a row, where its pieces begin
    tok[:, 10:20] = V - 1 - torch.arange(10, device=DEV)
    tok[:, 40:] = tok[:, 20:21]                                                   # the same token again and again
    labels = tok[:, 5].clone()
    labels[::7], labels[3] = -100, tok[3, 20]
    f = torch.rand(rows, device=DEV, generator=g) + 0.5
    ops()                                                      # registers them
    o, half = torch.ops.dispatcher, rows // 2
    _, kept = o.distillation_loss(z, t, tok, labels, 2.0, 0.5, -100, 0)
    whole = o.distillation_loss_grad(f, z, t, tok, labels, kept, 2.0, 0.5, -100, 0)
    for a, b in ((0, half), (half, rows)):
        part = o.distillation_loss_grad(f[a:b], z[a:b], t[a:b], tok[a:b], labels[a:b], kept[4 * a:4 * b + 4], 2.0, 0.5, -100, 0)
        assert torch.equal(part, whole[a:b])
    assert bool((whole[::7] == 0).all()) and bool((whole[1, tok[1]] != 0).all())


# ---- errors and foreign tensors -------------------------------------------------------------------------------------

def test_an_allocation_that_fails_is_torchs_error():
    """torch.OutOfMemoryError, as torch's own operations raise it, from the direct calls and the registered operations. The
    allocator refuses by its own limit: nothing is asked of the device."""
    W = torch.zeros(1, 1 << 20, device=DEV)
    ids = torch.zeros(1, dtype=torch.long, device=DEV).expand(1 << 20)
    z = torch.zeros(1, 1, 1, device=DEV).expand(1 << 10, 1 << 10, 1 << 22)
    t, tok = torch.zeros(1 << 10, 1 << 10, 1, device=DEV), torch.zeros(1 << 10, 1 << 10, 1, dtype=torch.long, device=DEV)
    torch.cuda.synchronize()
    torch.cuda.set_per_process_memory_fraction(0.05)
    try:
        for call in (lambda: ops().embed_tokens(ids, W), lambda: torch.ops.dispatcher.embed_tokens(W, ids, 1.0, -1, -1),
                     lambda: ops().top_logits(z, 1), lambda: ops().distillation_loss(z, t, tok)):
            with pytest.raises(torch.OutOfMemoryError, match="out of memory"):
                call()
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)


def test_targets_of_inference_mode():
    """A teacher run under torch.inference_mode sets targets for a training step; labels of that mode too."""
    g = gen(41)
    z, teacher = torch.randn(2, 7, 90, device=DEV, generator=g), torch.randn(2, 7, 90, device=DEV, generator=g)
    with torch.inference_mode():
        targets = ops().top_logits(teacher, 5)
        labels = torch.randint(0, 90, (2, 7), device=DEV, generator=g)
        frozen = ops().distillation_loss(z, *targets, labels, 2.0, 0.5)
    normal = [x.clone() for x in (*targets, labels)]
    losses, grads = [], []
    for t, tok, lb in ((*targets, labels), normal):
        for fn in (lambda *a: ops().distillation_loss(*a), lambda *a: torch.ops.dispatcher.distillation_loss(*a, -100, 1)[0]):
            leaf = z.clone().requires_grad_()
            losses.append(fn(leaf, t, tok, lb, 2.0, 0.5))
            grads.append(torch.autograd.grad(losses[-1], leaf)[0])
    assert all(torch.equal(x, losses[0]) for x in [*losses, frozen]) and all(torch.equal(x, grads[0]) for x in grads)
    leaf = z.clone().requires_grad_()
    one, = torch.autograd.grad(ops().distillation_loss(leaf, *targets, labels, 2.0, 0.5), leaf, create_graph=True)
    assert torch.autograd.grad(one.square().sum(), leaf)[0].isfinite().all()


def test_two_host_threads_with_wide_vocabularies_of_their_own():
    """The one-launch gradient at more than 64 KB of LDS, at two sizes at once."""
    import threading
    data = []
    for V, n in ((122001, 512), (105001, 300)):
        g = gen(V)
        data.append((torch.randn(n, 24, device=DEV, generator=g), torch.randint(0, V, (n,), device=DEV, generator=g), V))
    f = lambda dy, ids, V: ops()._lookup_grad(dy, ids, V, 1.0, -1)
    ref = [f(*d) for d in data]
    for (dy, ids, V), x in zip(data, ref):
        assert (x.double() - torch.zeros(V, 24, dtype=torch.float64, device=DEV).index_add_(0, ids, dy.double())).abs().max() < 1e-4
    torch.cuda.synchronize()
    got, begin = [[], []], threading.Barrier(2)

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            begin.wait(60)
            for _ in range(20):
                got[i].append(f(*data[i]))
            torch.cuda.current_stream().synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join(60)
    for outs, x in zip(got, ref):
        assert len(outs) == 20 and all(torch.equal(o, x) for o in outs)


# ---- top logits -----------------------------------------------------------------------------------------------------

def us(fn, turns=9):
    """Median time of a call among calls, in microseconds."""
    for _ in range(3):
        fn()
    marks = [torch.cuda.Event(enable_timing=True) for _ in range(turns + 1)]
    marks[0].record()
    for m in marks[1:]:
        fn()
        m.record()
    torch.cuda.synchronize()
    return sorted(a.elapsed_time(b) * 1e3 for a, b in zip(marks, marks[1:]))[turns // 2]


def check_top(x, k):
    values, tokens = ops().top_logits(x, k)
    ref, at = torch.sort(x.double(), dim=-1, descending=True, stable=True)
    assert torch.equal(tokens, at[..., :k]) and torch.equal(values, x.gather(-1, tokens))


@pytest.mark.parametrize("dtype,V", [(torch.bfloat16, 16384), (torch.float32, 8192)])
def test_many_targets_of_a_vocabulary_with_few_lines(V, dtype):
    """Just above where a row's groups may be whole lines there are as many lines as targets: neighbouring vocabularies cost
    alike (they were 8 to 15 times apart)."""
    times = []
    for v in (V - 8, V, V + 8, V + 600):
        x = (torch.randn(2048, v, device=DEV, generator=gen(v)) * 2).to(dtype)
        check_top(x[:600], 256)
        times.append(us(lambda: ops().top_logits(x, 256)))
    say("lines", dtype, V, times)
    assert max(times) < 3 * times[0]


ROWS = {"equal": lambda i, x: torch.full_like(x, 1.5),
        "masked": lambda i, x: torch.where(i < 40, x, -math.inf),                 # fewer tokens than targets
        "low": lambda i, x: torch.where((i < 30) | (i >= i.numel() - 9), x, torch.finfo(x.dtype).min),
        "steps": lambda i, x: (i // 512).to(x.dtype).expand_as(x),                # large values in few groups
        "falling steps": lambda i, x: (-(i // 5000)).to(x.dtype).expand_as(x),
        "halves": lambda i, x: torch.where(i % 2 == 0, 2.0, x.clamp(max=1.0)),    # ties in every piece
        "teeth": lambda i, x: ((i * 7919) % 4099 // 512).to(x.dtype).expand_as(x)}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,V", [(1, 50257), (600, 50257), (3, 400001), (700, 9001)])
@pytest.mark.parametrize("what", list(ROWS))
def test_top_logits_of_rows_with_more_candidates_than_fit(what, rows, V, dtype):
    say("top", what, rows, V, dtype)
    x = torch.randn(rows, V, device=DEV, generator=gen(rows + V)).to(dtype)
    x = ROWS[what](torch.arange(V, device=DEV), x)
    for k in (1, 20, 64, 256):
        check_top(x, k)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("what", ["equal", "masked", "steps"])
def test_what_a_masked_vocabulary_costs(what, dtype):
    """Rows of ties and few live tokens against ordinary ones: a few more reads (they took 70 to 150 times as long)."""
    x = (torch.randn(1024, 50257, device=DEV, generator=gen(3)) * 2).to(dtype)
    y = ROWS[what](torch.arange(50257, device=DEV), x).contiguous()
    for k in (64, 256):
        usual, odd = us(lambda: ops().top_logits(x, k)), us(lambda: ops().top_logits(y, k))
        say("cost", what, dtype, k, usual, odd)
        assert odd < 20 * usual


def test_numbers_past_32_bits_are_refused():
    """By the registered operations' names, where nothing else checks them; no rows, so that nothing needs memory."""
    ops()
    o, far = torch.ops.dispatcher, 2 ** 32
    z, tok = torch.zeros(0, 50, device=DEV), torch.zeros(0, 3, dtype=torch.long, device=DEV)
    for call in (lambda: o.top_logits(z, far + 1), lambda: o.distillation_loss(z, z[:, :3], tok, None, 1.0, 1.0, -100, far),
                 lambda: o.distillation_loss(z, z[:, :1].expand(0, far + 3), tok[:, :1].expand(0, far + 3), None, 1.0, 1.0, -100, 1)):
        with pytest.raises(ValueError):
            call()
