"""The post-training operators as programs use them: registered operations, compilers, captures, streams and threads, hooks, second
derivatives, tensors of inference mode, rows past the caches, sizes that do not fit, and a model's post-training steps."""

import threading

import pytest
import torch

from dispatcher_hybrid import logprobs as plain
from helpers import product_model, tiny

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
TYPES = [torch.bfloat16, torch.float32]
IGNORE = -100


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def ops():
    from dispatcher_hybrid import fused_logprobs
    return fused_logprobs


def say(*what):
    print(*what, flush=True)


def data(B, T, V, dtype, seed):
    """logits, tokens, old and reference log-probabilities, advantages, sums of a reference."""
    g = gen(seed)
    z = (torch.randn(B, T, V, device=DEV, generator=g) * 2).to(dtype)
    tokens = torch.randint(0, V, (B, T), device=DEV, generator=g)
    tokens[torch.rand(B, T, device=DEV, generator=g) < 0.2] = IGNORE
    lp = plain.token_logprobs(z.double(), tokens)
    old = (lp + 0.2 * torch.randn(B, T, device=DEV, generator=g)).float()
    ref = (lp + 0.2 * torch.randn(B, T, device=DEV, generator=g)).float()
    sums = (lp.sum(1) + torch.randn(B, device=DEV, generator=g)).float()
    return z, tokens, old, ref, torch.randn(B, device=DEV, generator=g), sums


def losses(f, z, tokens, old, ref, adv, sums):
    """The three differentiable operators' outputs in z."""
    return [*f.token_logprobs(z, tokens, 0.8, entropy=True), f.preference_loss(z, tokens, sums, beta=0.2, label_smoothing=0.1)[0],
            f.policy_loss(z, tokens, old, adv, ref, kl_weight=0.1, entropy_weight=0.02, reduction="sequence")[0]]


def step(z, *rest):
    """All values and the gradients of each, as one pass of each operator."""
    leaf = z.detach().requires_grad_()
    lp, ent, pref, pol = losses(ops(), leaf, *rest)
    w = torch.linspace(-1, 1, lp.numel(), device=z.device).view(lp.shape)
    return [lp.detach(), ent.detach(), pref.detach(), pol.detach(), torch.autograd.grad((lp, ent), leaf, (w, 0.1 * w))[0],
            torch.autograd.grad(pref, leaf)[0], torch.autograd.grad(pol, leaf)[0]]


def test_registered_operations_agree_with_the_direct_launches():
    z, tokens, old, ref, adv, sums = data(4, 9, 501, torch.float32, 1)
    o, h, w = torch.ops.dispatcher, torch.randn(4, 9, 64, device=DEV, generator=gen(2)), torch.randn(501, 64, device=DEV, generator=gen(3))
    for entropy in (False, True):
        for tau in (1.0, 0.5):
            a, b = z.clone().requires_grad_(), z.clone().requires_grad_()
            x = ops().token_logprobs(a, tokens, tau, entropy=entropy)
            x = x if entropy else (x,)
            y = o.token_logprobs(b, tokens, tau, IGNORE, entropy)
            sum(t.sum() for t in x).backward()
            sum(t.sum() for t in y[:-1]).backward()
            assert all(torch.equal(s, t) for s, t in zip(x, y)) and torch.equal(a.grad, b.grad) and y[-1].numel() == 4 * 36
        x = ops().head_logprobs(h, w, tokens, 0.7, entropy=entropy)
        y = o.head_logprobs(h, w, tokens, 0.7, IGNORE, entropy, False)
        assert all(torch.equal(s, t) for s, t in zip(x if entropy else (x,), y))
    for red in range(3):
        a, b = z.clone().requires_grad_(), z.clone().requires_grad_()
        x = ops().preference_loss(a, tokens, sums, reduction=plain.PAIR_REDUCTIONS[red])
        y = o.preference_loss(b, tokens, sums, 0, False, 0.1, 0.0, 0.0, IGNORE, red)
        x[0].sum().backward()
        y[0].sum().backward()
        assert torch.equal(x[0], y[0]) and torch.equal(x[1], y[1]) and torch.equal(a.grad, b.grad)
    for red in range(4):
        for w_ent in (0.0, 0.1):
            a, b = z.clone().requires_grad_(), z.clone().requires_grad_()
            x = ops().policy_loss(a, tokens, old, adv, ref, kl_weight=0.1, entropy_weight=w_ent, reduction=plain.TOKEN_REDUCTIONS[red])
            y = o.policy_loss(b, tokens, old, adv, ref, 0.2, 0.2, 0.1, w_ent, 1.0, IGNORE, red)
            x[0].sum().backward()
            y[0].sum().backward()
            assert torch.equal(x[0], y[0]) and torch.equal(x[1], y[1]) and torch.equal(a.grad, b.grad)
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode() as fake:
        f = lambda q: fake.from_tensor(q)
        assert [t.shape for t in ops().token_logprobs(f(z), f(tokens), entropy=True)] == [(4, 9), (4, 9)]
        assert ops().head_logprobs(f(h), f(w), f(tokens)).shape == (4, 9)
        assert [t.shape for t in ops().preference_loss(f(z), f(tokens), f(sums))] == [(), (4,)]
        assert [t.shape for t in ops().policy_loss(f(z), f(tokens), f(old), f(adv), reduction="none")] == [(4, 9), (4, 9)]


def test_under_a_compiler_and_a_transform():
    args = data(4, 9, 501, torch.float32, 5)
    h, w = torch.randn(4, 9, 64, device=DEV, generator=gen(2)), torch.randn(501, 64, device=DEV, generator=gen(3))

    def total(z, *rest):
        lp, ent, pref, pol = losses(ops(), z * 1.5, *rest)
        return lp.sum() + 0.1 * ent.sum() + pref + pol + ops().head_logprobs(h, w, rest[0]).sum()
    grads = []
    for fn in (total, torch.compile(total, backend="aot_eager", fullgraph=True)):
        leaf = args[0].clone().requires_grad_()
        loss = fn(leaf, *args[1:])
        grads.append([loss.detach(), *torch.autograd.grad(loss, leaf)])
    for x, y in zip(*grads):
        assert torch.equal(x, y)
    with pytest.raises(RuntimeError, match="functorch"):
        torch.func.grad(total)(*args)


def test_second_derivatives():
    args = data(4, 6, 37, torch.float32, 7)
    z, rest = args[0], args[1:]
    v = torch.randn(z.shape, device=DEV, generator=gen(8))
    for i in range(4):
        got = []
        for f, x in ((ops(), z), (plain, z.double())):
            leaf = x.clone().requires_grad_()
            out = losses(f, leaf, *rest)[i]
            g, = torch.autograd.grad(out.square().sum(), leaf, create_graph=True)
            got += [g.detach(), torch.autograd.grad((g * v).sum(), leaf)[0]]
        for a, b in ((got[0], got[2]), (got[1], got[3])):
            # fp32 formulas on 37 logits against fp64: some tens of roundings of the largest entry
            assert (a - b).abs().max() <= 128 * U * b.abs().max(), i


def test_gradients_scale_and_repeat():
    args = data(4, 9, 1003, torch.bfloat16, 9)
    one = step(*args)
    for x, y in zip(one, step(*args)):
        assert torch.equal(x, y)
    leaf = args[0].clone().requires_grad_()
    for loss in losses(ops(), leaf, *args[1:])[2:]:
        a, = torch.autograd.grad(loss, leaf, retain_graph=True)
        b, = torch.autograd.grad(loss, leaf, torch.full((), 4.0, device=DEV), retain_graph=True)
        c, = torch.autograd.grad(loss / 4, leaf)
        assert torch.equal(b, a * 4) and torch.equal(c, a / 4)     # a power of two: the same roundings
    lp, ent = ops().token_logprobs(leaf, args[1], entropy=True)
    lp.mul_(2.0)                                                  # an output may be changed in place
    a, = torch.autograd.grad(lp.sum(), leaf)
    b, = torch.autograd.grad(ops().token_logprobs(leaf, args[1]).sum(), leaf)
    assert torch.equal(a, b * 2)


def test_another_stream_and_two_calls_at_once():
    sets = [data(4, 33, 5003, torch.bfloat16, 11), data(4, 33, 5003, torch.bfloat16, 12)]
    heads = [(torch.randn(200, 128, device=DEV, generator=gen(i)).to(torch.bfloat16),
              torch.randn(5003, 128, device=DEV, generator=gen(9)).to(torch.bfloat16),
              torch.randint(0, 5003, (200,), device=DEV, generator=gen(i + 5))) for i in range(2)]

    def run(i):
        return [*step(*sets[i]), *ops().head_logprobs(*heads[i], entropy=True), ops().head_logprobs(*(t[:9] if t.shape[0] == 200 else t
                                                                                                for t in heads[i]))]
    ref = [run(i) for i in range(2)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append(run(i))
        torch.cuda.synchronize()
        for x, y in zip(got, ref):
            assert all(torch.equal(p, q) for p, q in zip(x, y))


def test_two_host_threads():
    sets = [data(2, 20, 3001, torch.float32, 13), data(2, 20, 3001, torch.float32, 14)]
    head = torch.randn(30, 256, device=DEV, generator=gen(1)), torch.randn(3001, 256, device=DEV, generator=gen(2)), \
        torch.randint(0, 3001, (30,), device=DEV, generator=gen(3))
    run = lambda i: [*step(*sets[i]), ops().head_logprobs(*head)]
    ref, got = [run(i) for i in range(2)], [None, None]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5):
                got[i] = run(i)
            torch.cuda.current_stream().synchronize()
    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    for x, y in zip(got, ref):
        assert all(torch.equal(p, q) for p, q in zip(x, y))


@pytest.mark.parametrize("T,V,d", [(40, 3001, 64), (300, 700, 128), (5, 9001, 64)])
def test_two_captured_steps_replayed_in_turn(T, V, d):
    """A policy step as a user runs it: the sampled tokens' old and reference log-probabilities from hidden states, the head, the
    loss and its gradient, and a preference loss beside it; captured twice with inputs of their own, replayed in turn, each replay
    against the eager result. The number of ignored positions changes between replays."""
    g = gen(16)
    W = (torch.randn(V, d, device=DEV, generator=g) * 0.3).to(torch.bfloat16)
    sets = [dict(x=torch.randn(4, T, d, device=DEV, generator=g).to(torch.bfloat16), x2=torch.randn(4, T, d, device=DEV, generator=g).to(torch.bfloat16),
                 tok=torch.randint(0, V, (4, T), device=DEV, generator=g), adv=torch.randn(4, device=DEV, generator=g)) for _ in range(2)]

    def run(s):
        old, ent = ops().head_logprobs(s["x2"], W, s["tok"], entropy=True)
        w = W.detach().requires_grad_()
        z = s["x"].view(-1, d).mm(w.t()).view(4, T, V)
        loss, lp = ops().policy_loss(z, s["tok"], old, s["adv"], old, kl_weight=0.1, entropy_weight=0.01, reduction="sequence")
        pref, sums = ops().preference_loss(z, s["tok"], old.sum(1))
        return [old, ent, loss.detach(), lp, pref.detach(), sums, *torch.autograd.grad(loss + pref, w)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in sets:
            run(s)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for s in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run(s)
        graphs.append((graph, out))
    for turn in range(3):
        for s in sets:
            for name in ("x", "x2", "adv"):
                s[name].normal_(generator=g)
            s["tok"].copy_(torch.randint(0, V, (4, T), device=DEV, generator=g))
            s["tok"][torch.rand(4, T, device=DEV, generator=g) < (0.0, 0.6, 1.0)[turn]] = IGNORE
            if turn == 2:
                s["tok"][0, 0] = 3
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for s, (_, out) in zip(sets, graphs):
            for a, b in zip(out, run(s)):
                assert torch.equal(a, b), turn


def test_saved_tensors_that_hooks_move():
    args = data(4, 9, 501, torch.bfloat16, 22)

    def strided(x):                                            # the same values at odd addresses and strides
        wide = torch.empty(x.numel() * 2 + 1, dtype=x.dtype, device=x.device)[1:].view(*x.shape, 2)[..., 0] if x.dim() else x
        return wide.copy_(x) if x.dim() else x
    ref = step(*args)
    with torch.autograd.graph.save_on_cpu():
        on_cpu = step(*args)
    with torch.autograd.graph.saved_tensors_hooks(lambda x: x, strided):
        moved = step(*args)
    for other in (on_cpu, moved):
        assert all(torch.equal(x, y) for x, y in zip(ref, other))


def test_tensors_of_inference_mode():
    z, tokens, old, ref, adv, sums = data(4, 9, 501, torch.float32, 23)
    want = step(z, tokens, old, ref, adv, sums)
    with torch.inference_mode():
        frozen = [t.clone() for t in (tokens, old, ref, adv, sums)]
        values = ops().token_logprobs(z, tokens, 0.8, entropy=True)
    assert all(torch.equal(a, b) for a, b in zip(step(z, *frozen), want)) and all(torch.equal(a, b) for a, b in zip(values, want))
    leaf = z.clone().requires_grad_()
    loss = torch.ops.dispatcher.policy_loss(leaf, *frozen[:2], frozen[3], frozen[2], 0.2, 0.2, 0.1, 0.02, 1.0, IGNORE, 3)[0]
    assert torch.equal(torch.autograd.grad(loss, leaf)[0], want[-1])


@pytest.mark.parametrize("shape", [(0, 5), (3, 0)])
def test_a_policy_step_of_nothing_with_a_reference(shape):
    z = torch.randn(*shape, 11, device=DEV, requires_grad=True)
    tok, none = torch.zeros(shape, dtype=torch.long, device=DEV), torch.zeros(shape, device=DEV)
    loss, lp = ops().policy_loss(z, tok, none, none, none, kl_weight=0.1, entropy_weight=0.1, reduction="sum")
    assert loss == 0 and lp.shape == shape and torch.autograd.grad(loss, z)[0].shape == z.shape


def test_constants_of_other_types():
    z, tokens, old, ref, adv, sums = data(4, 9, 501, torch.float32, 24)
    old, ref, adv, sums = (t.bfloat16().float() for t in (old, ref, adv, sums))
    want = step(z, tokens, old, ref, adv, sums)
    for dtype in (torch.bfloat16, torch.float64):
        got = step(z, tokens.int(), *(t.to(dtype) for t in (old, ref, adv, sums)))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    wide = torch.empty(4, 18, device=DEV)[:, ::2].copy_(old)
    assert all(torch.equal(a, b) for a, b in zip(step(z, tokens, wide, ref.t().contiguous().t(), adv, sums), want))


@pytest.mark.parametrize("dtype,rows,V", [(torch.bfloat16, 1100, 130001), (torch.float32, 1100, 65001), (torch.bfloat16, 40000, 4000)])
def test_rows_past_the_caches_have_the_bits_of_smaller_calls(dtype, rows, V):
    """286 MB of logits and gradient or more: read and stored past the caches, the same bits as in smaller calls."""
    g = gen(25)
    z = torch.randn(rows, V, device=DEV, generator=g).to(dtype)
    tokens = torch.randint(0, V, (rows,), device=DEV, generator=g)
    tokens[::7] = IGNORE
    a = torch.randn(rows, device=DEV, generator=g)
    a[::5] = 0.0

    def run(x, t, a):
        leaf = x.detach().requires_grad_()
        lp, ent = ops().token_logprobs(leaf, t, entropy=True)
        return [lp.detach(), ent.detach(), *torch.autograd.grad((lp, ent), leaf, (a, a * 0.5))]
    whole = run(z, tokens, a)
    half = rows // 2
    for part in (slice(0, half), slice(half, rows)):
        # (a slice that begins at another row has other 16-byte boundaries where rows are odd: its gradients' too)
        if part.start == 0 or V * z.element_size() % 16 == 0:
            for x, y in zip(run(z[part], tokens[part], a[part]), whole):
                assert torch.equal(x, y[part])
    assert not bool(whole[2][::35].any()) and bool((whole[2][1::35] != 0).any())


@pytest.mark.parametrize("rows,V", [(40, 50257), (1500, 1003), (1030, 9001)])
def test_broadcast_rows_and_offsets(rows, V):
    """One row of logits for many positions (stride 0): every position's values, and a gradient of each, equal."""
    z = torch.randn(1, V, device=DEV, generator=gen(26)).expand(rows, V)
    tokens = torch.full((rows,), 5, device=DEV)
    leaf = z.detach().requires_grad_()
    lp, ent = ops().token_logprobs(leaf, tokens, entropy=True)
    dz, = torch.autograd.grad((lp, ent), leaf, (torch.ones_like(lp), torch.ones_like(lp)))
    assert bool((lp == lp[0]).all()) and bool((ent == ent[0]).all())
    if V % 4 == 0 or rows * V % 2:                               # (the pieces of gradient rows begin at their own boundaries)
        assert (dz - dz[0]).abs().max() <= 8 * U * dz[0].abs().max()


def test_offsets_past_32_bits():
    """Logits of more than 2^32 elements by their strides, in rows far apart; hidden states likewise."""
    free, _ = torch.cuda.mem_get_info()
    if free < 40 << 30:
        pytest.skip("needs 20 GB")
    V = 1003
    big = torch.empty((1 << 32) + 5 * V, dtype=torch.bfloat16, device=DEV)
    far = 1 << 31
    z = torch.as_strided(big, (3, 2, V), (far, 2 * V, 1))
    z.copy_(torch.randn(3, 2, V, device=DEV, generator=gen(27)))
    tokens = torch.randint(0, V, (3, 2), device=DEV, generator=gen(28))
    near = z.contiguous()
    a, b = (ops().token_logprobs(x, tokens, entropy=True) for x in (z, near))
    assert (a[0] - b[0]).abs().max() < 1e-5 and (a[1] - b[1]).abs().max() < 1e-5
    h = torch.as_strided(big, (3, 64), (far, 1))
    w = torch.randn(V, 64, device=DEV, generator=gen(29)).to(torch.bfloat16)
    assert torch.equal(ops().head_logprobs(h.contiguous(), w, tokens[:, 0]).isfinite(), torch.ones(3, dtype=torch.bool, device=DEV))
    assert (ops().head_logprobs(h, w, tokens[:, 0]) - ops().head_logprobs(h.contiguous(), w, tokens[:, 0])).abs().max() < 1e-4
    wf = torch.as_strided(big, (3, 64), (far, 1))
    assert (ops().head_logprobs(w[:40], wf, tokens[:1, 0].expand(40) % 3)
            - ops().head_logprobs(w[:40], wf.contiguous(), tokens[:1, 0].expand(40) % 3)).abs().max() < 1e-4


def test_an_allocation_that_fails_is_torchs_error():
    z = torch.zeros(1, 1, 1, device=DEV).expand(1 << 10, 1 << 10, 1 << 22)
    tok = torch.zeros(1 << 10, 1 << 10, dtype=torch.long, device=DEV)
    zeros = torch.zeros(1 << 10, 1 << 10, device=DEV)
    torch.cuda.synchronize()
    torch.cuda.set_per_process_memory_fraction(0.05)
    try:
        for call in (lambda: ops().token_logprobs(z, tok), lambda: torch.ops.dispatcher.token_logprobs(z, tok, 1.0, IGNORE, False),
                     lambda: ops().preference_loss(z, tok), lambda: ops().policy_loss(z, tok, zeros, zeros),
                     lambda: ops().head_logprobs(z[..., :1 << 20], z[0, :1, :1 << 20], tok)):
            with pytest.raises(torch.OutOfMemoryError, match="out of memory"):
                call()
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)


def test_refusals_on_the_gpu():
    z, tokens, old, ref, adv, sums = data(4, 9, 51, torch.float32, 30)
    h, w = torch.randn(4, 9, 8, device=DEV), torch.randn(51, 8, device=DEV)
    for call in (lambda: ops().token_logprobs(z.half(), tokens), lambda: ops().preference_loss(z.half(), tokens),
                 lambda: ops().policy_loss(z.double(), tokens, old, adv), lambda: ops().head_logprobs(h.half(), w.half(), tokens)):
        with pytest.raises(TypeError, match="float32 and bfloat16"):
            call()
    for call in (lambda: ops().token_logprobs(z, tokens.cpu()), lambda: ops().preference_loss(z, tokens, sums.cpu()),
                 lambda: ops().policy_loss(z, tokens, old.cpu(), adv), lambda: ops().policy_loss(z, tokens, old, adv.cpu()),
                 lambda: ops().policy_loss(z, tokens, old, adv, ref.cpu(), kl_weight=0.1), lambda: ops().head_logprobs(h, w.cpu(), tokens),
                 lambda: ops().head_logprobs(h, w, tokens.cpu())):
        with pytest.raises(RuntimeError, match="one device"):
            call()
    with pytest.raises(RuntimeError, match="no gradient"):
        ops().head_logprobs(h.requires_grad_(), w, tokens)
    with torch.no_grad():
        assert not ops().head_logprobs(h, w, tokens).requires_grad


def test_launches_refuse_sizes_that_do_not_fit():
    """The registered operations by name, and tensors that a hook hands back smaller: nothing is launched."""
    o = torch.ops.dispatcher
    z, tokens, old, ref, adv, sums = data(4, 9, 51, torch.float32, 31)
    h, w = torch.randn(4, 9, 8, device=DEV), torch.randn(51, 8, device=DEV)
    kept = o.token_logprobs(z, tokens, 1.0, IGNORE, False)[-1]
    p, q = o.preference_loss(z, tokens, sums, 0, False, 0.1, 0.0, 0.0, IGNORE, 1), o.policy_loss(z, tokens, old, adv, None, 0.2, 0.2, 0.0, 0.0, 1.0, IGNORE, 1)
    one = torch.ones((), device=DEV)
    for exc, call in (
            (TypeError, lambda: o.token_logprobs(z, tokens.byte(), 1.0, IGNORE, False)),
            (ValueError, lambda: o.token_logprobs(z, tokens[:3], 1.0, IGNORE, False)),
            (ValueError, lambda: o.token_logprobs(z, tokens, 0.0, IGNORE, False)),
            (ValueError, lambda: o.token_logprobs_grad(old[:3], None, z, tokens, kept, 1.0, IGNORE)),
            (ValueError, lambda: o.token_logprobs_grad(None, old[:3], z, tokens, kept, 1.0, IGNORE)),
            (ValueError, lambda: o.token_logprobs_grad(old, None, z, tokens, kept[:-1], 1.0, IGNORE)),
            (ValueError, lambda: o.preference_loss(z[:3], tokens[:3], None, 0, False, 0.1, 0.0, 0.0, IGNORE, 1)),
            (ValueError, lambda: o.preference_loss(z[0], tokens[0], None, 0, False, 0.1, 0.0, 0.0, IGNORE, 1)),
            (ValueError, lambda: o.preference_loss(z, tokens, sums[:3], 0, False, 0.1, 0.0, 0.0, IGNORE, 1)),
            (ValueError, lambda: o.preference_loss(z, tokens, sums, 5, False, 0.1, 0.0, 0.0, IGNORE, 1)),
            (ValueError, lambda: o.preference_loss(z, tokens, sums, (1 << 32) + 1, False, 0.1, 0.0, 0.0, IGNORE, 1)),
            (ValueError, lambda: o.preference_loss(z, tokens, sums, 0, False, -1.0, 0.0, 0.0, IGNORE, 1)),
            (ValueError, lambda: o.preference_loss_grad(old[0, :3], z, tokens, p[2], IGNORE, 0)),
            (ValueError, lambda: o.preference_loss_grad(one, z, tokens, p[2][:-1], IGNORE, 1)),
            (ValueError, lambda: o.policy_loss(z, tokens, old[:3], adv, None, 0.2, 0.2, 0.0, 0.0, 1.0, IGNORE, 1)),
            (ValueError, lambda: o.policy_loss(z, tokens, old, adv[:3], None, 0.2, 0.2, 0.0, 0.0, 1.0, IGNORE, 1)),
            (ValueError, lambda: o.policy_loss(z, tokens, old, adv, ref[:3], 0.2, 0.2, 0.1, 0.0, 1.0, IGNORE, 1)),
            (ValueError, lambda: o.policy_loss(z, tokens, old, adv, None, 0.2, 0.2, 0.1, 0.0, 1.0, IGNORE, 1)),
            (ValueError, lambda: o.policy_loss(z, tokens, old, adv, None, 0.2, 0.2, 0.0, 0.0, 1.0, IGNORE, 4)),
            (ValueError, lambda: o.policy_loss_grad(one, z, tokens, q[2], 0.1, 1.0, IGNORE, 1)),
            (ValueError, lambda: o.policy_loss_grad(old, z, tokens, q[2], 0.0, 1.0, IGNORE, 1)),
            (TypeError, lambda: o.head_logprobs(h, w.bfloat16(), tokens, 1.0, IGNORE, False, False)),
            (ValueError, lambda: o.head_logprobs(h, w[:, :7], tokens, 1.0, IGNORE, False, False)),
            (ValueError, lambda: o.head_logprobs(h, w, tokens[:3], 1.0, IGNORE, False, False)),
            (TypeError, lambda: o.head_logprobs(h, w, tokens.byte(), 1.0, IGNORE, False, False))):
        with pytest.raises(exc):
            call()
    leaf = z.clone().requires_grad_()
    with torch.autograd.graph.saved_tensors_hooks(lambda x: x, lambda x: x[:2]):
        for loss in (ops().token_logprobs(leaf, tokens).sum(), ops().preference_loss(leaf, tokens)[0], ops().policy_loss(leaf, tokens, old, adv)[0]):
            with pytest.raises((ValueError, RuntimeError)):
                torch.autograd.grad(loss, leaf)
    torch.cuda.synchronize()


# ---- the model --------------------------------------------------------------------------------------------------------

def test_model_steps_against_torch():
    """Scores and losses of the model with the kernels against the same without them (fp32: the same layers, so the difference is
    the fp32 error of the head, the loss and the embedding alone)."""
    cfgd, sd = tiny("tiny_a")
    ids = torch.randint(0, 255, (4, 40), device=DEV, generator=gen(1))
    labels = ids.clone()
    labels[:, :9] = IGNORE
    labels[1, 30:] = IGNORE
    m = product_model(cfgd, sd, device=DEV)
    want = m.token_logprobs(ids, labels, 0.9, entropy=True)
    got = m.enable_fused_vocab().token_logprobs(ids, labels, 0.9, entropy=True)
    for a, b in zip(got, want):
        assert a.shape == (4, 40) and (a - b).abs().max() <= 64 * U * b.abs().max() and not bool(a[:, -1].any())
    # (what stands around the head is called)
    handle = m.lm_head.register_forward_hook(lambda mod, a, y: y * 0.5)
    hooked = m.token_logprobs(ids, labels, 0.9)
    assert (hooked - m.enable_fused_vocab(False).token_logprobs(ids, labels, 0.9)).abs().max() < 1e-4 and (hooked - got[0]).abs().max() > 1e-2
    handle.remove()
    old = want[0] + 0.1 * torch.randn(4, 40, device=DEV, generator=gen(2))
    adv = torch.randn(4, device=DEV, generator=gen(3))
    asks = [dict(preference=dict(reference=want[0].sum(1) + torch.randn(4, device=DEV, generator=gen(4)), beta=0.3)),
            dict(policy=dict(old_logprobs=old, advantages=adv, reference_logprobs=want[0], kl_weight=0.1, entropy_weight=0.01,
                             temperature=0.9, reduction="sequence"))]
    for ask in asks:
        results = []
        for fused in (False, True):
            m = product_model(cfgd, sd, device=DEV).train().enable_fused_vocab(fused)
            out = m(ids, labels=labels, **ask)
            out.loss.backward()
            results.append((out.loss.item(), out.logprobs, {n: p.grad for n, p in m.named_parameters()}))
        (l0, s0, g0), (l1, s1, g1) = results
        assert abs(l0 - l1) <= 256 * U * max(abs(l0), 1.0) and (s0 - s1).abs().max() <= 256 * U * s0.abs().max()
        for n in g0:
            # fp32 products and sums over the network in both: errors of some 2^-16 of the largest entry
            assert (g0[n] - g1[n]).abs().max() <= 2.0 ** -14 * g0[n].abs().max(), n


def test_a_bf16_model_scores_and_trains_with_all_kernels():
    cfgd, sd = tiny("tiny_b")
    m = product_model(cfgd, sd, device=DEV, dtype=torch.bfloat16).enable_fused_gates().enable_fused_vocab()
    V = cfgd["vocab_size"]
    ids = torch.randint(0, V - 1, (4, 33), device=DEV, generator=gen(5))
    old = m.token_logprobs(ids)
    with torch.no_grad():
        logits = m(ids).logits
    moved = torch.cat([ids[:, 1:], torch.full_like(ids[:, :1], IGNORE)], 1)
    stored = ops().token_logprobs(logits, moved)
    # equal but where the rounding of a logit falls the other way (the library's head sums in another order)
    assert (old - stored).abs().max() <= 2.0 ** -7 * logits.abs().max() and ((old - stored).abs() < 1e-3).double().mean() > 0.8
    m.train()
    out = m(ids, labels=ids, policy=dict(old_logprobs=old, advantages=torch.ones(4, device=DEV)))
    out.loss.backward()
    assert abs(out.loss.item() + 1.0) < 0.05                      # ratios near one, advantages of one
    assert all(p.grad is not None and bool(p.grad.isfinite().all()) for p in m.parameters())
    m.zero_grad()
    out = m(ids, labels=ids, preference=dict(reference=old.sum(1)))
    out.loss.backward()
    assert abs(out.loss.item() - 0.6931) < 0.1 and all(bool(p.grad.isfinite().all()) for p in m.parameters())
