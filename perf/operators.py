"""Timed cases of the operators at the vocabulary's ends of training: the embedding lookup with its gradient by sorted
tokens, a teacher's top logits, and the distillation loss on them with its gradient.

Shapes are the released 292M model's (vocabulary 50257, d 1024, contexts up to 4096) and, in drawn cases, other widths and
vocabularies.

`prepare` makes what a training program holds, `run` is one pass, `exact` the same in float64.
With `own` the passes are calls of dispatcher_hybrid.fused_vocab, otherwise plain torch in float32, rounded once.
"""

import math
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_PACKAGE = os.path.join(ROOT, "dispatcher-hybrid-2_amd")
if _PACKAGE not in sys.path:
    sys.path.insert(0, _PACKAGE)
os.environ.setdefault("TRANSFORMERS_VERBOSITY", "error")

own = False

DEV = "cuda"
VOCAB = 50257
IGNORE = -100
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # the next token's rows of sixteen lockstep sequences: the smallest call, launch latency
        {"name": "embed_decode", "kind": "embed", "grad": False, "dtype": "bf16", "b": 16, "T": 1, "V": VOCAB, "d": 1024,
         "scale": 32.0, "pad": 0.0},
        # fine-tuning on one short document: the gradient is almost all rows of zeros
        {"name": "embed_short", "kind": "embed", "grad": True, "dtype": "bf16", "b": 1, "T": 128, "V": VOCAB, "d": 1024,
         "scale": 1.0, "pad": 0.0},
        # a training batch of eight full contexts: the largest lookup and gradient
        {"name": "embed_train", "kind": "embed", "grad": True, "dtype": "bf16", "b": 8, "T": 4096, "V": VOCAB, "d": 1024,
         "scale": 1.0, "pad": 0.0},
        # float32 training of a padded batch of odd length: two fifths of the positions are one token
        {"name": "embed_fp32_padded", "kind": "embed", "grad": True, "dtype": "fp32", "b": 3, "T": 1001, "V": VOCAB,
         "d": 1024, "scale": 1.0, "pad": 0.4},
        # the teacher's distribution after a prompt: one row
        {"name": "top_one", "kind": "top", "dtype": "bf16", "rows": 1, "V": VOCAB, "k": 64},
        # a teacher's float32 logits over one document
        {"name": "top_fp32", "kind": "top", "dtype": "fp32", "rows": 509, "V": VOCAB, "k": 20},
        # targets of a whole micro-batch (four documents of 1024): the largest
        {"name": "top_batch", "kind": "top", "dtype": "bf16", "rows": 4096, "V": VOCAB, "k": 64},
        # a training step's loss on a few positions (an answer behind a long prompt)
        {"name": "distill_few", "kind": "distill", "grad": True, "dtype": "bf16", "b": 1, "T": 24, "V": VOCAB, "k": 16,
         "temperature": 2.0, "weight": 0.5, "labels": True, "empty": False},
        # held-out loss of every position, no gradient
        {"name": "distill_eval", "kind": "distill", "grad": False, "dtype": "bf16", "b": 2, "T": 1024, "V": VOCAB, "k": 64,
         "temperature": 2.0, "weight": 0.5, "labels": True, "empty": False},
        # a micro-batch of four documents, soft and hard targets: the largest loss and gradient
        {"name": "distill_train", "kind": "distill", "grad": True, "dtype": "bf16", "b": 4, "T": 1024, "V": VOCAB, "k": 64,
         "temperature": 2.0, "weight": 0.5, "labels": True, "empty": False},
        # float32, soft targets alone, odd length, teacher rows of different counts
        {"name": "distill_fp32", "kind": "distill", "grad": True, "dtype": "fp32", "b": 1, "T": 777, "V": VOCAB, "k": 20,
         "temperature": 1.0, "weight": 1.0, "labels": False, "empty": True},
    ]


_MOST_LOGITS = {"bf16": 4096 * VOCAB, "fp32": 1500 * VOCAB}


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["embed", "top", "distill"])
    dtype = "fp32" if rng.random() < 0.3 else "bf16"
    V = VOCAB if rng.random() < 0.5 else _spread(rng, 260, 65000)
    if kind == "embed":
        d = rng.choice([64, 128, 512, 1024, 1024, 2048, rng.randint(33, 1500)])
        grad = rng.random() < 0.8
        b = rng.choice([1, 1, 2, 3, 4, 8])
        most = (32768 * 1024 // (2 if dtype == "fp32" else 1)) // max(d, 1024)
        return {"kind": kind, "grad": grad, "dtype": dtype, "b": b, "T": _spread(rng, 1, min(4096, most // b)), "V": V,
                "d": d, "scale": rng.choice([1.0, round(math.sqrt(d), 3)]), "pad": rng.choice([0.0, 0.0, 0.3, 0.7])}
    most = _MOST_LOGITS[dtype] // V
    if kind == "top":
        return {"kind": kind, "dtype": dtype, "rows": _spread(rng, 1, min(4096, most)), "V": V, "k": _spread(rng, 1, 256)}
    b = rng.choice([1, 1, 2, 3, 4])
    weight = rng.choice([1.0, 0.5, 0.9, round(rng.uniform(0.1, 0.95), 3)])
    return {"kind": kind, "grad": rng.random() < 0.75, "dtype": dtype, "b": b, "T": _spread(rng, 1, min(4096, most) // b),
            "V": V, "k": _spread(rng, 1, 128), "temperature": rng.choice([1.0, 2.0, 4.0, round(rng.uniform(0.6, 6.0), 3)]),
            "weight": weight, "labels": weight < 1.0 or rng.random() < 0.5, "empty": rng.random() < 0.4}


# ---- inputs -------------------------------------------------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed * 1000003 + 29)


def _text_tokens(g, V, *shape):
    """Token ids with probability log((i + 4) / (i + 3)) / log((V + 3) / 3): as text has them, the low ids often, most ids
    hardly ever."""
    u = torch.rand(*shape, device=DEV, dtype=torch.float64, generator=g)
    return (3.0 * ((V + 3.0) / 3.0) ** u - 3.0).long().clamp_(0, V - 1)


def _peaked_logits(g, rows, V, tokens, values, dtype):
    """A language model's logits: a broad bulk, and the given tokens at the given values with noise of their own."""
    z = torch.randn(rows, V, device=DEV, generator=g).mul_(2.0)
    z.scatter_(1, tokens, values + torch.randn(values.shape, device=DEV, generator=g))
    return z.to(dtype)


def _teacher(g, rows, V, k):
    """k different tokens a row, their logits falling."""
    step = torch.randint(1, max(2, V // k), (rows, 1), device=DEV, generator=g)
    base = torch.randint(0, V, (rows, 1), device=DEV, generator=g)
    tokens = (base + step * torch.arange(k, device=DEV)) % V
    values = 13.0 - torch.cumsum(torch.rand(rows, k, device=DEV, generator=g) * (16.0 / k), 1)
    return values, tokens


def prepare(case, seed):
    g = _generator(seed)
    dtype = DTYPES[case["dtype"]]
    s = dict(case)
    if case["kind"] == "embed":
        b, T, V, d = case["b"], case["T"], case["V"], case["d"]
        tokens = _text_tokens(g, V, b, T)
        kept = T - int(case["pad"] * T)
        tokens[:, kept:] = V - 1
        s["tokens"] = tokens
        s["table"] = (torch.randn(V, d, device=DEV, generator=g) * 0.02).to(dtype)
        if case["grad"]:
            s["dy"] = (torch.randn(b, T, d, device=DEV, generator=g) * 0.01).to(dtype)
        return s
    if case["kind"] == "top":
        rows, V = case["rows"], case["V"]
        values, tokens = _teacher(g, rows, V, min(24, V))
        s["logits"] = _peaked_logits(g, rows, V, tokens, values, dtype)
        return s
    b, T, V, k = case["b"], case["T"], case["V"], case["k"]
    values, tokens = _teacher(g, b * T, V, k)
    s["logits"] = _peaked_logits(g, b * T, V, tokens[:, :8], values[:, :8], dtype).view(b, T, V)
    if case["empty"]:
        # rows hold any number of targets; the unused slots are marked by a token of -1
        used = torch.randint(0, k + 1, (b * T, 1), device=DEV, generator=g)
        tokens = torch.where(torch.arange(k, device=DEV) < used, tokens, torch.full_like(tokens, -1))
    s["teacher_logits"] = values.to(dtype).view(b, T, k)
    s["teacher_tokens"] = tokens.view(b, T, k)
    s["targets"] = None
    if case["labels"]:
        labels = _text_tokens(g, V, b, T)
        labels[:, T - T // 8:] = IGNORE              # the padded end of a document
        s["targets"] = labels
    return s


# ---- one pass -----------------------------------------------------------------------------------------------------

def run(state):
    if own:
        return _run_own(state)
    return {"embed": _plain_embed, "top": _plain_top, "distill": _plain_distill}[state["kind"]](state)


def _run_own(s):
    from dispatcher_hybrid.fused_vocab import distillation_loss, embed_tokens, top_logits
    if s["kind"] == "top":
        return list(top_logits(s["logits"], s["k"]))
    if s["kind"] == "embed":
        if not s["grad"]:
            with torch.no_grad():
                return [embed_tokens(s["tokens"], s["table"], scale=s["scale"])]
        table = s["table"].detach().requires_grad_()
        y = embed_tokens(s["tokens"], table, scale=s["scale"])
        return [y.detach(), torch.autograd.grad(y, table, s["dy"])[0]]
    z = s["logits"].detach().requires_grad_(s["grad"])
    loss = distillation_loss(z, s["teacher_logits"], s["teacher_tokens"], labels=s["targets"],
                             temperature=s["temperature"], weight=s["weight"],
                             reduction="mean" if s["grad"] else "none")
    if not s["grad"]:
        return [loss]
    return [loss.detach(), torch.autograd.grad(loss, z)[0]]


def _plain_embed(s):
    tokens, table, scale = s["tokens"], s["table"], s["scale"]
    y = (table[tokens].float() * scale).to(table.dtype)
    if not s["grad"]:
        return [y]
    dy = s["dy"].reshape(-1, table.shape[1]).float()
    dt = torch.zeros(table.shape, device=table.device).index_add_(0, tokens.reshape(-1), dy)
    return [y, (dt * scale).to(table.dtype)]


def _plain_top(s):
    z, k = s["logits"], min(s["k"], s["V"])
    # a whole number that orders by value, then by lower index; its k largest are the answer
    bits = (z.float() + 0.0).view(torch.int32)
    order = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long()
    key = order * (1 << 32) + (s["V"] - torch.arange(s["V"], device=z.device))
    tokens = s["V"] - (torch.topk(key, k, dim=1).values & 0xFFFFFFFF)
    return [z.gather(1, tokens), tokens]


def _plain_distill(s):
    V, tau, w = s["V"], s["temperature"], s["weight"]
    z = s["logits"].reshape(-1, V).float()
    n = z.shape[0]
    t = s["teacher_logits"].reshape(n, -1).float() / tau
    tokens = s["teacher_tokens"].reshape(n, -1)
    live = tokens >= 0
    index = tokens.clamp(min=0)
    some = live.any(1, keepdim=True)
    t = torch.where(live, t, torch.full_like(t, -math.inf))
    top = torch.where(some, t.max(1, keepdim=True).values, torch.zeros_like(t[:, :1]))
    e = torch.exp(t - top)
    total = torch.where(some, e.sum(1, keepdim=True), torch.ones_like(t[:, :1]))
    p = e / total
    log_p = t - top - torch.log(total)
    u = (z - z.max(1, keepdim=True).values) / tau
    eu = torch.exp(u)
    su = eu.sum(1, keepdim=True)
    log_q = u.gather(1, index) - torch.log(su)
    rows = w * tau * tau * torch.where(live, p * (log_p - log_q), torch.zeros_like(p)).sum(1)
    kept = torch.ones(n, dtype=torch.bool, device=z.device)
    if s["targets"] is not None:
        labels = s["targets"].reshape(n)
        kept = labels != IGNORE
        label = labels.clamp(min=0).unsqueeze(1)
        c = z - z.max(1, keepdim=True).values
        ec = torch.exp(c)
        sc = ec.sum(1, keepdim=True)
        rows = rows + (1.0 - w) * (torch.log(sc) - c.gather(1, label)).squeeze(1)
    rows = torch.where(kept, rows, torch.zeros_like(rows))
    if not s["grad"]:
        return [rows.view(s["logits"].shape[:-1])]
    count = kept.sum()
    loss = rows.sum() / count
    dz = w * tau * torch.where(some, eu / su, torch.zeros_like(eu))
    dz.scatter_add_(1, index, torch.where(live, -w * tau * p, torch.zeros_like(p)))
    if s["targets"] is not None:
        dz = dz + (1.0 - w) * (ec / sc)
        dz.scatter_add_(1, label, torch.full_like(c[:, :1], w - 1.0))
    dz = torch.where(kept.unsqueeze(1), dz, torch.zeros_like(dz)) / count
    return [loss, dz.to(s["logits"].dtype).view(s["logits"].shape)]


# ---- what a pass cannot do without --------------------------------------------------------------------------------

def _distinct(V, n):
    """Expected number of different ids among n draws of _text_tokens."""
    i = torch.arange(V, dtype=torch.float64)
    p = torch.log((i + 4.0) / (i + 3.0)) / math.log((V + 3.0) / 3.0)
    return float((1.0 - torch.exp(n * torch.log1p(-p))).sum())


def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    V = case["V"]
    if case["kind"] == "embed":
        n, d = case["b"] * case["T"], case["d"]
        rows = _distinct(V, case["b"] * (case["T"] - int(case["pad"] * case["T"]))) + (1 if case["pad"] else 0)
        moved = 8 * n + size * d * (rows + n)
        flops = n * d
        if case["grad"]:
            moved += size * d * (n + V)
            flops += n * d
        return {"bytes": int(moved), "flops": flops}
    if case["kind"] == "top":
        rows, k = case["rows"], min(case["k"], V)
        return {"bytes": rows * (V * size + k * (size + 8)), "flops": rows * V}
    n, k = case["b"] * case["T"], case["k"]
    kept = case["b"] * (case["T"] - case["T"] // 8) if case["labels"] else n
    moved = kept * (V * size + k * (size + 8)) + (8 * n if case["labels"] else 0) + 4 * (1 if case["grad"] else n)
    sums = (2 if case["labels"] and case["temperature"] != 1.0 and case["weight"] > 0 else 1)
    flops = kept * V * (2 + 2 * sums)
    if case["grad"]:
        moved += n * V * size
        flops += kept * V * (2 + 2 * sums)
    return {"bytes": int(moved), "flops": flops}


# ---- the definition in 64 bits ------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    V = case["V"]
    if case["kind"] == "embed":
        table = s["table"].double().requires_grad_(case["grad"])
        y = torch.nn.functional.embedding(s["tokens"], table) * case["scale"]
        if not case["grad"]:
            return [y]
        order = torch.argsort(s["tokens"].reshape(-1), stable=True)
        sums = torch.cat([torch.zeros(1, case["d"], dtype=torch.float64, device=DEV),
                          s["dy"].reshape(-1, case["d"])[order].double().cumsum(0)])
        ends = torch.bincount(s["tokens"].reshape(-1), minlength=V).cumsum(0)
        starts = torch.cat([ends.new_zeros(1), ends[:-1]])
        return [y.detach(), (sums[ends] - sums[starts]) * case["scale"]]
    if case["kind"] == "top":
        # (the values are the inputs' own; the choice itself is a whole number)
        return [torch.sort(s["logits"].double(), dim=1, descending=True).values[:, :min(case["k"], V)], None]
    tau, w = case["temperature"], case["weight"]
    z = s["logits"].double().reshape(-1, V).requires_grad_(case["grad"])
    n = z.shape[0]
    kept = torch.ones(n, dtype=torch.bool, device=DEV) if s["targets"] is None else s["targets"].reshape(n) != IGNORE
    rows = torch.nonzero(kept).squeeze(1)
    tokens = s["teacher_tokens"].reshape(n, -1)[rows]
    live = tokens >= 0
    filled = live.any(1)
    t = s["teacher_logits"].double().reshape(n, -1)[rows] / tau
    log_p = torch.log_softmax(t.masked_fill(~live, -1e30), 1)
    log_q = torch.log_softmax(z[rows] / tau, 1).gather(1, tokens.clamp(min=0))
    soft = (log_p.exp() * (log_p - log_q)).masked_fill(~(live & filled.unsqueeze(1)), 0.0).sum(1)
    loss = w * tau ** 2 * soft
    if s["targets"] is not None:
        picked = torch.log_softmax(z[rows], 1).gather(1, s["targets"].reshape(n)[rows].unsqueeze(1))
        loss = loss - (1.0 - w) * picked.squeeze(1)
    if not case["grad"]:
        return [torch.zeros(n, dtype=torch.float64, device=DEV).index_put((rows,), loss).view(case["b"], case["T"])]
    loss = loss.sum() / rows.numel()
    return [loss.detach(), torch.autograd.grad(loss, z)[0].view(s["logits"].shape)]
