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
