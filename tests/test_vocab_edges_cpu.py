"""Corners of the vocabulary-end operators that need no GPU: the formula's rows without a value, the entry points' refusals, the
library and the extension beside it."""

import pytest
import torch

from dispatcher_hybrid import distillation as plain


@pytest.mark.parametrize("weight,with_labels", [(1.0, False), (1.0, True), (0.5, True), (0.0, True)])
def test_a_bad_row_without_live_slots_has_a_gradient_of_nan(weight, with_labels):
    """A token or label past the vocabulary, whatever the row's other slots hold: loss and gradient are NaN together."""
    g = torch.Generator().manual_seed(1)
    z = torch.randn(5, 9, dtype=torch.float64, generator=g)
    t = torch.randn(5, 3, dtype=torch.float64, generator=g)
    tok = torch.tensor([[1, 2, 3], [9, -1, -1], [-1, -1, -1], [9, 2, -1], [-1, -1, -1]])
    labels = torch.tensor([0, 1, 99, 2, 3]) if with_labels else None
    leaf = z.clone().requires_grad_()
    rows = plain.distillation_loss(leaf, t, tok, labels, 2.0, weight, reduction="none")
    grad, = torch.autograd.grad(rows.sum(), leaf)
    bad = [False, weight > 0, with_labels, weight > 0, False]  # (the teacher is not read where weight is 0)
    assert rows.isnan().tolist() == bad
    assert torch.equal(grad.isnan(), torch.tensor(bad).unsqueeze(1).expand(5, 9))
    if weight == 1.0:
        assert rows[4] == 0 and bool((grad[4] == 0).all())
    if with_labels:                                            # an ignored row is not bad
        labels[2] = -100
        rows = plain.distillation_loss(leaf, t, tok, labels, 2.0, weight, reduction="none")
        grad, = torch.autograd.grad(rows.sum(), leaf)
        assert rows[2] == 0 and bool((grad[2] == 0).all()) and bool(rows[1].isnan()) == (weight > 0)


@pytest.mark.parametrize("host", ["/nonexistent/g++", "/bin/false"])
def test_the_kernel_library_is_built_where_the_extension_does_not_compile(host, tmp_path, monkeypatch, capsys):
    """With a stand-in for hipcc that leaves empty outputs: a host compiler that is missing, or one that fails."""
    from dispatcher_hybrid import _build
    hipcc = tmp_path / "hipcc"
    hipcc.write_text('#!/bin/sh\nwhile [ $# -gt 0 ]; do [ "$1" = -o ] && : > "$2"; shift; done\nexit 0\n')
    hipcc.chmod(0o755)
    out = tmp_path / "lib"
    out.mkdir()
    for name, value in (("HIPCC", str(hipcc)), ("OUT_DIR", str(out)), ("LIB", str(out / "lib.so")),
                        ("NODES_LIB", str(out / "nodes.so"))):
        monkeypatch.setattr(_build, name, value)
    (out / "nodes.so").write_text("of other sources")
    monkeypatch.setenv("CXX", host)
    assert _build.build() == str(out / "lib.so")
    assert [f.name for f in out.iterdir()] == ["lib.so"]
    assert "fused_vocab needs it" in capsys.readouterr().err


def test_an_extension_built_for_something_else_is_not_bound(monkeypatch):
    """Another version of the C interface, another torch, one that says neither."""
    from dispatcher_hybrid import _hip, _nodes
    bound = []

    class Loader:
        def __init__(self, *a):
            pass

        def create_module(self, spec):
            return None

        def exec_module(self, module):
            module.bind = lambda *a: bound.append(a)
            for name, value in says.items():
                setattr(module, name, value)
    monkeypatch.setattr(_nodes.importlib.machinery, "ExtensionFileLoader", Loader)
    right = dict(abi_version=_hip.ABI_VERSION, torch_version=str(torch.__version__))
    for says in (dict(right, abi_version=_hip.ABI_VERSION - 1), dict(right, torch_version="1.0"), {}):
        with pytest.raises(ImportError, match="rebuild"):
            _nodes.load(None)
    assert not bound
    says = right
    _nodes.load(None)
    assert len(bound) == 1


def test_the_extension_says_what_it_was_built_for():
    from dispatcher_hybrid import _hip, fused_vocab
    native = fused_vocab._native
    assert (native.abi_version, native.torch_version) == (_hip.ABI_VERSION, str(torch.__version__))


def test_the_loss_entry_points_refuse_results_off_their_elements():
    from dispatcher_hybrid import _hip
    lib, one, N = _hip.lib, 256, None                          # never dereferenced: every call is refused

    def fwd(**kw):
        a = dict(dtype=1, z=one, sb=8, st=8, B=1, T=2, V=8, td=1, tl=one, tt=one, bits=64, K=2, lb=N, lbits=64, ignore=-100,
                 tau=1.0, w=1.0, red=1, rows=one, kept=one, loss=one, div=one, ws=N, nb=0)
        a.update(kw)
        return lib.dh_distill_fwd(*a.values(), N)

    def bwd(**kw):
        a = dict(dtype=1, z=one, sb=8, st=8, B=1, T=2, V=8, td=1, tl=one, tt=one, bits=64, K=2, lb=N, lbits=64, ignore=-100,
                 tau=1.0, w=1.0, kept=one, dl=one, ds=0, div=one, dz=one)
        a.update(kw)
        return lib.dh_distill_bwd(*a.values(), N)
    for kw in (dict(rows=one + 2), dict(loss=one + 1), dict(div=one + 2)):
        assert fwd(**kw) == 1 and b"aligned" in lib.dh_last_error(), kw
    for kw in (dict(dl=one + 2), dict(div=one + 2), dict(dz=one + 1), dict(dtype=0, dz=one + 2)):
        assert bwd(**kw) == 1 and b"aligned" in lib.dh_last_error(), kw
