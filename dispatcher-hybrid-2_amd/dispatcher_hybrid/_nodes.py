"""The C++ side of ``fused_vocab`` and ``fused_logprobs``: launches and autograd nodes over libdh_mixer's entry points
(``csrc/host``).

Bound to the library that ``_hip`` loaded, by address. Loading it raises ImportError if the extension is missing, or was built
for another torch or another version of the library's interface.
"""

import ctypes
import importlib.machinery
import importlib.util
import os

import torch

from . import _hip

_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "_lib", "_vocab_nodes.so")
_ENTRIES = ("dh_embed_fwd", "dh_embed_bwd", "dh_embed_bwd_workspace_bytes", "dh_top_logits", "dh_distill_fwd", "dh_distill_bwd",
            "dh_distill_workspace_bytes", "dh_logprob_fwd", "dh_logprob_bwd", "dh_logprob_workspace_bytes", "dh_preference_fwd",
            "dh_preference_workspace_bytes", "dh_policy_fwd", "dh_policy_workspace_bytes", "dh_head_logprob", "dh_head_logprob_workspace_bytes",
            "dh_last_error")


def load(differentiable):
    """The extension module; `differentiable`: the loss's gradient as torch operations, for create_graph."""
    if not os.path.exists(_PATH):
        raise ImportError(f"{_PATH} not found: build it with `python -m dispatcher_hybrid._build`")
    loader = importlib.machinery.ExtensionFileLoader("_vocab_nodes", _PATH)
    module = importlib.util.module_from_spec(importlib.util.spec_from_loader("_vocab_nodes", loader))
    loader.exec_module(module)
    # (it calls bare addresses: with another interface it would hand the kernels shifted arguments)
    built = getattr(module, "abi_version", None), getattr(module, "torch_version", None)
    if built != (_hip.ABI_VERSION, str(torch.__version__)):
        raise ImportError(f"{_PATH} was built for ABI version {built[0]} and torch {built[1]}, not {_hip.ABI_VERSION} and "
                          f"{torch.__version__}; rebuild it")
    module.bind({name: ctypes.cast(getattr(_hip.lib, name), ctypes.c_void_p).value for name in _ENTRIES}, differentiable)
    return module
