"""Loads the native host side (`csrc/host_calls.cpp`): the calls' checks and launches in C++, and the
registered torch op.

`calls` is the module. Its functions launch what they accept and say so; what they refuse has not
been enqueued, and the Python front end (`runtime/`) finds out why. Until `connect()` has given
it the kernel library's entry points it refuses everything, so that the first call of a process goes
through the front end, which builds or verifies that library.

Where the module cannot be had (a torch without CUDA, no compiler) the package still imports and traces:
a stand-in refuses everything, and `connect()`, on the way of every call with CUDA tensors, says why.
"""

from __future__ import annotations

import ctypes as ct
import functools
import importlib.machinery
import importlib.util
import numbers

import torch  # noqa: F401  (its libraries are what the module links against)

from .build import build_host_library
from .diagnostics import CompileError


def _load():
    path = build_host_library()
    loader = importlib.machinery.ExtensionFileLoader("_host_calls", str(path))
    module = importlib.util.module_from_spec(importlib.util.spec_from_loader("_host_calls", loader))
    loader.exec_module(module)
    return module


class _Unavailable:
    """Refuses every call; registers the op for tracing, with calls that go through the front end."""

    def __init__(self, error):
        self.error = error

    def configure(self, attention, select, append, fallback):
        if not hasattr(self, "registration"):
            self.registration = torch.library.Library("ascendflow_b200", "DEF")
            self.registration.define(SCHEMA, tags=(torch.Tag.pt2_compliant_tag,))
            self.registration.impl("sparse_mla", fallback, "CUDA")

    def sparse_mla(self, *tensors):
        return False

    def topk_indices(self, *arguments):
        return None

    def cache_append(self, *arguments):
        return None

    def rotary(self, *arguments):
        return False

    latent_append = latent_attention = latent_prefill = rotary

    def set_latent_fallback(self, fallback):
        self.latent_registration = torch.library.Library("ascendflow_b200", "FRAGMENT")
        for schema in LATENT_SCHEMAS:
            name = schema[: schema.index("(")]
            self.latent_registration.define(schema, tags=(torch.Tag.pt2_compliant_tag,))
            self.latent_registration.impl(name, functools.partial(fallback, name), "CUDA")

    def read_status(self):
        raise RuntimeError("the native host side is not available") from self.error

    def release_workspaces(self):
        pass


SCHEMA = ("sparse_mla(Tensor q, Tensor ori_kv, Tensor cmp_kv, Tensor cmp_sparse_indices, Tensor ori_block_table, "
          "Tensor cmp_block_table, Tensor cu_seqlens_q, Tensor seqused_ori_kv, Tensor seqused_cmp_kv, "
          "Tensor cmp_residual_kv, Tensor ori_topk_length, Tensor sinks, Tensor(a12!) attention_out) -> ()")
LATENT_SCHEMAS = (
    "rotary(Tensor x, Tensor positions, Tensor inv_freq, bool halves, bool inverse, float amplitude, Tensor(a!) out) -> ()",
    "latent_append(Tensor latent, Tensor rope, Tensor(a!) cache, Tensor block_table, Tensor cu_seqlens_q, Tensor seqused_kv, Tensor inv_freq, bool halves, "
    "float amplitude) -> ()",
    "latent_attention(Tensor q, Tensor cache, Tensor block_table, Tensor cu_seqlens_q, Tensor seqused_kv, float scale, Tensor? sinks, Tensor(a!) out, "
    "Tensor(b!)? lse) -> ()",
    "latent_prefill(Tensor q, Tensor k, Tensor v, Tensor k_rope, Tensor cu_seqlens_q, Tensor cu_seqlens_k, float scale, bool causal, Tensor(a!) out, "
    "Tensor(b!)? lse) -> ()",
)

try:
    calls = _load()
except (CompileError, ImportError, OSError) as error:
    calls = _Unavailable(error)
_fallback = None
_connected = False
_latent_connected = False


def set_fallback(function):
    """The front end's call for what the registered op refuses."""
    global _fallback, _connected
    _fallback = function
    calls.configure(0, 0, 0, function)
    _connected = False  # the neighbouring steps may have handed the entry points over before this was imported


def connect():
    """Hand the verified kernel library's entry points over, once; true when they were not there before."""
    global _connected
    if _connected:
        return False
    if isinstance(calls, _Unavailable):
        raise RuntimeError("the native host side is not available") from calls.error
    from .build import library_path
    from .runtime.torch import _library

    library = _library(library_path())
    addresses = (ct.cast(getattr(library, name), ct.c_void_p).value for name in (
        "launch_sparse_mla_kept_status", "launch_sparse_mla_topk_indices", "launch_sparse_mla_cache_append_flagged"))
    calls.configure(*addresses, _fallback)
    _connected = True
    return True


def connect_latent():
    """The same for the operators around dense latent attention."""
    global _latent_connected
    if _latent_connected:
        return False
    if isinstance(calls, _Unavailable):
        raise RuntimeError("the native host side is not available") from calls.error
    from .build import library_path
    from .runtime.torch import _library

    library = _library(library_path())
    calls.configure_latent(*(ct.cast(getattr(library, name), ct.c_void_p).value for name in (
        "launch_latent_rotary", "launch_latent_append", "launch_latent_attention", "launch_latent_prefill", "workspace_size_latent_attention",
        "workspace_size_latent_prefill")), numbers.Real)
    _latent_connected = True
    return True
