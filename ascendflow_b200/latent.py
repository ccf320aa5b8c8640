"""Operators around dense latent attention, for the layers and contexts where every cached row is attended to.

`rotary` turns the rope part of queries, `rotary_append` puts a step's new rows (their rope part turned on the way)
into the paged cache, `latent_attention` attends to that cache in absorbed form (one row per token is key and value
of all heads: single tokens, drafts, short chunks), `latent_prefill` computes prompts in expanded form (keys and
values per head and one shared rope key per token). The reference leaves all four to its caller
(`docs/operators/sparse-mla.md:8, 263-266`); next to its operator they make the dense layers of the same models.

All launch on torch's current stream and never wait. They have no gradient and refuse tensors that want one. What a
launch has to report (a block-table entry outside of the cache) is read with `ops.status()`, as for `ops.sparse_mla`.
A call normally stays in native code (`csrc/latent_calls.cpp`); what that refuses, and the first call of a process, comes
back here, where the violated rule is put into words. Nothing is ever cast, copied or padded implicitly.

While a graph is traced (`torch.compile`, `torch.export`, fake tensors, any dispatch mode) the functions call the registered ops of the same work,
`torch.ops.ascendflow_b200.rotary` and so on, which write outputs that are given.
"""

from __future__ import annotations

import math
import numbers

import torch
from torch.autograd import forward_ad
from torch.compiler import is_compiling
from torch.utils._python_dispatch import _get_current_dispatch_mode

from . import host
from .diagnostics import CompileError, ErrorKind, require

VALUES, NOPE, ROPE, MOST_PAIRS, MOST_ROWS = 512, 128, 64, 128, 1 << 30
MOST_FLOAT = torch.finfo(torch.float32).max
_HALVES = {"interleaved": False, "half": True}
_STORED = (torch.bfloat16, torch.float16)


def rotary_frequencies(dims, *, base=10000.0, scaling="none", factor=1.0, original_length=4096, beta_fast=32.0, beta_slow=1.0,
                       device="cuda"):
    """Radians per position of each of `dims / 2` pairs, float64: `base ** (-2 i / dims)`, and for contexts `factor` times the trained one

    "linear"  divided by the factor (positions are interpolated);
    "ntk"     with the base grown so that the slowest pair is divided by the factor and the fastest is left;
    "yarn"    pairs that turn less than `beta_slow` times within `original_length` positions divided by the factor, those that turn
              more than `beta_fast` times left, a ramp between; `rotary_amplitude(factor)` goes with it, see there.

    What a program keeps: computed once, on the host.
    """
    require(isinstance(dims, int) and dims >= 2 and dims % 2 == 0, "rotary dims must be an even number of features")
    require(base > 1 and factor >= 1, "rotary base must be above 1 and factor at least 1")
    half = dims // 2
    exponent = torch.arange(half, dtype=torch.float64) / half
    if scaling == "ntk" and half > 1:
        base = base * factor ** (half / (half - 1))
    plain = float(base) ** -exponent
    if scaling in ("none", "ntk"):
        return plain.to(device)
    if scaling == "linear":
        return (plain / factor).to(device)
    require(scaling == "yarn", "rotary scaling is one of none, linear, ntk, yarn", kind=ErrorKind.UNSUPPORTED)
    require(beta_fast > beta_slow > 0 and original_length > 0, "yarn needs beta_fast above beta_slow above 0 and an original length")

    def pair_of(turns):  # the pair that turns so many times within the original length
        return half * math.log(original_length / (turns * 2 * math.pi)) / math.log(base)

    # (the ramp may end behind the last pair, which then is on it; it is bounded by the number of features, as published)
    low, high = max(math.floor(pair_of(beta_fast)), 0), min(math.ceil(pair_of(beta_slow)), dims - 1)
    ramp = ((torch.arange(half, dtype=torch.float64) - low) / max(high - low, 1e-3)).clamp(0, 1)
    return (plain * (1 - ramp) + plain / factor * ramp).to(device)


def rotary_amplitude(factor, mscale=1.0):
    """The amplitude that goes with "yarn" stretching a context `factor` times: scores are to grow by its square.

    Where a head is turned as a whole, it is the `amplitude` of queries and keys. Where only a part is (64 of 192 or 576 features here) that would leave the
    other features' scores as they were: the turn's amplitude stays 1, and its square goes into the attention call's `scale`.
    """
    return 1.0 if factor <= 1 else 0.1 * mscale * math.log(factor) + 1.0


def rotary(x, positions, inv_freq, *, layout="interleaved", inverse=False, amplitude=1.0, out=None):
    """`x` `[T, H, D]` or `[T, D]` (bf16, f16, f32; strided rows) with the last `2 len(inv_freq)` features of every head turned by
    `positions[t] * inv_freq[i]` radians and multiplied by `amplitude`; the features in front are copied.

    layout: pair i is features (2 i, 2 i + 1) of the turned part ("interleaved") or (i, i + len(inv_freq)) ("half").
    inverse: turned back (an attention output whose rows carried positions). out: allocated when None; `x` itself for a turn in place.
    positions: int32 or int64, any value; inv_freq: float64, see `rotary_frequencies`.
    """
    halves = _HALVES.get(layout)
    if halves is None:
        raise CompileError("rotary layout is interleaved or half", kind=ErrorKind.UNSUPPORTED)
    if out is None:
        require(isinstance(x, torch.Tensor), "x: expected a Torch tensor")
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    arguments = (x, positions, inv_freq, halves, inverse, amplitude, out)
    if is_compiling() or not _rotary(*arguments):
        _otherwise("rotary", arguments)
    return out


def rotary_append(latent, rope, cache, block_table, cu_seqlens_q, seqused_kv, inv_freq, *, layout="interleaved", amplitude=1.0):
    """Write rows `[latent | turned rope]` into the paged `cache` `[BLOCKS, PAGE_ROWS, 1, W]` in place; returns it.

    latent `[T, W - 2 len(inv_freq)]`, rope `[T, 2 len(inv_freq)]` (both may be slices of a wider projection). Row j of the n of
    request b goes to position `seqused_kv[b] - n + j`, which is also what its rope part is turned by (`seqused_kv` counts the new rows,
    as it does for the attention call that follows). Unlike `neighbours.cache_append` it does not wait: a row without a legal page
    is not written and reported in `ops.status()`. Rows behind the last request are left out.
    """
    halves = _HALVES.get(layout)
    if halves is None:
        raise CompileError("rotary layout is interleaved or half", kind=ErrorKind.UNSUPPORTED)
    arguments = (latent, rope, cache, block_table, cu_seqlens_q, seqused_kv, inv_freq, halves, amplitude)
    if is_compiling() or not _latent_append(*arguments):
        _otherwise("latent_append", arguments)
    return cache


def latent_attention(q, cache, block_table, cu_seqlens_q, seqused_kv, *, scale, sinks=None, out=None, lse=None):
    """Causal attention of q `[T, H, W]` over the paged `cache` `[BLOCKS, PAGE_ROWS, 1, W]`, W 512 or 576: returns out `[T, H, 512]`.

    Scores are `scale * q . row`, values the first 512 features of the same row. Token j of the n of request b sees the first
    `seqused_kv[b] - n + j + 1` rows of its request. sinks `[H]` float32: a logit per head in the denominator. lse `[T, H]` float32,
    written when given: the natural logarithm of the denominator. A token that sees nothing gets zeros (and -inf, or its sink);
    tokens behind the last request are left as they were. A page outside of the cache is masked and reported in `ops.status()`.
    Cache rows behind a request's length may hold anything; those within it have to be finite.
    """
    if out is None:
        require(isinstance(q, torch.Tensor) and q.dim() == 3, "q: expected a [T, H, W] Torch tensor")
        out = torch.empty((*q.shape[:2], VALUES), dtype=q.dtype, device=q.device)
    arguments = (q, cache, block_table, cu_seqlens_q, seqused_kv, scale, sinks, out, lse)
    if is_compiling() or not _latent_attention(*arguments):
        _otherwise("latent_attention", arguments)
    return out


def latent_prefill(q, k, v, k_rope, cu_seqlens_q, cu_seqlens_k, *, scale, causal=True, out=None, lse=None):
    """Attention of ragged prompts in expanded form: q `[T, H, 192]`, k and v `[S, H, 128]`, k_rope `[S, 64]`; returns out `[T, H, 128]`.

    A head's key is `[k | k_rope]`. Request b owns queries `cu_seqlens_q[b]..` and keys `cu_seqlens_k[b]..`; causal: token j of n sees the
    first K - n + j + 1 of its K keys (a chunk behind a context has more keys than queries), otherwise all K. q, k, v and k_rope
    may be strided (k and v halves of one projection). lse, rows that see nothing and rows behind the last request: as in `latent_attention`. Values of a request
    have to be finite, those of keys that a token does not see yet too (their weights of zero are multiplied); what lies outside of the requests may be anything.
    """
    if out is None:
        require(isinstance(q, torch.Tensor) and q.dim() == 3, "q: expected a [T, H, 192] Torch tensor")
        out = torch.empty((*q.shape[:2], NOPE), dtype=q.dtype, device=q.device)
    arguments = (q, k, v, k_rope, cu_seqlens_q, cu_seqlens_k, scale, causal, out, lse)
    if is_compiling() or not _latent_prefill(*arguments):
        _otherwise("latent_prefill", arguments)
    return out


def _otherwise(name, arguments):
    """A call while a graph is traced (or a dispatch mode looks on), which is the registered op's, or one that the native side refused."""
    if is_compiling() or _get_current_dispatch_mode() is not None or any(_traced(argument) for argument in arguments):
        getattr(torch.ops.ascendflow_b200, name)(*arguments)
    else:
        _checked(name, *arguments)


def _traced(argument):
    """A tensor that stands for another or for none, as in tracing."""
    return isinstance(argument, torch.Tensor) and type(argument).__torch_dispatch__ is not torch.Tensor.__torch_dispatch__


def _checked(name, *arguments):
    """A refused call: the rule that it violates, or (the first call of a process) a second attempt with the entry points at hand."""
    _CHECKS[name](*arguments)
    host.connect_latent()
    require(getattr(host.calls, name)(*arguments), "call refused by the native host side")


def _tensor(tensor, name, dtypes, shape=None):
    require(type(tensor) in (torch.Tensor, torch.nn.Parameter), f"{name}: expected a Torch tensor")
    require(tensor.is_cuda and tensor.layout == torch.strided, f"{name}: expected a CUDA tensor")
    require(tensor.dtype in dtypes, f"{name}: expected {' or '.join(map(str, dtypes))}")
    require(not tensor.is_conj() and not tensor.is_neg(), f"{name}: lazily negated tensors are not supported")
    wanted = tensor.requires_grad and torch.is_grad_enabled() or forward_ad.unpack_dual(tensor).tangent is not None
    require(not wanted, f"{name}: the operator has no gradient", kind=ErrorKind.UNSUPPORTED)
    require(tensor.device.index == torch.cuda.current_device(), f"{name}: expected a tensor on the current CUDA device")
    if shape is not None:
        require(tuple(tensor.shape) == tuple(shape), f"{name}: expected shape {list(shape)}")
        require(tensor.is_contiguous(), f"{name}: expected contiguous tensor storage")


def _rows(tensor, name):
    """Rows that 16-byte loads can take: features follow each other, rows start on 16-byte boundaries."""
    if tensor.numel() == 0:
        return
    strides = [s for n, s in zip(tensor.shape[:-1], tensor.stride()[:-1]) if n > 1]
    require((tensor.shape[-1] <= 1 or tensor.stride(-1) == 1) and tensor.data_ptr() % 16 == 0
            and all(s * tensor.element_size() % 16 == 0 for s in strides),
            f"{name}: features must be contiguous and rows start on 16-byte boundaries")


def _span(tensor):
    if tensor.numel() == 0:
        return 0, 0
    last = sum((n - 1) * s for n, s in zip(tensor.shape, tensor.stride()))
    return tensor.data_ptr(), tensor.data_ptr() + (last + 1) * tensor.element_size()


def _disjoint(written, others):
    first, last = _span(written)
    for other in others:
        if other is not None:
            begin, end = _span(other)
            require(begin == end or first == last or end <= first or last <= begin, "tensors that are written must not overlap others")


def _number(value, name, least, most):
    require(isinstance(value, numbers.Real) and least <= value <= most, f"{name}: expected a finite number from {least:g} to {most:g}")


def _check_frequencies(inv_freq):
    _tensor(inv_freq, "inv_freq", (torch.float64,))
    require(inv_freq.dim() == 1 and inv_freq.is_contiguous() and 8 <= inv_freq.shape[0] <= MOST_PAIRS and inv_freq.shape[0] % 8 == 0,
            f"inv_freq: expected a multiple of 8 up to {MOST_PAIRS} frequencies")


def _check_rotary(x, positions, inv_freq, halves, inverse, amplitude, out):
    _number(amplitude, "amplitude", -MOST_FLOAT, MOST_FLOAT)
    require(isinstance(inverse, bool), "inverse: expected True or False")
    for tensor, name in ((x, "x"), (out, "out")):
        _tensor(tensor, name, (*_STORED, torch.float32))
        require(tensor.dim() in (2, 3), f"{name}: expected [T, H, D] or [T, D]")
        _rows(tensor, name)
    require(out.shape == x.shape and out.dtype == x.dtype, "out: expected the shape and type of x")
    _tensor(positions, "positions", (torch.int32, torch.int64), x.shape[:1])
    _check_frequencies(inv_freq)
    require(x.shape[-1] % 8 == 0 and 2 * inv_freq.shape[0] <= x.shape[-1] <= 65536, "x: features must be a multiple of 8, and hold the turned part")
    require(x.shape[1:-1].numel() <= 65536 and x.shape[:-1].numel() <= MOST_ROWS, "x: too many rows")
    extent = 1
    for stride, size in sorted((s, n) for n, s in zip(out.shape, out.stride()) if n > 1):
        require(stride >= extent, "out: entries share memory")
        extent += stride * (size - 1)
    same = all(a == b for n, a, b in zip(x.shape, x.stride(), out.stride()) if n > 1)
    _disjoint(out, (positions, inv_freq) + (() if x.data_ptr() == out.data_ptr() and same else (x,)))


def _check_paged(cache, block_table, cu_seqlens_q, seqused_kv, dtype):
    _tensor(cache, "cache", (dtype,))
    require(cache.dim() == 4 and cache.shape[2] == 1 and cache.is_contiguous() and cache.shape[1] >= 64 and cache.shape[1] % 64 == 0,
            "cache: expected contiguous [BLOCKS, PAGE_ROWS, 1, W] with pages of a multiple of 64 rows")
    _rows(cache, "cache")
    require(isinstance(block_table, torch.Tensor) and block_table.dim() == 2, "block_table: expected [B, PAGES]")
    batches, pages = block_table.shape
    _tensor(block_table, "block_table", (torch.int32,), (batches, pages))
    require(max(cache.shape[0], pages) * cache.shape[1] < (1 << 31) - 128, "cache and block_table: positions must fit 31 bits")
    _tensor(cu_seqlens_q, "cu_seqlens_q", (torch.int32,), (batches + 1,))
    _tensor(seqused_kv, "seqused_kv", (torch.int32,), (batches,))


def _check_append(latent, rope, cache, block_table, cu_seqlens_q, seqused_kv, inv_freq, halves, amplitude, held=None):
    _number(amplitude, "amplitude", -MOST_FLOAT, MOST_FLOAT)
    for tensor, name in ((latent, "latent"), (rope, "rope")):
        _tensor(tensor, name, _STORED)
        require(tensor.dim() == 2, f"{name}: expected [T, features]")
    _rows(latent, "latent")
    require(rope.dtype == latent.dtype and (rope.numel() == 0 or rope.stride(1) == 1), "rope: expected the type of latent and contiguous features")
    _check_paged(cache, block_table, cu_seqlens_q, seqused_kv, held or latent.dtype)
    _check_frequencies(inv_freq)
    turned = 2 * inv_freq.shape[0]
    require(tuple(rope.shape) == (latent.shape[0], turned) and latent.shape[1] + turned == cache.shape[3], "expected latent [T, W - R], rope [T, R] and cache rows of W")
    require(cache.shape[3] % 8 == 0 and cache.shape[3] <= 65536 and latent.shape[0] <= MOST_ROWS, "cache: rows must be a multiple of 8 features")
    _disjoint(cache, (latent, rope, block_table, cu_seqlens_q, seqused_kv, inv_freq))


def _check_written(out, lse, inputs):
    _disjoint(out, (*inputs, lse))
    if lse is not None:
        _disjoint(lse, inputs)


def _check_attention(q, cache, block_table, cu_seqlens_q, seqused_kv, scale, sinks, out, lse, held=None):
    _number(scale, "scale", 1e-30, 1e30)
    _tensor(q, "q", _STORED)
    require(q.dim() == 3 and q.shape[2] in (512, 576) and q.shape[1] >= 1 and q.is_contiguous(), "q: expected contiguous [T, H, 512] or [T, H, 576]")
    require(q.shape[:2].numel() <= MOST_ROWS, "q: too many rows")
    _rows(q, "q")
    _check_paged(cache, block_table, cu_seqlens_q, seqused_kv, held or q.dtype)
    require(cache.shape[3] == q.shape[2], "cache: rows must be as wide as q")
    _tensor(out, "out", (q.dtype,), (*q.shape[:2], VALUES))
    _rows(out, "out")
    if sinks is not None:
        _tensor(sinks, "sinks", (torch.float32,), q.shape[1:2])
    if lse is not None:
        _tensor(lse, "lse", (torch.float32,), q.shape[:2])
    _check_written(out, lse, (q, cache, block_table, cu_seqlens_q, seqused_kv, sinks))


def _check_prefill(q, k, v, k_rope, cu_seqlens_q, cu_seqlens_k, scale, causal, out, lse):
    _number(scale, "scale", 1e-30, 1e30)
    require(isinstance(causal, bool), "causal: expected True or False")
    _tensor(q, "q", _STORED)
    require(q.dim() == 3 and q.shape[2] == NOPE + ROPE and 1 <= q.shape[1] <= 65535, "q: expected [T, H, 192]")
    require(isinstance(k, torch.Tensor) and k.dim() == 3, "k: expected [S, H, 128]")
    keys, heads = k.shape[0], q.shape[1]
    for tensor, name, shape in ((q, "q", q.shape), (k, "k", (keys, heads, NOPE)), (v, "v", (keys, heads, NOPE)), (k_rope, "k_rope", (keys, ROPE))):
        _tensor(tensor, name, (q.dtype,))
        require(tuple(tensor.shape) == tuple(shape), f"{name}: expected shape {list(shape)}")
        _rows(tensor, name)
        require(tensor.shape[0] <= 1 or tensor.stride(0) > 0, f"{name}: tokens must not share memory")
    require(q.shape[:2].numel() <= MOST_ROWS and keys <= MOST_ROWS, "too many rows")
    require(isinstance(cu_seqlens_q, torch.Tensor) and cu_seqlens_q.dim() == 1 and cu_seqlens_q.shape[0] >= 1, "cu_seqlens_q: expected [B + 1]")
    require((q.shape[0] // 256 + cu_seqlens_q.shape[0] - 1) * heads < 1 << 31, "too many requests and heads")
    for tensor, name in ((cu_seqlens_q, "cu_seqlens_q"), (cu_seqlens_k, "cu_seqlens_k")):
        _tensor(tensor, name, (torch.int32,), cu_seqlens_q.shape)
    _tensor(out, "out", (q.dtype,), (*q.shape[:2], NOPE))
    _rows(out, "out")
    if lse is not None:
        _tensor(lse, "lse", (torch.float32,), q.shape[:2])
    _check_written(out, lse, (q, k, v, k_rope, cu_seqlens_q, cu_seqlens_k))


# `torch.ops.ascendflow_b200.rotary`, `.latent_append`, `.latent_attention` and `.latent_prefill` are registered by the native module when it is loaded: no result,
# outputs mutated, CUDA only, no gradient. Tracing needs nothing computed.
_CHECKS = {"rotary": _check_rotary, "latent_append": _check_append, "latent_attention": _check_attention, "latent_prefill": _check_prefill}
_rotary, _latent_append, _latent_attention, _latent_prefill = (getattr(host.calls, name) for name in _CHECKS)
host.calls.set_latent_fallback(_checked)
for _name in _CHECKS:
    torch.library.register_fake(f"ascendflow_b200::{_name}", lambda *arguments: None)
