"""A latent cache held in 8 bits: the append of rotated rows to it and attention over it, beside `latent.py`'s for 16 bits.

A cache of `torch.float8_e4m3fn` `[BLOCKS, PAGE_ROWS, 1, W]` goes with scales of `torch.float8_e8m0fnu` `[BLOCKS, PAGE_ROWS / G]`, one for every block of G
rows of a page (the one head that a latent cache has): what a number stands for is its product with its block's scale. G is a power of two up to 64; 1 keeps rows
apart, 64 is what long prompts cost least with. Scales are powers of two, so that the product is exact and nothing is rounded but the stored
number. Pages, tables, lengths and offsets are those of `latent.rotary_append` and `latent.latent_attention`; memory and traffic are half of
theirs.

Calls launch on torch's current stream and never wait, have no gradient, report to `ops.status()`, may be captured in CUDA graphs and traced (they are
then `torch.ops.ascendflow_b200.latent_append8` and `latent_attention8`).
"""

from __future__ import annotations

import torch
from torch.compiler import is_compiling

from . import host
from .diagnostics import CompileError, ErrorKind, require
from .latent import VALUES, _CHECKS, _HALVES, _check_append, _check_attention, _disjoint, _otherwise, _tensor

HELD, SCALE = torch.float8_e4m3fn, torch.float8_e8m0fnu


def rotary_append8(latent, rope, cache, scales, block_table, cu_seqlens_q, seqused_kv, inv_freq, *, layout="interleaved", amplitude=1.0):
    """Write rows `[latent | turned rope]` into the paged `cache` and its `scales` in place; returns both.

    Arguments as `latent.rotary_append`'s; `latent` and `rope` are bf16 or f16, W is a multiple of 16. A block's scale becomes the least power of two s with
    |v| <= 448 s for all its new rows, and not less than it was where rows in front of the new ones share the block: where it grows, their numbers are divided by the growth (exact
    but for subnormal ones). A block that begins with a new row forgets its scale. Rows are worked out in FP32 and rounded once, to nearest. Of f16 rows,
    what is beyond 61440 is held as that (the next number would not fit f16). A row that is not finite makes its block's scale NaN, also for the rows in front of it.
    What a row does to its block stays when the row is given up (a draft that was not taken): scales do not shrink before a new row begins the block. With G = 1 rows do nothing to each other.
    The page of a row that is appended must not be shared with another request (`pages.fork` sees to that).
    """
    halves = _HALVES.get(layout)
    if halves is None:
        raise CompileError("rotary layout is interleaved or half", kind=ErrorKind.UNSUPPORTED)
    arguments = (latent, rope, cache, scales, block_table, cu_seqlens_q, seqused_kv, inv_freq, halves, amplitude)
    if is_compiling() or not _append8(*arguments):
        _otherwise("latent_append8", arguments)
    return cache, scales


def latent_attention8(q, cache, scales, block_table, cu_seqlens_q, seqused_kv, *, scale, sinks=None, out=None, lse=None):
    """Causal attention of q `[T, H, W]` (bf16 or f16), W 512 or 576, over the paged `cache` and its `scales`: returns out `[T, H, 512]` in the type of q.

    As `latent.latent_attention` over a cache that holds the numbers times their scales (in the type of q: for f16 they have to be finite there, and scales up to 2^22).
    In large calls bf16 queries are split into two numbers of 8 bits, which leaves out what is below 2^-21.8 of a row's greatest. What is large is told by the table: its columns are
    the longest that requests may be (or the cache's pages, where those are fewer), so short requests under a wide table are worked out in this way too and have other bits than under a narrow one.
    Rows behind a request's length may hold anything; a number NaN among the others is not looked for, a scale NaN makes what sees its rows NaN and nothing else.
    """
    if out is None:
        require(isinstance(q, torch.Tensor) and q.dim() == 3, "q: expected a [T, H, W] Torch tensor")
        out = torch.empty((*q.shape[:2], VALUES), dtype=q.dtype, device=q.device)
    arguments = (q, cache, scales, block_table, cu_seqlens_q, seqused_kv, scale, sinks, out, lse)
    if is_compiling() or not _attention8(*arguments):
        _otherwise("latent_attention8", arguments)
    return out


def _check_scales(cache, scales, others):
    require(isinstance(scales, torch.Tensor) and scales.dim() == 2 and scales.shape[1] >= 1 and cache.shape[1] % scales.shape[1] == 0
            and cache.shape[1] // scales.shape[1] in (1, 2, 4, 8, 16, 32, 64),
            "scales: expected [BLOCKS, PAGE_ROWS / G] with G a power of two up to 64")
    _tensor(scales, "scales", (SCALE,), (cache.shape[0], scales.shape[1]))
    _disjoint(scales, others)


def _check_append8(latent, rope, cache, scales, block_table, cu_seqlens_q, seqused_kv, inv_freq, halves, amplitude):
    _check_append(latent, rope, cache, block_table, cu_seqlens_q, seqused_kv, inv_freq, halves, amplitude, HELD)
    require(cache.shape[3] % 16 == 0, "cache: rows must be a multiple of 16 features")
    require(block_table.shape[0] <= 1 << 26, "block_table: too many requests")
    _check_scales(cache, scales, (latent, rope, cache, block_table, cu_seqlens_q, seqused_kv, inv_freq))


def _check_attention8(q, cache, scales, block_table, cu_seqlens_q, seqused_kv, scale, sinks, out, lse):
    _check_attention(q, cache, block_table, cu_seqlens_q, seqused_kv, scale, sinks, out, lse, HELD)
    _check_scales(cache, scales, (out, lse))


_append8, _attention8 = host.calls.latent_append8, host.calls.latent_attention8
_CHECKS.update(latent_append8=_check_append8, latent_attention8=_check_attention8)
for _name in ("latent_append8", "latent_attention8"):
    torch.library.register_fake(f"ascendflow_b200::{_name}", lambda *arguments: None)
