"""The pages of a cache on the device: `resize` gives requests the pages that they need and takes back the others, `fork` lets rows of the block table continue
others (samples of one prompt, beams in a new order, requests that ended left out), `compact` moves the pages in use to the front.

A block table `[B, PAGES]` int32 names pages of 0 .. BLOCKS - 1, everything else is an empty entry (written as -1); `counts` `[BLOCKS]` int32 says how many entries
name each page, 0 for a free one. A program begins with a table of -1 and counts of 0 and leaves the rest to these calls, between which the attention and append calls use the
table. Results are the same for the same inputs, whatever the timing: the free page of lowest number goes to the first request and entry.

The calls return new tables and counts; with `out=` they write given ones, `counts` in place if that is what is given (and the table too, for `resize` and `compact`).
They launch on torch's current stream and never wait, so a step that includes them may be captured in a CUDA graph (an `out=` of the inputs
makes every replay continue where the last one ended). Reports go to `ops.status()`: 3, request (`fork`: row of the new table), entry where no free page was left (the entry stays empty, and what is appended
there is reported in turn); 1, request, length for a length behind the table. While a graph is traced they are
`torch.ops.ascendflow_b200.pages_resize`, `pages_fork` and `pages_compact`.
"""

from __future__ import annotations

import torch
from torch.compiler import is_compiling

from . import host
from .diagnostics import require
from .latent import _CHECKS, _disjoint, _otherwise, _span, _tensor

MOST_BLOCKS, MOST_CACHES = 1 << 23, 128


def resize(block_table, counts, lengths, *, page_rows, out=None):
    """Request b gets the pages of `lengths[b]` rows: its first ceil(lengths[b] / page_rows) entries keep their page or, where empty, get a free one; the pages of
    its other entries are given back (and free at once, if nobody else has them). Returns (block_table, counts).

    Lengths may grow (a step's new rows, a new prompt), shrink (drafts that were not taken) or be 0 (a request that ended; another may begin there with the next call). Pages stay
    shared: a request that shrinks to less than it had when it was forked, and goes on, is to be forked at that length first.
    """
    given = _given(out)
    if not is_compiling() and (result := _resize(block_table, counts, lengths, page_rows, *given)):
        return result
    outputs = _outputs(given, block_table, counts)
    _otherwise("pages_resize", (block_table, counts, lengths, page_rows, *outputs))
    return outputs


def fork(caches, block_table, counts, parents, lengths, *, page_rows, out=None):
    """A table of len(parents) rows, row i continuing request `parents[i]` of `block_table` at its length `lengths[parents[i]]`. Returns (block_table, counts).

    A request may be continued by any number of rows: they share its full pages, and each but the first has a copy of the partly filled last one, so that all can be appended to (the first
    too, if that page's count is above 1 because others name it). A request that no row continues gives its pages back; a row whose parent is no request (-1) is empty. Only the
    entries that the length counts go on. The new lengths are `lengths[parents]` where every parent is a request; a row without one has length 0:
    `torch.where((parents >= 0) & (parents < B), lengths[parents.clamp(0, B - 1)], 0)`. (As an index -1 is the last request, whose length would be the empty row's, and a number of B or more an error on the device.)
    caches: tensors `[BLOCKS, R, ...]` of any type whose pages the table names, R a divisor of page_rows (a cache of 16 or 8 bits, its scales; of all layers, up to
    128). Their filled rows are copied. The given table is not changed, and `out`'s must not overlap with it.
    """
    given = _given(out)
    if not is_compiling() and (result := _fork(caches, block_table, counts, parents, lengths, page_rows, *given)):
        return result
    require(isinstance(parents, torch.Tensor) and parents.dim() == 1, "parents: expected [N]")
    outputs = _outputs(given, block_table, counts, rows=parents.shape[0])
    _otherwise("pages_fork", (_listed(caches), block_table, counts, parents, lengths, page_rows, *outputs))
    return outputs


def compact(caches, block_table, counts, *, out=None, places=None):
    """The pages in use moved to numbers 0 .. U - 1, of `caches` (tensors `[BLOCKS, ...]`, up to 128) in place: the k-th of those from number U on goes to the k-th free page
    in front. Returns (block_table, counts, places); `places` `[BLOCKS]` int32 has every page's new number, -1 for free pages, for whoever else keeps
    numbers. Pages from U on are free then and may be given back to the system.
    """
    given = _given(out)
    if not is_compiling() and (result := _compact(caches, block_table, counts, *given, places)):
        return result
    outputs = (*_outputs(given, block_table, counts), torch.empty_like(counts) if places is None else places)
    _otherwise("pages_compact", (_listed(caches), block_table, counts, *outputs))
    return outputs


def _given(out):
    require(out is None or isinstance(out, (tuple, list)) and len(out) == 2 and all(t is not None for t in out), "out: expected (block_table, counts)")
    return (None, None) if out is None else tuple(out)


def _outputs(given, block_table, counts, rows=None):
    """Given outputs, or new ones, where the native side does not make them."""
    if given[0] is not None:
        return given
    require(isinstance(block_table, torch.Tensor) and block_table.dim() == 2 and isinstance(counts, torch.Tensor), "block_table, counts: expected [B, PAGES] and [BLOCKS]")
    table = torch.empty_like(block_table) if rows is None else torch.empty((rows, block_table.shape[1]), dtype=block_table.dtype, device=block_table.device)
    return table, torch.empty_like(counts)


def _listed(caches):
    require(isinstance(caches, (tuple, list)), "caches: expected a list of tensors")
    return list(caches)


def _apart(written, other, name):
    """The same memory, or none of it."""
    if written.data_ptr() != other.data_ptr() or written.shape != other.shape:
        _disjoint(written, (other,))


def _check_pages(block_table, counts, page_rows, table_out, counts_out, rows, lengths=None):
    require(isinstance(page_rows, int) and not isinstance(page_rows, bool) and 1 <= page_rows < 1 << 31, "page_rows: expected a number of rows")
    require(isinstance(block_table, torch.Tensor) and block_table.dim() == 2, "block_table: expected [B, PAGES]")
    _tensor(block_table, "block_table", (torch.int32,), block_table.shape)
    require(isinstance(counts, torch.Tensor) and counts.dim() == 1, "counts: expected [BLOCKS]")
    _tensor(counts, "counts", (torch.int32,), counts.shape)
    require(counts.shape[0] <= MOST_BLOCKS, f"counts: expected up to {MOST_BLOCKS} pages")
    _tensor(table_out, "out", (torch.int32,), (rows, block_table.shape[1]))
    require(max(block_table.numel(), table_out.numel(), *block_table.shape) < (1 << 31) - 1, "block_table: too many entries")
    _tensor(counts_out, "out", (torch.int32,), counts.shape)
    if lengths is not None:
        _tensor(lengths, "lengths", (torch.int32,), block_table.shape[:1])
    _apart(counts_out, counts, "counts")
    _disjoint(counts_out, (block_table, table_out, lengths))
    _disjoint(table_out, (counts, lengths))
    _disjoint(counts, (block_table,))


def _check_caches(caches, blocks, page_rows, others):
    require(len(caches) <= MOST_CACHES, f"caches: expected up to {MOST_CACHES} tensors")
    for cache in caches:
        require(isinstance(cache, torch.Tensor), "caches: expected Torch tensors")
        _tensor(cache, "caches", (cache.dtype,))
        require(cache.is_contiguous() and cache.dim() >= 1 + (page_rows is not None) and cache.shape[0] == blocks, "caches: expected contiguous [BLOCKS, ...]")
        if page_rows is not None:
            require(cache.shape[1] >= 1 and page_rows % cache.shape[1] == 0, "caches: expected [BLOCKS, R, ...] with R a divisor of page_rows")
        _disjoint(cache, others)
    spans = sorted(_span(cache) for cache in caches if cache.numel())
    require(all(a[1] <= b[0] for a, b in zip(spans, spans[1:])), "caches: tensors that are written must not overlap others")


def _check_resize(block_table, counts, lengths, page_rows, table_out, counts_out):
    _check_pages(block_table, counts, page_rows, table_out, counts_out, block_table.shape[0], lengths)
    require(isinstance(lengths, torch.Tensor), "lengths: expected a Torch tensor")
    _apart(table_out, block_table, "block_table")


def _check_fork(caches, block_table, counts, parents, lengths, page_rows, table_out, counts_out):
    _tensor(parents, "parents", (torch.int32,), parents.shape)
    require(isinstance(lengths, torch.Tensor), "lengths: expected a Torch tensor")
    _check_pages(block_table, counts, page_rows, table_out, counts_out, parents.shape[0], lengths)
    _disjoint(table_out, (block_table, parents))
    _disjoint(counts_out, (parents,))
    _check_caches(caches, counts.shape[0], page_rows, (block_table, counts, parents, lengths, table_out, counts_out))


def _check_compact(caches, block_table, counts, table_out, counts_out, places):
    _check_pages(block_table, counts, 1, table_out, counts_out, block_table.shape[0])
    _tensor(places, "places", (torch.int32,), counts.shape)
    _apart(table_out, block_table, "block_table")
    _disjoint(places, (block_table, counts, table_out, counts_out))
    _check_caches(caches, counts.shape[0], None, (block_table, counts, table_out, counts_out, places))


_resize, _fork, _compact = host.calls.pages_resize, host.calls.pages_fork, host.calls.pages_compact
_CHECKS.update(pages_resize=_check_resize, pages_fork=_check_fork, pages_compact=_check_compact)
for _name in ("pages_resize", "pages_fork", "pages_compact"):
    torch.library.register_fake(f"ascendflow_b200::{_name}", lambda *arguments: None)
