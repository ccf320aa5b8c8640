"""The pages of a cache at the ends of what the calls allow: tables of no columns, rows without a parent, the most pages, none left, caches behind 32 bits."""

import random

import pytest
import torch

from ascendflow_b200 import latent8, ops, pages
from tests import latent8_reference as E
from tests.test_gpu_pages import compacted, counted, equal, forked, i32, resized, same, state_of, tensor

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("blocks", [0, 5])
def test_a_length_behind_a_table_of_no_columns_is_reported(in_place, blocks):
    table, counts, lengths = torch.empty((3, 0), dtype=torch.int32, device="cuda"), i32([0] * blocks), i32([0, 0, 7])
    ops.status()
    got = pages.resize(table, counts, lengths, page_rows=64, out=(table, counts) if in_place else None)
    assert got[0].shape == (3, 0) and torch.equal(got[1], i32([0] * blocks)) and ops.status()[:3] == (1, 2, 7)
    out = (torch.empty((2, 0), dtype=torch.int32, device="cuda"), counts) if in_place else None
    got = pages.fork([], table, counts, i32([2, 0]), lengths, page_rows=64, out=out)
    assert got[0].shape == (2, 0) and torch.equal(got[1], i32([0] * blocks)) and ops.status()[:3] == (1, 2, 7)
    pages.resize(table, counts, i32([0, -4, 0]), page_rows=64, out=(table, counts))
    assert ops.status()[0] == 0


def test_rows_without_a_parent_go_on_as_empty_ones():
    """The lengths that the documentation gives for behind a fork: steps go on, and rows whose parent is no request have no pages and see nothing."""
    table, counts, lengths = i32([[4, 1, -1], [2, -1, -1], [0, 3, -1]]), i32([1] * 5 + [0] * 4), i32([70, 9, 128])
    cache = torch.zeros((9, 64, 1, 576), dtype=torch.uint8, device="cuda").view(E.HELD)
    scales = torch.full((9, 4), 127, dtype=torch.uint8, device="cuda").view(E.SCALE)
    parents = i32([0, -1, 3, 2, 0, -7, 1 << 30])
    table, counts = pages.fork([cache, scales], table, counts, parents, lengths, page_rows=64)
    heirs = (parents >= 0) & (parents < len(lengths))
    lengths = torch.where(heirs, lengths[parents.clamp(0, len(lengths) - 1)], 0)
    assert lengths.tolist() == [70, 0, 0, 128, 70, 0, 0]
    before = table.clone()
    table, counts = pages.resize(table, counts, lengths, page_rows=64)
    assert torch.equal(table, before) and (table[~heirs] == -1).all()
    q = torch.randn((7, 8, 576), device="cuda").bfloat16()
    lse = torch.empty((7, 8), device="cuda")
    out = latent8.latent_attention8(q, cache, scales, table, i32(range(8)), lengths, scale=0.04, lse=lse)
    assert (out == 0).all() and (lse[~heirs] == -float("inf")).all() and torch.isfinite(lse[heirs]).all() and ops.status()[0] == 0


def test_the_last_pages_of_a_large_cache_go_to_the_front_in_order():
    """Pages in use in all eight parts that blocks of threads share out."""
    blocks = pages.MOST_BLOCKS
    used = [7, *(blocks // 8 * k + 11 * k for k in range(1, 8)), blocks - 1]
    counts = torch.zeros(blocks, dtype=torch.int32, device="cuda")
    counts[used] = i32(range(1, 10))
    cache = torch.zeros((blocks, 2), dtype=torch.uint8, device="cuda")
    cache[used, 1] = torch.arange(1, 10, dtype=torch.uint8, device="cuda")
    table, counts, places = pages.compact([cache], i32([used]), counts)
    order = [7, 0, 1, 2, 3, 4, 5, 6, 8]  # page 7 is in front already; the others take the free ones in front, in order
    assert table.tolist() == [order] and places[used].tolist() == order and int((places >= 0).sum()) == 9
    expected = [order.index(p) + 1 for p in range(9)]
    assert counts[:9].tolist() == expected and int((counts != 0).sum()) == 9
    assert cache[:9, 1].tolist() == expected and ops.status()[0] == 0


def test_rows_that_get_no_page_in_a_fork_are_reported():
    requests, entries, blocks, page_rows, children = 9, 3, 12000, 16, 20000
    rng = random.Random(77)
    table, counts, lengths = state_of(rng, requests, entries, blocks, page_rows)
    parents = [rng.randrange(-1, requests) for _ in range(children)]
    expected = forked([], table, counts, parents, lengths, page_rows)
    ops.status()
    got = pages.fork([], tensor(table, entries), i32(counts), i32(parents), i32(lengths), page_rows=page_rows)
    same(got, *expected[:2], entries)
    without = {(r, n - 1) for r, p in enumerate(parents) if p >= 0 and (n := counted(lengths[p], page_rows, entries)) and expected[0][r][n - 1] < 0 <= table[p][n - 1]}
    status = ops.status()
    assert status[0] == 3 and (status[1], status[2]) in without


def test_pages_behind_32_bits():
    """A cache of 5 GB: pages of its end copied there and moved to its front."""
    blocks = 70000
    cache = torch.zeros((blocks, 64, 1152), dtype=torch.uint8, device="cuda")
    own = torch.randint(1, 256, (4, 64, 1152), dtype=torch.uint8, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    cache[blocks - 4 :] = own
    counts = torch.ones(blocks, dtype=torch.int32, device="cuda")  # pages that somebody else keeps, but for four
    counts[[3, 60000, blocks - 6, blocks - 5]] = 0
    table = i32([[blocks - 1, blocks - 2], [blocks - 3, blocks - 4]])
    table, counts = pages.fork([cache], table, counts, i32([0, 0, 1, 1, 1]), i32([64 + 9, 128]), page_rows=64)
    last = [blocks - 1, blocks - 2], [blocks - 3, blocks - 4]
    assert table.tolist() == [last[0], [blocks - 1, 3], last[1], last[1], last[1]]
    assert torch.equal(cache[3, :9], own[2, :9]) and not cache[3, 9:].any() and torch.equal(cache[blocks - 4 :], own)
    table, counts = pages.fork([cache], table, counts, i32([0, 0, 1, 2]), i32([64 + 9, 64 + 9, 0, 0, 0]), page_rows=64)
    assert table.tolist() == [last[0], [blocks - 1, 60000], [blocks - 1, 3], [-1, -1]]
    assert torch.equal(cache[60000, :9], own[2, :9]) and not cache[60000, 9:].any()
    counts[5 : blocks - 8] = 0
    counts[[0, 1, 2, 4]] = 0
    table = torch.where((table >= 5) & (table < blocks - 8), -1, table)
    table, counts, places = pages.compact([cache], table, counts)
    used = [3, blocks - 8, blocks - 7, blocks - 2, blocks - 1]
    assert places[used].tolist() == [3, 0, 1, 2, 4] and int((places >= 0).sum()) == 5
    assert table.tolist() == [[4, 2], [4, -1], [4, 3], [-1, -1]]
    assert torch.equal(cache[2], own[2]) and torch.equal(cache[4], own[3]) and not cache[:2].any() and ops.status()[0] == 0


@pytest.mark.parametrize("requests,children", [(40, 40), (10, 60), (80, 80), (81, 80), (159, 1), (160, 1), (1, 159), (700, 3), (3, 700)])
@pytest.mark.parametrize("tensors", [0, 2])
def test_rows_by_the_plan_and_by_a_kernel_of_their_own(requests, children, tensors):
    """Forks on both sides of the number of rows from which these are the second kernel's, with and without pages to copy."""
    rng, generator = random.Random(requests), torch.Generator(device="cuda").manual_seed(children)
    table, counts, lengths = state_of(rng, requests, 6, 6 * requests + 400, 64)
    caches, parents = [torch.randint(0, 256, (len(counts), 64, 24), dtype=torch.uint8, device="cuda", generator=generator) for _ in range(tensors)], [rng.randrange(-1, requests) for _ in range(children)]
    expected = forked(caches, table, counts, parents, lengths, 64)
    same(pages.fork(caches, tensor(table, 6), i32(counts), i32(parents), i32(lengths), page_rows=64), *expected[:2], 6)
    assert equal(caches, expected[2]) and ops.status()[0] in (0, 3)


@pytest.mark.parametrize("units", [159, 160, 161, 162])
def test_copies_by_the_plan_and_by_a_kernel_of_their_own(units):
    """Calls on both sides of the number of units from which copies are the second kernel's."""
    rng, generator = random.Random(units), torch.Generator(device="cuda").manual_seed(units)

    def cache_of(blocks, rows):
        return torch.randint(0, 256, (blocks, rows, 96), dtype=torch.uint8, device="cuda", generator=generator)

    table, counts, lengths = state_of(rng, 30, 7, 400, 64)
    caches, parents = [cache_of(400, 64)], [rng.randrange(-1, 30) for _ in range(units)]
    expected = forked(caches, table, counts, parents, lengths, 64)
    same(pages.fork(caches, tensor(table, 7), i32(counts), i32(parents), i32(lengths), page_rows=64), *expected[:2], 7)
    assert equal(caches, expected[2])
    table, counts, _ = state_of(rng, 40, 5, 2 * units, 64)
    caches = [cache_of(2 * units, 3)]
    expected = compacted(caches, table, counts)
    got = pages.compact(caches, tensor(table, 5), i32(counts))
    same(got[:2], *expected[:2], 5)
    assert got[2].tolist() == expected[2] and equal(caches, expected[3]) and ops.status()[0] in (0, 3)


@pytest.mark.parametrize("requests,entries", [(1, 2048), (1, 2049), (5, 2049), (32, 2048), (2, 9001)])
@pytest.mark.parametrize("in_place", [False, True])
def test_long_rows_are_resized_by_blocks_of_their_own(requests, entries, in_place):
    """Rows on both sides of the length from which a warp does not go through them alone."""
    rng = random.Random(entries)
    table, counts, lengths = state_of(rng, requests, entries, requests * entries + 9, 16)
    for _ in range(2):
        lengths = [min(max(length + rng.choice([-300, -1, 0, 1, 700, 40000]), 0), 16 * entries) for length in lengths]
        given = tensor(table, entries), i32(counts)
        got = pages.resize(*given, i32(lengths), page_rows=16, out=given if in_place else None)
        table, counts = resized(table, counts, lengths, 16)
        same(got, table, counts, entries)
        assert ops.status()[0] == 0
