"""The pages of a cache at the ends of what the calls allow."""

import pytest
import torch

from ascendflow_b200 import latent8, ops, pages
from tests import latent8_reference as E
from tests.test_gpu_pages import i32

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
