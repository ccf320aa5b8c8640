"""The pages of a cache at the ends of what the calls allow."""

import pytest
import torch

from ascendflow_b200 import ops, pages
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
