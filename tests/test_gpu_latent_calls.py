"""How the calls around dense latent attention treat what they are given: places in the cache, numbers, versions, tangents, empty and very wide calls, threads."""

import threading

import numpy as np
import pytest
import torch

from ascendflow_b200 import latent, ops
from ascendflow_b200.diagnostics import CompileError
from tests import latent_reference as R

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def normal(seed, *shape, dtype=BF16):
    return torch.randn(shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(dtype)


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("starts,counts", [([0, 5], [3]), ([0, 2, 7], [2, 1]), ([-4, 2, 3], [2, 1]), ([-9, -1, 1 << 30], [0, 3])])
def test_append_puts_rows_where_attention_reads_them(starts, counts):
    """Offsets outside of the tokens are clamped: the last rows of a request are its last tokens, for the append as for the attention call behind it."""
    lengths = [130, 70][: len(counts)]
    rows, rope, inv_freq = normal(1, 3, 512), normal(2, 3, 64), latent.rotary_frequencies(64)
    cache, table = normal(3, 6, 64, 1, 576), i32([[4, 0, 2], [1, 3, 5]][: len(counts)])
    expected = R.append(rows, rope, cache, table, counts, lengths, inv_freq, "interleaved")
    clamped = cache.clone()
    ops.status()
    latent.rotary_append(rows, rope, cache, table, i32(starts), i32(lengths), inv_freq)
    assert ops.status()[0] == 0
    R.within(cache, expected, R.HALF_STEP[BF16] * expected.abs() + 16 * 2.0 ** -24 * 8, "cache")
    latent.rotary_append(rows, rope, clamped, table, i32([min(max(s, 0), 3) for s in starts]), i32(lengths), inv_freq)
    assert torch.equal(cache, clamped)
