"""Attention over a latent cache in 8 bits at the ends of what queries, scales and masks may be, against the definition in 64 bits."""

import math

import pytest
import torch

from ascendflow_b200 import latent8, ops
from tests import latent8_reference as E
from tests import latent_reference as R
from tests.test_gpu_latent8 import held, i32, large, normal, starts, tables

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16
FORMS = [(BF16, False), (BF16, True), (F16, False)]  # type of the queries; worked out the other way round


def pages_for(seed, counts, lengths, heads, turned, page_rows=64):
    """A table, as wide as the other way round asks for, and the number of pages."""
    table, blocks = tables(seed, lengths, page_rows)
    if turned:
        wide = large(heads, sum(counts), table, page_rows)
        blocks = max(blocks, wide)
        table = torch.cat([table, torch.full((len(table), max(wide - table.shape[1], 0)), -1, dtype=torch.int32, device="cuda")], 1)
    return table, blocks


def attend(q, cache, scales, table, counts, lengths, scale, sinks=None):
    lse = torch.full(q.shape[:2], 7.0, device="cuda")
    out = latent8.latent_attention8(q, cache, scales, table, starts(counts), i32(lengths), scale=scale, sinks=sinks, lse=lse)
    assert ops.status()[0] == 0
    return out, lse


def check(got, q, cache, scales, table, counts, lengths, scale, turned, sinks=None):
    wide, token, page_rows = E.values(cache, scales), 0, cache.shape[1]
    for b, (n, length) in enumerate(zip(counts, lengths)):
        own = wide[table[b, : -(-length // page_rows)].long()].view(1, -1, q.shape[2])[:, :length]
        seen = torch.arange(length, device="cuda") < (length - n + 1 + torch.arange(n, device="cuda"))[:, None]
        queries = q[token : token + n]
        expected, expected_lse, error, lse_error = R.attention(queries, own, own[..., :512], seen, scale, sinks)
        if turned and length:
            # Two numbers of 8 bits hold a query to 2^-14 of 2^e, its scale, with 224 < |q| / 2^e <= 448 and e >= -126: 2^-14 / 224 < 1.5 * 2^-22 of its greatest, or of 2^-118.
            greatest = queries.double().abs().amax(-1, keepdim=True).clamp(min=2.0 ** -118)
            split = 1.5 * 2.0 ** -22 * scale * greatest * own.abs().sum(-1).amax()
            error, lse_error = error + 2 * split * own[..., :512].abs().amax(), lse_error + split[..., 0]
        R.within(got[0][token : token + n], expected, error, f"request {b}")
        R.within(got[1][token : token + n], expected_lse, lse_error, f"request {b}, lse")
        token += n


# ---- sizes of queries -----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,turned", FORMS)
@pytest.mark.parametrize("width,block", [(576, 16), (512, 1)])
@pytest.mark.parametrize("with_sinks", [False, True])
def test_rows_of_zeros_and_of_tiny_numbers(dtype, turned, width, block, with_sinks):
    """As warm-up calls and padded batches have them; beside ordinary rows of the same tile, with lengths that end within a chunk."""
    counts, lengths, heads = [1, 3, 2, 1, 6, 1], [1, 70, 200, 64, 37, 1999], 16
    table, blocks = pages_for(1, counts, lengths, heads, turned)
    cache, scales = held(2, blocks, 64, width, block, 117, 123)
    sizes = [0.0, 1.0, 2.0 ** -120, 0.0, 2.0 ** -60, 2.0 ** -126, 2.0 ** -113] if dtype == BF16 else [0.0, 1.0, 2.0 ** -14, 0.0, 2.0 ** -20, 2.0 ** -24, 2.0 ** -10]
    own = torch.tensor(sizes, device="cuda")[torch.arange(sum(counts) * heads, device="cuda") % len(sizes)].view(-1, heads, 1)
    q = (normal(3, sum(counts), heads, width, spread=0.3) * own).to(dtype)
    sinks = normal(4, heads) if with_sinks else None
    for queries in (q, torch.zeros_like(q)):
        got = attend(queries, cache, scales, table, counts, lengths, width ** -0.5, sinks)
        assert torch.isfinite(got[0]).all() and torch.isfinite(got[1]).all()
        check(got, queries, cache, scales, table, counts, lengths, width ** -0.5, turned, sinks)


@pytest.mark.parametrize("dtype,turned", FORMS)
@pytest.mark.parametrize("exponent", [0, -14, -110])
def test_a_cache_of_zeros(dtype, turned, exponent):
    """Scale bytes 0: every key counts alike."""
    counts, lengths, heads = [2, 1], [100, 33], 24
    table, blocks = pages_for(5, counts, lengths, heads, turned)
    cache, scales = (torch.zeros(shape, dtype=torch.uint8, device="cuda").view(t) for shape, t in (((blocks, 64, 1, 576), E.HELD), ((blocks, 4), E.SCALE)))
    out, lse = attend(normal(6, 3, heads, 576, spread=2.0 ** exponent).to(dtype), cache, scales, table, counts, lengths, 0.04)
    assert (out == 0).all()
    expected = torch.tensor([99.0, 100.0, 33.0], device="cuda", dtype=torch.float64).log()[:, None].expand(3, heads)
    R.within(lse, expected, 2.0 ** -18 + 2.0 ** -22 * expected)


@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("exponent,scale", [(0, 1e-30), (-30, 1e-30), (-100, 1e-30), (-118, 1.0), (-100, 1e30), (-126, 1e30), (60, 1e-20)])
def test_sizes_and_scales_at_the_ends(turned, exponent, scale):
    """The scale of a score times its query's may be none of FP32's normal numbers where the score is one."""
    counts, lengths, heads = [2, 1, 3], [100, 33, 130], 16
    table, blocks = pages_for(7, counts, lengths, heads, turned)
    cache, scales = held(8, blocks, 64, 576, 4, 117, 123)
    q = (normal(9, sum(counts), heads, 576, spread=0.3) * 2.0 ** exponent).bfloat16()
    check(attend(q, cache, scales, table, counts, lengths, scale), q, cache, scales, table, counts, lengths, scale, turned)


@pytest.mark.parametrize("turned", [False, True])
def test_tiny_queries_of_large_scales(turned):
    """Queries of 2^-118 and values of 2^100 and more: scores of ordinary size out of a query's scale that FP32 holds no product of."""
    counts, lengths, heads = [2, 1, 1], [100, 33, 1], 16
    table, blocks = pages_for(10, counts, lengths, heads, turned)
    cache, scales = held(11, blocks, 64, 576, 2, 224, 228)
    q = (normal(12, sum(counts), heads, 576) * 2.0 ** -118).bfloat16()
    check(attend(q, cache, scales, table, counts, lengths, 2.0 ** -4), q, cache, scales, table, counts, lengths, 2.0 ** -4, turned)


# ---- what is masked ---------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,turned", FORMS)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_a_query_without_a_number_that_sees_no_key(dtype, turned, value):
    """Its output is zeros, whatever it holds, beside tokens of the same tile that see some."""
    counts, lengths, heads = [5, 3], [3, 100], 8
    table, blocks = pages_for(13, counts, lengths, heads, turned)
    cache, scales = held(14, blocks, 64, 576, 8, 117, 123)
    q = normal(15, 8, heads, 576, spread=0.3).to(dtype)
    clean = attend(q, cache, scales, table, counts, lengths, 0.04)
    q[0, :, 7] = q[1, 3] = value  # the first request's first two tokens see nothing
    out, lse = attend(q, cache, scales, table, counts, lengths, 0.04)
    assert (out[:2] == 0).all() and (lse[:2] == -math.inf).all()
    assert torch.equal(out, clean[0]) and torch.equal(lse, clean[1])


@pytest.mark.parametrize("dtype,turned", FORMS)
@pytest.mark.parametrize("block", [1, 8, 64])
@pytest.mark.parametrize("width,heads", [(576, 16), (512, 64)])
def test_a_scale_without_a_number_leaves_alone_what_does_not_see_it(dtype, turned, block, width, heads):
    """The last block of rows of every other request: a draft that overflowed. Tokens in front of it, in the same tile, do not see it."""
    counts, lengths = [7, 2, 4, 1, 3, 66], [70, 100, 3, 64, 3009, 130]
    table, blocks = pages_for(16, counts, lengths, heads, turned)
    cache, scales = held(17, blocks, 64, width, block, 117, 123)
    q = normal(18, sum(counts), heads, width, spread=0.3).to(dtype)
    clean = attend(q, cache, scales, table, counts, lengths, width ** -0.5)
    spoilt, token = torch.zeros(sum(counts), dtype=torch.bool, device="cuda"), 0
    for b, (n, length) in enumerate(zip(counts, lengths)):
        if b % 2 == 0 or b == 5:
            first = (length - 1) // block * block  # of the block's rows
            scales.view(torch.uint8)[table[b, first // 64], first % 64 // block] = 255
            spoilt[token : token + n] = length - n + 1 + torch.arange(n, device="cuda") > first
        token += n
    out, lse = attend(q, cache, scales, table, counts, lengths, width ** -0.5)
    assert torch.equal(out[~spoilt], clean[0][~spoilt]) and torch.equal(lse[~spoilt], clean[1][~spoilt])
    assert torch.isnan(out[spoilt]).all() and torch.isnan(lse[spoilt]).all() and 0 < int(spoilt.sum()) < len(spoilt)


@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("low,exponent", [(6, 110), (0, 118), (230, -100)])
@pytest.mark.parametrize("behind", [0, 64, 127, 254, 255])
def test_scales_behind_the_rows_may_be_anything(turned, low, exponent, behind):
    """What an earlier request has left there does not move the scales of rows that count."""
    counts, lengths, heads = [1, 2, 1], [70, 2, 129], 16
    table, blocks = pages_for(19, counts, lengths, heads, turned)
    cache, scales = held(20, blocks, 64, 576, 1, low, low + 4)
    cache = torch.where(cache.float().abs() < 2, 2.0, cache.float()).to(E.HELD)  # (normal numbers of bfloat16 with every scale)
    q = (normal(21, 4, heads, 576) * 2.0 ** exponent).bfloat16()
    clean = attend(q, cache, scales, table, counts, lengths, 0.02)
    for b, length in enumerate(lengths):
        scales.view(torch.uint8)[table[b, length // 64], length % 64 :] = behind
    out, lse = attend(q, cache, scales, table, counts, lengths, 0.02)
    assert torch.isfinite(lse).all() and (lse.amax(1) != lse.amin(1)).all()  # (scores that count)
    assert torch.equal(out, clean[0]) and torch.equal(lse, clean[1])
