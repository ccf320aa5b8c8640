"""A latent cache held in 8 bits on a GPU: the append against its definition in 64 bits, attention against the definition and (half queries, whose products are the same) bit by bit
against attention over the 16-bit cache that holds the same values."""

import itertools

import pytest
import torch

from ascendflow_b200 import latent, latent8, ops
from ascendflow_b200.diagnostics import CompileError
from tests import latent8_reference as E
from tests import latent_reference as R

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def normal(seed, *shape, dtype=torch.float32, spread=1.0):
    generator = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, device="cuda", generator=generator) * spread).to(dtype)


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def starts(counts):
    return i32([0, *itertools.accumulate(counts)])


def held(seed, blocks, page_rows, width, block, low=117, high=131):
    """Random numbers (no NaN) and scale bytes low .. high - 1."""
    generator = torch.Generator(device="cuda").manual_seed(seed)
    cache = torch.randint(0, 256, (blocks, page_rows, 1, width), dtype=torch.uint8, device="cuda", generator=generator)
    cache = torch.where((cache & 127) == 127, cache ^ 1, cache).view(E.HELD)
    scales = torch.randint(low, high, (blocks, page_rows // block), dtype=torch.uint8, device="cuda", generator=generator)
    return cache, scales.view(E.SCALE)


def tables(seed, lengths, page_rows, spare=3):
    """A permuted table, with -1 behind each request's pages."""
    used = [-(-length // page_rows) for length in lengths]
    blocks = sum(used) + spare
    order = torch.randperm(blocks, generator=torch.Generator().manual_seed(seed)).tolist()
    table, at = [[-1] * (max(used, default=0) + 1) for _ in lengths], 0
    for row, n in zip(table, used):
        row[:n] = order[at : at + n]
        at += n
    return i32(table).reshape(len(lengths), -1), blocks


# ---- append ------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,layout", [(BF16, "interleaved"), (BF16, "half"), (F16, "half"), (F16, "interleaved")])
@pytest.mark.parametrize("block", [1, 2, 4, 8, 16, 32, 64])
@pytest.mark.parametrize("page_rows,width,pairs", [(64, 576, 32), (128, 512, 32), (192, 1040, 8), (64, 528, 128)])
def test_append(dtype, layout, block, page_rows, width, pairs):
    counts, lengths = [1, 6, 0, 70, 130, 3], [1, 300, 40, 71, 130, 66]
    table, blocks = tables(block, lengths, page_rows)
    cache, scales = held(1, blocks, page_rows, width, block)
    tokens = sum(counts) + 2  # two behind the last request
    rows = normal(2, tokens, width, spread=3.0) * torch.exp(normal(3, tokens, 1, spread=2.0))
    new, inv_freq = rows.to(dtype), latent.rotary_frequencies(2 * pairs)
    front = width - 2 * pairs
    found = E.append(new[:, :front], new[:, front:], cache, scales, table, counts, lengths, inv_freq, layout, 1.25)
    before = cache.clone(), scales.clone()
    got = latent8.rotary_append8(new[:, :front].contiguous(), new[:, front:], cache, scales, table, starts(counts), i32(lengths), inv_freq, layout=layout, amplitude=1.25)
    assert got[0] is cache and got[1] is scales and ops.status()[0] == 0
    E.check_append(found, cache, scales)
    # nothing else has changed
    for page, number, place, new_rows, _, _, _, older in found:
        for now, old in ((cache, before[0]), (scales, before[1])):
            now, old = now.view(torch.uint8), old.view(torch.uint8)
            part = slice(number * block, place + len(new_rows)) if now.dim() == 4 else slice(number, number + 1)
            old[page, part] = now[page, part]
    assert torch.equal(cache.view(torch.uint8), before[0].view(torch.uint8)) and torch.equal(scales.view(torch.uint8), before[1].view(torch.uint8))


@pytest.mark.parametrize("block", [4, 16, 64])
def test_a_block_scale_grows_with_its_rows(block):
    """Rows one at a time, of sizes up and down: the numbers in front are divided by the growth and rounded."""
    cache, scales = held(4, 2, 64, 576, block)
    inv_freq, table = latent.rotary_frequencies(64), i32([[1]])
    for position in range(2 * block if block < 64 else 64):
        rows = normal(10 + position, 1, 576, dtype=BF16, spread=2.0 ** ((7 * position) % 23 - 8))
        found = E.append(rows[:, :512], rows[:, 512:], cache, scales, table, [1], [position + 1], inv_freq, "half")
        latent8.rotary_append8(rows[:, :512], rows[:, 512:], cache, scales, table, i32([0, 1]), i32([position + 1]), inv_freq, layout="half")
        E.check_append(found, cache, scales)


def test_largest_and_smallest_rows():
    """The whole range of either type; zeros; what no finite scale serves."""
    inv_freq = torch.zeros(32, dtype=torch.float64, device="cuda")  # turned by nothing
    for dtype, sizes in ((BF16, [3.3e38, 448.0, 449.0, 2.0 ** -100, 2.0 ** -125, 0.0, float("inf"), float("nan")]), (F16, [65504.0, 61440.0, 2.0 ** -24, 1.0, 0.0, float("-inf"), float("nan"), 480.0])):
        rows = torch.zeros((8, 576), dtype=dtype, device="cuda")
        rows[:, 0] = torch.tensor(sizes, device="cuda").to(dtype)
        rows[:, 1] = rows[:, 0] / 3
        rows[:, 575] = rows[:, 0] / 16
        cache, scales = held(5, 1, 64, 576, 1)
        found = E.append(rows[:, :512], rows[:, 512:], cache, scales, i32([[0]]), [8], [8], inv_freq, "half")
        latent8.rotary_append8(rows[:, :512], rows[:, 512:], cache, scales, i32([[0]]), i32([0, 8]), i32([8]), inv_freq, layout="half")
        E.check_append(found, cache, scales)
        if dtype == F16:
            assert E.values(cache, scales)[0, 0, 0, 0].item() == 61440 and torch.isfinite(E.values(cache, scales)[0, :5].to(F16)).all()


def test_rows_without_a_page_are_reported_and_left_out():
    cache, scales = held(6, 3, 64, 576, 16)
    before = cache.clone(), scales.clone()
    inv_freq, rows = latent.rotary_frequencies(64), normal(7, 12, 576, dtype=BF16)
    table = i32([[0, 7], [-1, 1], [2, -1]])
    counts, lengths = [4, 4, 4], [66, 66, 2]  # into pages 0 and 7; nowhere and 1; before the beginning and 2
    found = E.append(rows[:, :512], rows[:, 512:], cache, scales, table, counts, lengths, inv_freq, "half")
    ops.status()
    latent8.rotary_append8(rows[:, :512], rows[:, 512:], cache, scales, table, starts(counts), i32(lengths), inv_freq, layout="half")
    assert ops.status()[0] == 1 and len(found) == 3
    E.check_append(found, cache, scales)
    assert torch.equal(cache[0, :48].view(torch.uint8), before[0][0, :48].view(torch.uint8)) and torch.equal(cache[2, 2:].view(torch.uint8), before[0][2, 2:].view(torch.uint8))
    # a length behind the table, and no requests or tokens
    latent8.rotary_append8(rows[:1, :512], rows[:1, 512:], cache, scales, table[:1], i32([0, 1]), i32([129]), inv_freq)
    assert ops.status()[0] == 1
    latent8.rotary_append8(rows[:0, :512], rows[:0, 512:], cache, scales, table[:1], i32([0, 0]), i32([1]), inv_freq)
    latent8.rotary_append8(rows[:2, :512], rows[:2, 512:], cache, scales, table[:0], i32([0]), i32([]), inv_freq)
    assert ops.status()[0] == 0


# ---- attention -----------------------------------------------------------------------------------------------------------

def both(q, cache, scales, table, cu, lengths, **options):
    """Attention over the cache in 8 bits, and over the one in 16 bits that holds the same values."""
    wide = E.values(cache, scales)
    assert torch.equal(wide.to(q.dtype).double().nan_to_num(0), wide.nan_to_num(0))
    outs = []
    for held8 in (True, False):
        lse = torch.full(q.shape[:2], 7.0, device="cuda")
        out = torch.full((*q.shape[:2], 512), 7.0, dtype=q.dtype, device="cuda")
        if held8:
            latent8.latent_attention8(q, cache, scales, table, cu, lengths, out=out, lse=lse, **options)
        else:
            latent.latent_attention(q, wide.to(q.dtype), table, cu, lengths, out=out, lse=lse, **options)
        outs.append((out, lse))
    return outs


CASES = [
    # counts, lengths, heads, page rows
    ([1], [1], 1, 64), ([1, 1, 1], [63, 64, 65], 64, 64), ([1] * 7, [0, 1, 128, 127, 129, 640, 2000], 64, 128),
    ([3, 0, 7, 1], [3, 100, 333, 6000], 16, 192), ([500], [700], 8, 64), ([6] * 12, [500 + 37 * i for i in range(12)], 64, 128),
    ([2] * 40, [17 * i for i in range(40)], 24, 64), ([1] * 149, [300] * 149, 64, 64), ([5, 4], [3, 2], 128, 64),
]


def large(heads, tokens, table, page_rows):
    """So many pages, of a cache and of a table, that a call of bfloat16 queries goes the other way round: 32 chunks to each of 148 blocks if requests are as long as the table."""
    tiles = max(-(-tokens * heads // 64), min(len(table), tokens))
    return -(-33 * 148 // (max(tiles, 1) * (page_rows // 64)))


@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("dtype,width,block,turned", [(BF16, 576, 1, False), (BF16, 512, 64, False), (F16, 576, 16, False), (F16, 512, 1, False), (BF16, 576, 32, False), (F16, 576, 64, False),
                                                      (BF16, 576, 1, True), (BF16, 512, 64, True), (BF16, 576, 16, True), (BF16, 512, 1, True)])
def test_attention(case, dtype, width, block, turned):
    counts, lengths, heads, page_rows = CASES[case]
    table, blocks = tables(case, lengths, page_rows)
    tokens = sum(counts) + 3  # three behind the last request
    if turned:
        pages = large(heads, tokens, table, page_rows)
        blocks = max(blocks, pages)
        table = torch.cat([table, torch.full((len(table), max(pages - table.shape[1], 0)), -1, dtype=torch.int32, device="cuda")], 1)
    cache, scales = held(case, blocks, page_rows, width, block, 117, 123)
    q = normal(20 + case, tokens, heads, width, dtype=dtype, spread=0.3)
    q[0] *= 2.0 ** -40  # rows of other sizes, and of few numbers
    q[min(1, tokens - 1), :, 1:] *= 2.0 ** -12
    sinks = normal(30, heads) if case % 2 else None
    (out, lse), (out16, lse16) = both(q, cache, scales, table, starts(counts), i32(lengths), scale=width ** -0.5, sinks=sinks)
    assert ops.status()[0] == 0
    if not turned:  # the products are the same
        assert torch.equal(out, out16) and torch.equal(lse, lse16)
    assert (out[-3:] == 7).all() and (lse[-3:] == 7).all()
    wide, token = E.values(cache, scales), 0
    for b, (n, length) in enumerate(zip(counts, lengths)):
        own = wide[table[b, : -(-length // page_rows)].long()].view(1, -1, width)[:, :length]
        seen = torch.arange(length, device="cuda") < (length - n + 1 + torch.arange(n, device="cuda"))[:, None]
        expected, expected_lse, error, lse_error = R.attention(q[token : token + n], own, own[..., :512], seen, width ** -0.5, sinks)
        if turned and length:  # a query is held by two numbers of 8 bits: to 2^-22 of its greatest, and half of that
            split = 1.5 * 2.0 ** -22 * width ** -0.5 * q[token : token + n].double().abs().amax(-1, keepdim=True) * own.abs().sum(-1).amax()
            lse_error = lse_error + split[..., 0]
            error = error + 2 * split * own[..., :512].abs().amax()
        R.within(out[token : token + n], expected, error, f"request {b}")
        R.within(lse[token : token + n], expected_lse, lse_error, f"request {b}, lse")
        token += n


@pytest.mark.parametrize("spread", [1.0, 30.0])
def test_long_rows_the_other_way_round(spread):
    """Many chunks to a block, pieces that begin and end within tiles, references that move (queries of a spread of 30: scores of hundreds)."""
    counts, lengths, heads, page_rows = [1, 2, 1, 3, 1, 1], [40000, 23456, 1, 30011, 64, 51000], 64, 128
    table, blocks = tables(9, lengths, page_rows)
    cache, scales = held(19, blocks, page_rows, 576, 8, 117, 121)
    q = normal(29, sum(counts), heads, 576, dtype=BF16, spread=0.3 * spread)
    lse = torch.empty(q.shape[:2], device="cuda")
    out = latent8.latent_attention8(q, cache, scales, table, starts(counts), i32(lengths), scale=576 ** -0.5, lse=lse)
    assert torch.equal(out, latent8.latent_attention8(q, cache, scales, table, starts(counts), i32(lengths), scale=576 ** -0.5)) and ops.status()[0] == 0
    wide, token = E.values(cache, scales), 0
    for b, (n, length) in enumerate(zip(counts, lengths)):
        own = wide[table[b, : -(-length // page_rows)].long()].view(1, -1, 576)[:, :length]
        seen = torch.arange(length, device="cuda") < (length - n + 1 + torch.arange(n, device="cuda"))[:, None]
        expected, expected_lse, error, lse_error = R.attention(q[token : token + n], own, own[..., :512], seen, 576 ** -0.5)
        split = 1.5 * 2.0 ** -22 * 576 ** -0.5 * q[token : token + n].double().abs().amax(-1, keepdim=True) * own.abs().sum(-1).amax()
        R.within(out[token : token + n], expected, error + 2 * split * own[..., :512].abs().amax(), b)
        R.within(lse[token : token + n], expected_lse, lse_error + split[..., 0], b)
        token += n


@pytest.mark.parametrize("blocks", [9, 2500])  # (2500: the other way round)
@pytest.mark.parametrize("dtype,low,high", [(BF16, 0, 40), (BF16, 130, 140), (BF16, 120, 200), (F16, 104, 112), (F16, 130, 137)])
def test_scales_of_the_whole_range(dtype, low, high, blocks):
    """Also those above 2^7, whose multiplication takes two steps, and those that leave subnormal numbers; values are kept where both types hold them."""
    cache, scales = held(8, blocks, 64, 576, 4, low, high)
    wide = E.values(cache, scales)
    fits = (wide.to(dtype).double() == wide).view(blocks, 16, -1).all(-1)
    cache = torch.where(fits.repeat_interleave(4, 1)[..., None, None], cache.view(torch.uint8), torch.zeros_like(cache.view(torch.uint8))).view(E.HELD)
    q = normal(9, 6, 64, 576, dtype=dtype)
    scale = 2.0 ** -max(high - 127, 0) * 576 ** -0.5 / 448
    table, lengths = torch.full((2, blocks), -1, dtype=torch.int32, device="cuda"), [130, 192]
    table[:, :3] = i32([[8, 1, 2], [3, 7, 5]])
    (out, lse), (out16, lse16) = both(q, cache, scales, table, i32([0, 3, 6]), i32(lengths), scale=scale)
    assert torch.isfinite(out).all()
    if dtype == F16 or blocks == 9:
        assert torch.equal(out, out16) and torch.equal(lse, lse16)
    for b, length in enumerate(lengths):
        own = E.values(cache, scales)[table[b, :3].long()].view(1, -1, 576)[:, :length]
        seen = torch.arange(length, device="cuda") < (length - 2 + torch.arange(3, device="cuda"))[:, None]
        expected, expected_lse, error, lse_error = R.attention(q[3 * b : 3 * b + 3], own, own[..., :512], seen, scale)
        split = 1.5 * 2.0 ** -22 * scale * q[3 * b : 3 * b + 3].double().abs().amax(-1, keepdim=True) * own.abs().sum(-1).amax() * (blocks > 9)
        # (what is below the smallest normal number counts as zero in FP32 sums: one for every key)
        R.within(out[3 * b : 3 * b + 3], expected, error + 2 * split * own[..., :512].abs().amax() + 2.0 ** -126 * length, b)
        R.within(lse[3 * b : 3 * b + 3], expected_lse, lse_error + split[..., 0], b)


@pytest.mark.parametrize("blocks", [9, 2500])
@pytest.mark.parametrize("exponent,low,high", [(-100, 228, 236), (100, 0, 6), (100, 25, 35), (-110, 228, 231)])
def test_queries_that_bring_scales_back(exponent, low, high, blocks):
    """Scores of ordinary size out of tiny queries and large scales, or the other way round: sums of products with either alone would not fit."""
    cache, scales = held(28, blocks, 64, 576, 2, low, high)
    q = normal(38, 4, 64, 576, dtype=BF16) * 2.0 ** exponent
    scale = 2.0 ** (127 - high - exponent - 8) * 576 ** -0.5
    if not 2.0 ** -100 <= scale <= 2.0 ** 100:
        scale = 0.5
    lengths, table = [100, 128], torch.full((2, blocks), -1, dtype=torch.int32, device="cuda")
    table[:, :2] = i32([[8, 1], [3, 7]])
    lse = torch.empty((4, 64), device="cuda")
    out = latent8.latent_attention8(q, cache, scales, table, i32([0, 2, 4]), i32(lengths), scale=scale, lse=lse)
    for b, length in enumerate(lengths):
        own = E.values(cache, scales)[table[b, :2].long()].view(1, -1, 576)[:, :length]
        seen = torch.arange(length, device="cuda") < (length - 1 + torch.arange(2, device="cuda"))[:, None]
        expected, expected_lse, error, lse_error = R.attention(q[2 * b : 2 * b + 2], own, own[..., :512], seen, scale)
        split = 1.5 * 2.0 ** -22 * scale * q[2 * b : 2 * b + 2].double().abs().amax(-1, keepdim=True) * own.abs().sum(-1).amax()
        R.within(out[2 * b : 2 * b + 2], expected, error + 2 * split * own[..., :512].abs().amax() + 2.0 ** -126 * length, b)
        R.within(lse[2 * b : 2 * b + 2], expected_lse, lse_error + split[..., 0], b)


@pytest.mark.parametrize("columns", [4, 2500])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_a_query_without_a_number_spoils_its_row(value, columns):
    lengths, page_rows = [200, 250], 64
    table, blocks = tables(6, lengths, page_rows, columns)
    table = torch.cat([table, torch.full((2, columns), -1, dtype=torch.int32, device="cuda")], 1)
    cache, scales = held(16, blocks, page_rows, 576, 8)
    q = normal(17, 2, 64, 576, dtype=BF16)
    arguments = (cache, scales, table, i32([0, 1, 2]), i32(lengths))
    clean = latent8.latent_attention8(q, *arguments, scale=0.04)
    for feature in (3, 511, 575):
        spoilt, lse = q.clone(), torch.empty((2, 64), device="cuda")
        spoilt[0, 5, feature] = spoilt[1, 63, feature] = value
        out = latent8.latent_attention8(spoilt, *arguments, scale=0.04, lse=lse)
        assert torch.isnan(out[0, 5]).all() and torch.isnan(out[1, 63]).all() and torch.isnan(lse[0, 5]) and torch.isnan(lse[1, 63])
        keep = torch.ones((2, 64), dtype=torch.bool, device="cuda")
        keep[0, 5] = keep[1, 63] = False
        assert torch.equal(out[keep], clean[keep]) and torch.isfinite(lse[keep]).all()


@pytest.mark.parametrize("turned", [False, True])
def test_what_lies_behind_the_rows_may_be_anything(turned):
    """NaN numbers and scales behind a request's length and in pages that are nobody's."""
    lengths, page_rows, block = [70, 1, 200, 128], 128, 16
    table, blocks = tables(3, lengths, page_rows, 700 if turned else 3)
    if turned:
        table = torch.cat([table, torch.full((4, 700), -1, dtype=torch.int32, device="cuda")], 1)
    cache, scales = held(11, blocks, page_rows, 576, block)
    q = normal(12, 4, 64, 576, dtype=BF16)
    clean = latent8.latent_attention8(q, cache, scales, table, starts([1] * 4), i32(lengths), scale=0.01)
    used = torch.zeros((blocks, page_rows), dtype=torch.bool, device="cuda")
    for b, length in enumerate(lengths):
        for i in range(length):
            used[table[b, i // page_rows], i % page_rows] = True
    cache.view(torch.uint8)[~used] = 127
    scales.view(torch.uint8)[~used.view(blocks, -1, block).any(-1)] = 255
    assert torch.equal(latent8.latent_attention8(q, cache, scales, table, starts([1] * 4), i32(lengths), scale=0.01), clean)


@pytest.mark.parametrize("turned", [False, True])
def test_a_scale_without_a_number_spoils_what_sees_it_and_nothing_else(turned):
    lengths, page_rows = [100, 100, 30], 64
    table, blocks = tables(5, lengths, page_rows, 2500 if turned else 3)
    if turned:
        table = torch.cat([table, torch.full((3, 2500), -1, dtype=torch.int32, device="cuda")], 1)
    cache, scales = held(13, blocks, page_rows, 576, 1)
    q, cu = normal(14, 6, 16, 576, dtype=BF16), starts([2, 2, 2])
    clean = latent8.latent_attention8(q, cache, scales, table, cu, i32(lengths), scale=0.01)
    scales.view(torch.uint8)[table[1, 99 // 64], 99 % 64] = 255  # the last row of the second request: its last token sees it
    out = latent8.latent_attention8(q, cache, scales, table, cu, i32(lengths), scale=0.01)
    assert torch.equal(out[[0, 1, 4, 5]], clean[[0, 1, 4, 5]]) and torch.isnan(out[3]).all()


@pytest.mark.parametrize("turned", [False, True])
def test_pages_outside_of_the_cache_are_masked_and_reported(turned):
    cache, scales = held(15, 2000 if turned else 6, 64, 576, 16)
    q, cu = normal(16, 3, 64, 576, dtype=BF16), i32([0, 1, 2, 3])
    table = i32([[0, 1, 2], [3, 9999, 4], [-1, -5, 2000]])
    if turned:
        table = torch.cat([table, torch.full((3, 2000), -1, dtype=torch.int32, device="cuda")], 1)
    ops.status()
    out = latent8.latent_attention8(q, cache, scales, table, cu, i32([150, 150, 150]), scale=0.01)
    assert ops.status()[0] == 1
    own = E.values(cache, scales)[[3, 0, 4]].view(1, -1, 576)[:, :150]
    seen = torch.ones((1, 150), dtype=torch.bool, device="cuda")
    seen[:, 64:128] = False
    expected, _, error, _ = R.attention(q[1:2], own, own[..., :512], seen, 0.01)
    R.within(out[1:2], expected, error)
    assert (out[2] == 0).all()
    empty = cache[:0], scales[:0]
    assert (latent8.latent_attention8(q, *empty, table, cu, i32([150, 0, 3]), scale=0.01) == 0).all()
    assert ops.status()[0] == 1


def test_offsets_behind_32_bits():
    """A cache of 5 GB: rows of its last pages, written and read."""
    blocks = 70000
    cache = torch.zeros((blocks, 128, 1, 576), dtype=torch.uint8, device="cuda").view(E.HELD)
    scales = torch.full((blocks, 8), 127, dtype=torch.uint8, device="cuda").view(E.SCALE)
    table, inv_freq = i32([[69999, 5, 69998]]), latent.rotary_frequencies(64)
    rows = normal(17, 300, 576, dtype=BF16)
    small = torch.zeros((2500, 128, 1, 576), dtype=torch.uint8, device="cuda").view(E.HELD), torch.zeros((2500, 8), dtype=torch.uint8, device="cuda").view(E.SCALE)
    for c, s, t in ((cache, scales, table), (*small, i32([[0, 1, 2]]))):
        latent8.rotary_append8(rows[:, :512], rows[:, 512:], c, s, t, i32([0, 300]), i32([300]), inv_freq)
    q = normal(18, 2, 64, 576, dtype=BF16)
    outs = [latent8.latent_attention8(q, c, s, t, i32([0, 2]), i32([300]), scale=0.05) for c, s, t in ((cache, scales, table), (*small, i32([[0, 1, 2]])))]
    assert torch.equal(*outs) and ops.status()[0] == 0
    more = torch.full((1, 2497), -1, dtype=torch.int32, device="cuda")  # the other way round
    tables_ = torch.cat([table, more], 1), torch.cat([i32([[0, 1, 2]]), more], 1)
    turned = [latent8.latent_attention8(q, c, s, t, i32([0, 2]), i32([300]), scale=0.05) for c, s, t in ((cache, scales, tables_[0]), (*small, tables_[1]))]
    assert torch.equal(*turned) and not torch.equal(turned[0], outs[0]) and ops.status()[0] == 0
    # weights and outputs are rounded by half a step, 2^-8, in either form; both are averages of values that the rows bound
    assert (turned[0].double() - outs[0].double()).abs().max() < 4.1 * 2.0 ** -8 * E.values(*small).abs().max()


# ---- how calls are made --------------------------------------------------------------------------------------------------

def arguments(turned=False):
    table, blocks = tables(1, [100, 200], 64, 2500 if turned else 3)
    if turned:
        table = torch.cat([table, torch.full((2, 2500), -1, dtype=torch.int32, device="cuda")], 1)
    cache, scales = held(1, blocks, 64, 576, 16)
    return {"q": normal(2, 4, 8, 576, dtype=BF16), "cache": cache, "scales": scales, "block_table": table, "cu_seqlens_q": i32([0, 2, 4]), "seqused_kv": i32([100, 200]), "scale": 0.04}


def test_refused_attention_calls():
    latent8.latent_attention8(**arguments())
    wrong = [("cache", lambda t: t.bfloat16()), ("cache", lambda t: t.view(torch.uint8)), ("cache", lambda t: t[:, :32]), ("scales", lambda t: t.view(torch.uint8)), ("scales", lambda t: t[:, :3]),
             ("scales", lambda t: t[:-1]), ("scales", lambda t: t.view(torch.uint8).repeat_interleave(32, 1).view(E.SCALE)), ("scales", lambda t: t.cpu()), ("scales", lambda t: None),
             ("q", lambda t: t.float()), ("q", lambda t: t[..., :512].contiguous()), ("q", lambda t: t.transpose(0, 1)), ("scale", lambda s: 0.0), ("scale", lambda s: "1"),
             ("block_table", lambda t: t.long()), ("seqused_kv", lambda t: t[:1]), ("cache", lambda t: t.view(torch.uint8).transpose(0, 1).contiguous().transpose(0, 1).view(E.HELD))]
    for name, change in wrong:
        own = arguments()
        own[name] = change(own[name])
        with pytest.raises(CompileError):
            latent8.latent_attention8(**own)
    own = arguments()
    with pytest.raises(CompileError):  # the output over an input
        latent8.latent_attention8(**own, out=own["q"].view(-1)[: 4 * 8 * 512].view(4, 8, 512))
    own["q"].requires_grad_()
    with pytest.raises(CompileError):
        latent8.latent_attention8(**own)
    assert ops.status()[0] == 0


def test_refused_append_calls():
    def call(**changes):
        own = arguments()
        rows = normal(3, 4, 576, dtype=BF16)
        own = dict(latent=rows[:, :512], rope=rows[:, 512:], cache=own["cache"], scales=own["scales"], block_table=own["block_table"], cu_seqlens_q=own["cu_seqlens_q"],
                   seqused_kv=own["seqused_kv"], inv_freq=latent.rotary_frequencies(64)) | changes
        return latent8.rotary_append8(**own)

    call()
    rows = normal(3, 4, 576, dtype=BF16)
    cache, scales = held(1, 5, 64, 568, 16)
    for changes in ({"latent": rows[:, :511]}, {"latent": rows[:, :512].float()}, {"rope": rows[:, 512:].half()}, {"latent": rows[:, :504], "cache": cache, "scales": scales}, {"layout": "both"},
                    {"amplitude": float("nan")}, {"scales": arguments()["scales"].view(torch.uint8)}, {"inv_freq": latent.rotary_frequencies(64).float()}, {"cache": arguments()["cache"].half()},
                    {"latent": rows[:, 1:513]}):
        with pytest.raises(CompileError):
            call(**changes)
    assert ops.status()[0] == 0


@pytest.mark.parametrize("turned", [False, True])
def test_two_streams_and_two_graphs(turned):
    """Calls that run at the same time, captured ones among them, have workspaces of their own."""
    own = [arguments(turned) for _ in range(2)]
    for k, a in enumerate(own):
        a["q"] = normal(40 + k, 4, 8, 576, dtype=BF16)
    expected = [latent8.latent_attention8(**a) for a in own]
    streams, graphs, outs = [torch.cuda.Stream() for _ in own], [], []
    for a, s in zip(own, streams):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            outs.append([latent8.latent_attention8(**a) for _ in range(3)])
        graphs.append(graph)
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    eager = []
    for a, s in zip(own, streams):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            eager.append([latent8.latent_attention8(**a) for _ in range(10)])
    torch.cuda.synchronize()
    for e, captured, called in zip(expected, outs, eager):
        assert all(torch.equal(e, out) for out in captured + called)


@pytest.mark.parametrize("turned", [False, True])
def test_a_captured_step_replays_with_new_lengths(turned):
    """Append and attention in a graph whose lengths the program moves on between replays."""
    table, blocks = tables(2, [64, 130], 64, 2500 if turned else 3)
    if turned:
        table = torch.cat([table, torch.full((2, 2500), -1, dtype=torch.int32, device="cuda")], 1)
    cache, scales = held(21, blocks, 64, 576, 16)
    rows, q, lengths, cu, inv_freq = normal(22, 2, 576, dtype=BF16), normal(23, 2, 8, 576, dtype=BF16), i32([9, 100]), i32([0, 1, 2]), latent.rotary_frequencies(64)
    out = torch.empty((2, 8, 512), dtype=BF16, device="cuda")

    def step(c, s):
        latent8.rotary_append8(rows[:, :512], rows[:, 512:], c, s, table, cu, lengths, inv_freq)
        latent8.latent_attention8(q, c, s, table, cu, lengths, scale=0.04, out=out)

    other = cache.clone(), scales.clone()
    step(cache.clone(), scales.clone())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(cache, scales)
    for k in range(12):
        rows.copy_(normal(50 + k, 2, 576, dtype=BF16, spread=2.0 ** (k - 5)))
        lengths.copy_(i32([9 + k, 100 + k]))
        graph.replay()
        got = out.clone()
        step(*other)
        assert torch.equal(got, out) and torch.equal(cache.view(torch.uint8), other[0].view(torch.uint8)) and torch.equal(scales.view(torch.uint8), other[1].view(torch.uint8))
