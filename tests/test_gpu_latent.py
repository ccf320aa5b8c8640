"""Operators around dense latent attention on a GPU, against their definitions in 64 bits."""

import functools
import itertools

import pytest
import torch

from ascendflow_b200 import latent, ops
from ascendflow_b200.diagnostics import CompileError
from tests import latent_reference as R

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def normal(seed, *shape, dtype=BF16, spread=1.0):
    generator = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, device="cuda", generator=generator) * spread).to(dtype)


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def starts(counts):
    return i32([0, *itertools.accumulate(counts)])


# ---- rotary ----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("tokens,heads,features,pairs", [(1, 64, 64, 32), (3, 5, 192, 32), (130, 1, 64, 32), (7, 128, 512, 32), (2, 3, 256, 128), (5, 2, 24, 8), (300, 9, 128, 64)])
def test_rotary(dtype, layout, tokens, heads, features, pairs):
    x = normal(1, tokens, heads, features, dtype=dtype)
    positions = torch.randint(0, 200000, (tokens,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    inv_freq = latent.rotary_frequencies(2 * pairs)
    front = features - 2 * pairs
    for inverse, amplitude, index in ((False, 1.0, torch.int32), (True, 1.2079, torch.int64)):
        out = latent.rotary(x, positions.to(index), inv_freq, layout=layout, inverse=inverse, amplitude=amplitude)
        expected = R.turn(x[..., front:], positions, inv_freq, layout, amplitude, inverse)
        R.within(out[..., front:], expected, R.turn_tolerance(x, expected, pairs, amplitude), "turned")
        assert torch.equal(out[..., :front], x[..., :front])
        own = x.clone()
        assert latent.rotary(own, positions.to(index), inv_freq, layout=layout, inverse=inverse, amplitude=amplitude, out=own) is own
        assert torch.equal(own, out)
        flat = latent.rotary(x[:, 0].contiguous(), positions.to(index), inv_freq, layout=layout, inverse=inverse, amplitude=amplitude)
        assert torch.equal(flat, out[:, 0])


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_rotary_far_positions_keep_their_angles(layout):
    positions = torch.tensor([0, 1, -1, 131071, (1 << 31) - 1, -(1 << 31), (1 << 40) + 12345, 7], device="cuda")
    x = normal(3, 8, 4, 64, dtype=F32)
    inv_freq = latent.rotary_frequencies(64, base=500000.0)
    out = latent.rotary(x, positions, inv_freq, layout=layout)
    # the reference's product position * frequency is off by 2^-53 of itself, and so is the frequency as a fraction of a turn
    expected = R.turn(x, positions, inv_freq, layout)
    off = positions.double().abs().view(-1, 1, 1) * 2.0 ** -51 * x.double().abs().amax(-1, keepdim=True)
    R.within(out, expected, R.turn_tolerance(x, expected, 32) + off, layout)


def test_rotary_takes_slices_and_leaves_the_rest_alone():
    projected, q = normal(4, 9, 6, 192), normal(5, 9, 6, 576)
    before, positions, inv_freq = q.clone(), i32(range(100, 109)), latent.rotary_frequencies(64)
    latent.rotary(projected[..., 128:], positions, inv_freq, out=q[..., 512:])
    assert torch.equal(q[..., :512], before[..., :512])
    assert torch.equal(q[..., 512:], latent.rotary(projected[..., 128:].contiguous(), positions, inv_freq))
    turned = projected.transpose(0, 1)  # heads in front of tokens
    assert torch.equal(latent.rotary(turned, i32(range(6)), inv_freq), latent.rotary(turned.contiguous(), i32(range(6)), inv_freq))
    shared = projected[:, :1].expand(9, 6, 192)  # one head for all
    assert torch.equal(latent.rotary(shared, positions, inv_freq), latent.rotary(shared.contiguous(), positions, inv_freq))
    back = latent.rotary(latent.rotary(projected.float(), positions, inv_freq), positions, inv_freq, inverse=True)
    assert torch.allclose(back, projected.float(), atol=1e-5)


def test_rotary_of_nothing():
    inv_freq = latent.rotary_frequencies(64)
    assert latent.rotary(normal(0, 0, 4, 64), i32([]), inv_freq).shape == (0, 4, 64)
    assert latent.rotary(normal(0, 2, 0, 64), i32([1, 2]), inv_freq).shape == (2, 0, 64)


def test_rotary_refusals():
    x, positions, inv_freq = normal(6, 4, 2, 64), i32([0, 1, 2, 3]), latent.rotary_frequencies(64)
    latent.rotary(x, positions, inv_freq)
    buffer = normal(7, 4, 2, 130)
    for message, call in (
        ("float64", lambda: latent.rotary(x, positions, inv_freq.float())),
        ("positions", lambda: latent.rotary(x, positions.float(), inv_freq)),
        ("shape", lambda: latent.rotary(x, positions[:3], inv_freq)),
        ("multiple of 8", lambda: latent.rotary(x, positions, inv_freq[:20])),
        ("turned part", lambda: latent.rotary(x[..., :48], positions, inv_freq)),
        ("16-byte", lambda: latent.rotary(buffer[..., 1:65], positions, inv_freq)),
        ("16-byte", lambda: latent.rotary(buffer[..., ::2][..., :64], positions, inv_freq)),
        ("share memory", lambda: latent.rotary(x, positions, inv_freq, out=normal(8, 4, 1, 64).expand(4, 2, 64))),
        ("overlap", lambda: latent.rotary(x[:3], positions[:3], inv_freq, out=x[1:])),
        ("shape and type", lambda: latent.rotary(x, positions, inv_freq, out=x.half())),
        ("gradient", lambda: latent.rotary(x.clone().requires_grad_(), positions, inv_freq)),
        ("expected", lambda: latent.rotary(x.double(), positions, inv_freq)),
        ("CUDA tensor", lambda: latent.rotary(x, positions.cpu(), inv_freq)),
    ):
        with pytest.raises(CompileError, match=message):
            call()
    with torch.no_grad():
        latent.rotary(x.clone().requires_grad_(), positions, inv_freq)


# ---- paged caches ----------------------------------------------------------------------------------------------------

def paged(seed, lengths, width, page, dtype, spare=3, pages=None, spread=1.0):
    """A cache in which unused pages and rows behind a request's length hold NaN, and its table (-1 where a request has no page)."""
    used = [-(-max(length, 0) // page) for length in lengths]
    order = torch.randperm(sum(used) + spare, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed + 1)).tolist()
    table = torch.full((len(lengths), max([pages or 1, *used])), -1, dtype=torch.int32)
    cache = torch.full((len(order), page, 1, width), float("nan"), dtype=dtype, device="cuda")
    rows = normal(seed, max(1, sum(used)), page, 1, width, dtype=dtype, spread=spread)
    place = 0
    for b, (count, length) in enumerate(zip(used, lengths)):
        for column in range(count):
            table[b, column] = order[place]
            valid = min(page, length - column * page)
            cache[order[place], :valid] = rows[place, :valid]
            place += 1
    return cache, table.cuda()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("counts,lengths,width,page", [
    ([1], [1], 576, 128), ([3, 0, 5], [64, 0, 130], 576, 64), ([2, 2], [1, 700], 512, 192), ([200], [200], 576, 128), ([1] * 70, list(range(1, 71)), 512, 64)])
def test_append(dtype, layout, counts, lengths, width, page):
    cache, table = paged(1, lengths, width, page, dtype)
    tokens = sum(counts)
    rows, rope = normal(2, tokens, width - 64, dtype=dtype), normal(3, tokens, width, dtype=dtype)[:, -64:]
    inv_freq = latent.rotary_frequencies(64)
    ops.status()
    expected = R.append(rows, rope, cache, table, counts, lengths, inv_freq, layout, 1.25)
    before = cache.clone()
    assert latent.rotary_append(rows, rope, cache, table, starts(counts), i32(lengths), inv_freq, layout=layout, amplitude=1.25) is cache
    written = (expected != before.double()) & ~(expected.isnan() & before.isnan())
    assert torch.equal(cache[~written].view(torch.int16), before[~written].view(torch.int16))
    front = cache[..., : width - 64].double()
    assert torch.equal(front.nan_to_num(7), expected[..., : width - 64].nan_to_num(7))
    R.within(cache[..., width - 64 :].double().nan_to_num(7), expected[..., width - 64 :].nan_to_num(7),
             R.HALF_STEP[dtype] * expected[..., width - 64 :].nan_to_num(7).abs() + 16 * 2.0 ** -24 * 8 * 1.25, "rope")
    # request 1 of the second and third calls has fewer rows than tokens: what has no position is reported
    short = any(n > length for n, length in zip(counts, lengths))
    assert (ops.status()[0] == 1) == short


def test_append_reports_bad_pages_and_leaves_padding_out():
    cache, table = paged(1, [200, 200], 576, 64, BF16)
    rows, rope, inv_freq = normal(2, 9, 512), normal(3, 9, 64), latent.rotary_frequencies(64)
    good, before = cache.clone(), cache.clone()
    ops.status()
    latent.rotary_append(rows, rope, good, table, i32([2, 4, 7]), i32([200, 200]), inv_freq)  # tokens 0, 1, 7 and 8 belong to nobody
    assert ops.status()[0] == 0
    expected = R.append(rows[2:7], rope[2:7], cache, table, [2, 3], [200, 200], inv_freq, "interleaved")
    changed = (good.view(torch.int16) != before.view(torch.int16)).any(-1)  # (single features may be what they were)
    assert torch.equal(changed, ((expected != before.double()) & ~(expected.isnan() & before.isnan())).any(-1)) and changed.sum() == 5
    for wrong in (-1, cache.shape[0], 1 << 30):
        bad = table.clone()
        bad[1, 3] = wrong
        cache.copy_(before)
        latent.rotary_append(rows, rope, cache, bad, i32([2, 4, 7]), i32([200, 200]), inv_freq)
        report = ops.status()
        assert report[0] == 1 and 4 <= report[1] < 7 and 197 <= report[2] < 200
        assert not torch.equal(cache.view(torch.int16), before.view(torch.int16))
    cache.copy_(before)
    latent.rotary_append(rows[:1], rope[:1], cache, table, i32([0, 1, 1]), i32([64 * 4 + 1, 0]), inv_freq)  # behind the table
    assert ops.status()[0] == 1 and torch.equal(cache.view(torch.int16), before.view(torch.int16))


def test_append_refusals():
    cache, table = paged(1, [100], 576, 64, BF16)
    rows, rope, cu, lengths, inv_freq = normal(2, 2, 512), normal(3, 2, 64), i32([0, 2]), i32([100]), latent.rotary_frequencies(64)
    call = lambda **k: latent.rotary_append(*{**dict(a=rows, b=rope, c=cache, d=table, e=cu, f=lengths, g=inv_freq), **k}.values())  # noqa: E731
    call()
    for message, change in (
        ("cache rows of W", dict(a=rows[:, :504].contiguous())), ("cache rows of W", dict(b=rope[:1])), ("type of latent", dict(b=rope.half())),
        ("multiple of 64 rows", dict(c=cache[:, :32].contiguous())), ("contiguous", dict(c=normal(1, 4, 64, 1, 1152)[..., ::2])), ("shape", dict(e=i32([0]))),
        ("shape", dict(f=i32([1, 2]))), ("int32", dict(d=table.long())), ("float64", dict(g=inv_freq.float())),
        ("16-byte", dict(a=normal(2, 2, 516)[:, 2:514])), ("overlap", dict(a=cache.view(-1, 576)[:2, :512])),
    ):
        with pytest.raises(CompileError, match=message):
            call(**change)


# ---- attention over the paged cache -------------------------------------------------------------------------------------

def check_attention(q, cache, table, counts, lengths, scale, sinks=None, bad=(), first=0):
    """The call against the definition; `bad`: (request, page column) without a legal page."""
    tokens, heads, width = q.shape
    lse = torch.full((tokens, heads), 77.0, device="cuda")
    out = torch.full((tokens, heads, 512), 77.0, dtype=q.dtype, device="cuda")
    cu = i32([first, *(first + n for n in itertools.accumulate(counts))])
    ops.status()
    assert latent.latent_attention(q, cache, table, cu, i32(lengths), scale=scale, sinks=sinks, out=out, lse=lse) is out
    report = ops.status()
    page, token = cache.shape[1], first
    for b, (n, length) in enumerate(zip(counts, lengths)):
        reach = max(length, 0)
        index = torch.arange(reach, device="cuda")
        legal = torch.tensor([(b, p) not in bad for p in range(-(-reach // page) or 1)], device="cuda").repeat_interleave(page)[:reach]
        pages = torch.nn.functional.pad(table[b].long(), (0, -(-reach // page)))[: -(-reach // page)]  # behind the table: any
        rows = cache[pages.clamp(0, cache.shape[0] - 1)].view(1, -1, width)[:, :reach]
        rows = torch.where(legal[:, None], rows, torch.zeros_like(rows))
        seen = (index < torch.arange(length - n + 1, length + 1, device="cuda")[:, None]) & legal
        own = slice(token, token + n)
        expected, log, error, log_error = R.attention(q[own], rows, rows[..., :512], seen, scale, sinks)
        R.within(out[own], expected, error, f"request {b}")
        R.within(lse[own], log, log_error, f"lse of request {b}")
        token += n
    for rest in (slice(0, first), slice(token, None)):
        assert (out[rest] == 77).all() and (lse[rest] == 77).all()
    assert (report[0] == 1) == bool(bad) and report[0] != 2, report
    plain = latent.latent_attention(q, cache, table, cu, i32(lengths), scale=scale, sinks=sinks)
    assert torch.equal(plain[first:token], out[first:token])  # the same bits again, without lse
    return out


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("width", [576, 512])
@pytest.mark.parametrize("heads,counts,lengths,page", [
    (64, [1], [1], 128),
    (64, [1], [64], 64),
    (64, [1], [65], 64),
    (64, [1, 1, 1], [63, 129, 1000], 128),
    (64, [6, 0, 3], [70, 5, 500], 64),
    (128, [2, 1], [300, 64], 128),
    (16, [5, 1, 7], [333, 31, 1025], 64),
    (1, [1, 130], [40, 200], 192),
    (5, [13, 1], [13, 1], 64),
    (24, [9], [2000], 128),
    (65, [3], [190], 64),
    (64, [1], [5000], 128),
])
def test_attention(dtype, width, heads, counts, lengths, page):
    cache, table = paged(1, lengths, width, page, dtype)
    check_attention(normal(2, sum(counts), heads, width, dtype=dtype), cache, table, counts, lengths, 192 ** -0.5)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_attention_sinks(dtype):
    cache, table = paged(1, [100, 1, 0, 3000], 576, 64, dtype)
    sinks = normal(3, 16, dtype=F32, spread=4.0)
    sinks[0], sinks[1], sinks[2] = -1e30, 50.0, -torch.inf
    check_attention(normal(2, 7, 16, 576, dtype=dtype), cache, table, [3, 1, 1, 2], [100, 1, 0, 3000], 0.05, sinks)


def test_attention_tokens_that_see_nothing():
    """Lengths of zero, below zero, and more tokens than rows."""
    lengths = [0, 3, -5, 2, 64]
    cache, table = paged(1, lengths, 576, 64, BF16)
    check_attention(normal(2, 16, 64, 576), cache, table, [1, 6, 2, 1, 6], lengths, 0.07)
    check_attention(normal(2, 10, 3, 576), cache, table, [1, 6, 1, 1, 1], lengths, 0.07, normal(4, 3, dtype=F32))


@pytest.mark.parametrize("heads", [64, 7])
def test_attention_padded_batch(heads):
    lengths = [130, 0, 65]
    cache, table = paged(1, lengths, 576, 64, BF16)
    check_attention(normal(2, 13, heads, 576), cache, table, [2, 0, 3], lengths, 0.07, first=3)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("spread", [0.01, 3.0, 12.0])
def test_attention_flat_and_steep_scores(dtype, spread):
    """From nearly equal weights to rows in which one key has all of it, keys growing along the row."""
    lengths = [900, 260]
    cache, table = paged(1, lengths, 576, 128, dtype, spread=0.5)
    flat = cache[table[0, :8].long().clamp(min=0)]
    cache[table[0, :8].long()] = flat * torch.linspace(0.1, 2.0, 8 * 128, device="cuda").view(8, 128, 1, 1).to(dtype)
    check_attention(normal(2, 4, 64, 576, dtype=dtype, spread=spread), cache, table, [2, 2], lengths, 0.07)


def test_attention_bad_pages():
    lengths = [500, 300, 70]
    for column, wrong in ((0, -1), (3, 1 << 30), (7, -7)):
        cache, table = paged(1, lengths, 576, 64, BF16)
        table[0, column] = wrong
        check_attention(normal(2, 5, 64, 576), cache, table, [2, 2, 1], lengths, 0.07, bad=[(0, column)])
    cache, table = paged(1, lengths, 576, 64, BF16)
    table[2] = cache.shape[0]  # a request without any page
    check_attention(normal(2, 5, 64, 576), cache, table, [2, 2, 1], lengths, 0.07, bad=[(2, 0), (2, 1)])
    cache, table = paged(1, lengths, 576, 64, BF16)
    check_attention(normal(2, 5, 16, 576), cache, table[:, :6].contiguous(), [2, 2, 1], lengths, 0.07, bad=[(0, 6), (0, 7)])  # a table that is too narrow


@pytest.mark.parametrize("heads,requests,queries,length", [(64, 1, 1, 70001), (16, 1, 3, 40000), (64, 5, 2, 9000), (128, 40, 1, 700), (64, 3, 70, 1500), (8, 300, 1, 90)])
def test_attention_long_and_many(heads, requests, queries, length):
    lengths = [max(queries, length - 97 * b) for b in range(requests)]
    cache, table = paged(1, lengths, 576, 64, BF16)
    check_attention(normal(2, requests * queries, heads, 576), cache, table, [queries] * requests, lengths, 192 ** -0.5)


@pytest.mark.parametrize("requests,heads", [(600, 16), (1100, 3), (40, 64), (150, 64), (300, 64)])
def test_attention_ragged_batches(requests, heads):
    """Requests of every kind in one call, more than a block has threads among them: without tokens, without keys, of many tiles. What one block
    does alone and what several share follows from the whole batch, so two batches of each."""
    generator = torch.Generator().manual_seed(requests)
    for longest in (300, 4000):
        counts = torch.randint(-1, 4, (requests,), generator=generator).clamp(min=0).tolist()
        lengths = (torch.rand(requests, generator=generator) ** 4 * longest).int().tolist()
        counts[requests // 2] = 50
        cache, table = paged(requests, lengths, 576, 64, BF16)
        check_attention(normal(2, sum(counts), heads, 576), cache, table, counts, lengths, 192 ** -0.5)


@pytest.mark.parametrize("heads,queries,lengths", [
    (64, 1, [1000] * 149), (64, 2, [640] * 74), (64, 1, [130] * 148), (64, 3, [2000] * 50), (128, 1, [700] * 75), (16, 9, [3000, 3000, 64]), (64, 200, [200, 900]),
])
def test_attention_batches_between_sharing_and_not(heads, queries, lengths):
    cache, table = paged(1, lengths, 576, 128, BF16)
    check_attention(normal(2, queries * len(lengths), heads, 576), cache, table, [queries] * len(lengths), lengths, 192 ** -0.5)


@pytest.mark.parametrize("heads", [1, 9, 23, 64])
@pytest.mark.parametrize("requests,length,ragged", [(1, 20000, 0), (3, 12000, 0), (7, 7000, 500), (16, 5000, 0), (40, 3500, 61)])
def test_attention_sums_of_shared_tiles(heads, requests, length, ragged):
    """Tiles of few to many parts, rows that are no multiple of eight; scores that rise along the keys, so that each part's reference is another, sinks, and
    parts none of whose pages is in the cache."""
    lengths = [length - ragged * b for b in range(requests)]
    cache, table = paged(requests, lengths, 576, 64, BF16)
    for b, n in enumerate(lengths):
        pages = table[b, : -(-n // 64)].long()
        cache[pages] *= torch.linspace(0.2, 1.5, len(pages), device="cuda").to(BF16).view(-1, 1, 1, 1)
    q = normal(2, requests, heads, 576, spread=2.0)
    check_attention(q, cache, table, [1] * requests, lengths, 0.06, normal(3, heads, dtype=F32, spread=4.0))
    bad = [(0, column) for column in range(20, min(lengths[0] // 64, 60))]
    for _, column in bad:
        table[0, column] = -1
    check_attention(q, cache, table, [1] * requests, lengths, 0.06, bad=bad)


def test_attention_offsets_beyond_32_bits():
    """A cache of more than 2^32 bytes and 2^31 features, its last pages in use."""
    blocks = 4_000_000 // 64
    cache = torch.full((blocks, 64, 1, 576), float("nan"), dtype=BF16, device="cuda")
    table = (blocks - 1 - torch.arange(20, dtype=torch.int32, device="cuda")).view(2, 10).contiguous()
    cache[-20:] = normal(1, 20, 64, 1, 576)
    cache[table[0, 9].item(), 5:] = float("nan")
    q, rows, rope, inv_freq = normal(2, 3, 64, 576), normal(3, 1, 512), normal(4, 1, 64), latent.rotary_frequencies(64)
    latent.rotary_append(rows, rope, cache, table, i32([0, 1, 1]), i32([581, 0]), inv_freq)
    assert torch.equal(cache[table[0, 9].item(), 4, 0, :512], rows[0])
    check_attention(q, cache, table, [1, 2], [581, 640], 0.06)


def test_attention_streams_threads_and_graphs():
    lengths = [3000, 50, 700]
    cache, table = paged(1, lengths, 576, 64, BF16)
    calls = [normal(10 + i, 6, 64, 576) for i in range(4)]
    cu, seq = starts([2, 1, 3]), i32(lengths)
    expected = [latent.latent_attention(q, cache, table, cu, seq, scale=0.07) for q in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    outs = [[] for _ in calls]
    for _ in range(20):  # all at once
        for q, stream, found in zip(calls, streams, outs):
            with torch.cuda.stream(stream):
                found.append(latent.latent_attention(q, cache, table, cu, seq, scale=0.07))
    torch.cuda.synchronize()
    for found, want in zip(outs, expected):
        assert all(torch.equal(out, want) for out in found)
    graphs, held = [], []
    for q in calls[:2]:  # two graphs, replayed at once on two streams
        graph, own = torch.cuda.CUDAGraph(), q.clone()
        with torch.cuda.graph(graph):
            held.append((own, latent.latent_attention(own, cache, table, cu, seq, scale=0.07)))
        graphs.append(graph)
    for _ in range(10):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for (own, out), want in zip(held, expected):
        assert torch.equal(out, want)
    held[0][0].copy_(calls[2])  # other queries, then other lengths in the same graph
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(held[0][1], expected[2])
    seq.copy_(i32([200, 40, 3]))
    graphs[0].replay()
    assert torch.equal(held[0][1], latent.latent_attention(calls[2], cache, table, cu, seq, scale=0.07))
    assert ops.status()[0] == 0


def test_attention_of_nothing():
    cache, table = paged(1, [10], 576, 64, BF16)
    assert latent.latent_attention(normal(0, 0, 64, 576), cache, table, i32([0, 0]), i32([10]), scale=1.0).shape == (0, 64, 512)
    empty = torch.full((2, 4, 512), 7.0, dtype=BF16, device="cuda")
    latent.latent_attention(normal(0, 2, 4, 576), cache, table[:0], i32([0]), i32([]), scale=1.0, out=empty)
    assert (empty == 7).all()
    check_attention(normal(2, 2, 4, 576), cache[:0], torch.zeros((1, 0), dtype=torch.int32, device="cuda"), [2], [0], 1.0)


@pytest.mark.parametrize("call", ["attention", "prefill", "append"])
def test_first_call_of_a_process_may_be_captured(call):
    """A fresh process whose first call of an operator is made while a graph is captured."""
    import subprocess
    import sys
    from pathlib import Path

    program = """
import torch
from ascendflow_b200 import latent
cache, table = torch.randn((4, 64, 1, 576), device="cuda").half(), torch.arange(4, dtype=torch.int32, device="cuda").view(1, 4)
cu, seq = torch.tensor([0, 3], dtype=torch.int32, device="cuda"), torch.tensor([200], dtype=torch.int32, device="cuda")
q, kv = torch.randn((3, 8, 576), device="cuda").half(), torch.randn((3, 8, 256), device="cuda").half()
frequencies = latent.rotary_frequencies(64)
calls = {
    "attention": lambda: latent.latent_attention(q, cache, table, cu, seq, scale=0.1),
    "prefill": lambda: latent.latent_prefill(q[..., :192], kv[..., :128], kv[..., 128:], q[:, 0, 512:], cu, cu, scale=0.1),
    "append": lambda: latent.rotary_append(q[:, 0, :512], q[:, 0, 512:], cache, table, cu, seq, frequencies),
}
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = calls["CALL"]()
graph.replay()
replayed = out.clone()
assert torch.equal(replayed, calls["CALL"]()) and replayed.isfinite().all()
print("done")
""".replace("CALL", call)
    result = subprocess.run([sys.executable, "-c", program], cwd=Path(__file__).resolve().parents[1], capture_output=True, text=True, timeout=120)
    assert result.stdout.strip() == "done", result.stderr[-2000:]


def test_attention_refusals():
    cache, table = paged(1, [100], 576, 64, BF16)
    q, cu, seq = normal(2, 3, 8, 576), i32([0, 3]), i32([100])
    call = lambda scale=0.1, sinks=None, out=None, lse=None, **k: latent.latent_attention(  # noqa: E731
        *{**dict(q=q, cache=cache, table=table, cu=cu, seq=seq), **k}.values(), scale=scale, sinks=sinks, out=out, lse=lse)
    call()
    big = normal(3, 3, 8, 1024)
    for message, change in (
        ("scale", dict(scale=-1.0)), ("scale", dict(scale="1")), ("scale", dict(scale=1e300)), ("576", dict(q=normal(2, 3, 8, 640))), ("contiguous", dict(q=big[..., :576])),
        ("as wide", dict(q=big[..., :512].contiguous())), ("expected torch.bfloat16", dict(q=q, cache=cache.half())), ("float16", dict(q=q.float())),
        ("multiple of 64 rows", dict(cache=cache.view(-1, 32, 1, 576))), ("int32", dict(seq=seq.long())), ("shape", dict(cu=i32([0, 1, 3]))),
        ("sinks", dict(sinks=normal(1, 7, dtype=F32))), ("sinks", dict(sinks=normal(1, 8))), ("lse", dict(lse=normal(1, 3, 8))),
        ("out", dict(out=normal(1, 3, 8, 576))), ("overlap", dict(out=cache.view(-1)[: 3 * 8 * 512].view(3, 8, 512))), ("gradient", dict(q=q.clone().requires_grad_())),
        ("Torch tensor", dict(sinks=[1.0] * 8)),
    ):
        with pytest.raises(CompileError, match=message):
            call(**change)


# ---- prompts in expanded form -------------------------------------------------------------------------------------------

def check_prefill(q, kv, rope, counts, lengths, scale, causal=True, first=0, first_key=0):
    tokens, heads, _ = q.shape
    lse = torch.full((tokens, heads), 77.0, device="cuda")
    out = torch.full((tokens, heads, 128), 77.0, dtype=q.dtype, device="cuda")
    cu_q = i32([first, *(first + n for n in itertools.accumulate(counts))])
    cu_k = i32([first_key, *(first_key + n for n in itertools.accumulate(lengths))])
    ops.status()
    assert latent.latent_prefill(q, kv[..., :128], kv[..., 128:], rope, cu_q, cu_k, scale=scale, causal=causal, out=out, lse=lse) is out
    assert ops.status()[0] == 0
    token, key = first, first_key
    for b, (n, length) in enumerate(zip(counts, lengths)):
        own, keys = slice(token, token + n), slice(key, key + length)
        k = torch.cat([kv[keys, :, :128], rope[keys, None].expand(-1, heads, -1)], -1).transpose(0, 1)
        end = torch.arange(length - n + 1, length + 1, device="cuda") if causal else torch.full((n,), length, device="cuda")
        seen = torch.arange(length, device="cuda") < end[:, None]
        expected, log, error, log_error = R.attention(q[own], k, kv[keys, :, 128:].transpose(0, 1), seen, scale)
        R.within(out[own], expected, error, f"request {b}")
        R.within(lse[own], log, log_error, f"lse of request {b}")
        token, key = token + n, key + length
    for rest in (slice(0, first), slice(token, None)):
        assert (out[rest] == 77).all() and (lse[rest] == 77).all()
    plain = latent.latent_prefill(q, kv[..., :128], kv[..., 128:], rope, cu_q, cu_k, scale=scale, causal=causal)
    assert torch.equal(plain[first:token], out[first:token])


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,counts,lengths", [
    (1, [1], [1]),
    (2, [128], [128]),
    (3, [129], [129]),
    (2, [256, 1, 0, 300], [256, 1, 4, 300]),
    (4, [5, 64, 1], [700, 64, 1000]),
    (2, [257], [1024]),
    (16, [33, 127], [33, 130]),
    (1, [600], [600]),
])
def test_prefill(dtype, causal, heads, counts, lengths):
    keys = sum(lengths)
    check_prefill(normal(1, sum(counts), heads, 192, dtype=dtype), normal(2, keys, heads, 256, dtype=dtype), normal(3, keys, 64, dtype=dtype), counts, lengths, 192 ** -0.5, causal)


@pytest.mark.parametrize("heads", [1, 5])
def test_prefill_ragged_batches(heads):
    """More requests than a warp has threads, without tokens and without keys among them, and more items than blocks run at a time."""
    generator = torch.Generator().manual_seed(heads)
    counts = torch.randint(-3, 40, (170,), generator=generator).clamp(min=0).tolist()
    lengths = (torch.rand(170, generator=generator) ** 3 * 400).int().tolist()
    counts[33], lengths[33] = 700, 900
    counts[64:100] = [0] * 36
    check_prefill(normal(1, sum(counts), heads, 192), normal(2, sum(lengths), heads, 256), normal(3, sum(lengths), 64), counts, lengths, 192 ** -0.5)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,counts,lengths", [
    (1, [1], [1537]), (1, [1], [20000]), (16, [3], [5000]), (5, [300], [4001]), (4, [1000], [3333]), (2, [257, 0, 1, 130], [2000, 5000, 1, 7001]), (1, [40] * 9, [128 * b for b in range(9)] ),
    (24, [129], [9000]), (2, [2000], [1700]), (37, [1, 1], [3000, 6000]), (74, [2], [1664]), (75, [2], [1664]),
])
def test_prefill_of_few_queries_and_many_keys(dtype, causal, heads, counts, lengths):
    """Calls whose items are cut into pieces, and those next to them: pieces that rows do not reach, pieces that end inside a tile of keys, requests too
    short to be cut beside long ones, tokens that see nothing, as many items as are still cut, and one more."""
    q, kv, rope = normal(1, sum(counts), heads, 192, dtype=dtype), normal(2, sum(lengths), heads, 256, dtype=dtype), normal(3, sum(lengths), 64, dtype=dtype)
    check_prefill(q, kv, rope, counts, lengths, 192 ** -0.5, causal=causal)


@pytest.mark.parametrize("spread", [0.01, 12.0])
def test_prefill_pieces_of_flat_and_steep_scores(spread):
    """Every piece with another reference, the last keys with nearly all of the weight."""
    kv, rope = normal(2, 6000, 4, 256), normal(3, 6000, 64)
    kv[..., :128] *= torch.linspace(0.1, 2.0, 6000, device="cuda").to(BF16).view(-1, 1, 1)
    check_prefill(normal(1, 70, 4, 192, spread=spread), kv, rope, [70], [6000], 0.07)


def test_prefill_pieces_leave_padding_alone_and_do_not_see_others():
    counts, lengths = [3, 5], [2500, 3100]
    kv, rope = normal(2, 6000, 2, 256), normal(3, 6000, 64)
    kv[:100], kv[5700:], rope[:100], rope[5700:] = (torch.nan,) * 4
    check_prefill(normal(1, 20, 2, 192), kv, rope, counts, lengths, 0.07, first=4, first_key=100)


def test_prefill_in_pieces_in_graphs_and_on_two_streams():
    """Sums between the two kernels are a call's own: two captured graphs and calls of another stream, in turn and at once."""
    calls = []
    for seed, (heads, count, length) in enumerate([(16, 200, 5000), (3, 1, 9000), (16, 200, 5000)]):
        q, kv, rope = normal(seed, count, heads, 192), normal(seed + 10, length, heads, 256), normal(seed + 20, length, 64)
        cu_q, cu_k, out = i32([0, count]), i32([0, length]), torch.empty((count, heads, 128), dtype=BF16, device="cuda")
        calls.append((functools.partial(latent.latent_prefill, q, kv[..., :128], kv[..., 128:], rope, cu_q, cu_k, scale=0.07, out=out), out))
    expected = []
    for call, out in calls:
        call()
        torch.cuda.synchronize()
        expected.append(out.clone())
    graphs = []
    for call, _ in calls[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        graphs.append(graph)
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    for _, out in calls:
        out.zero_()
    torch.cuda.synchronize()
    for _ in range(20):
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
        with torch.cuda.stream(other):
            calls[2][0]()
    torch.cuda.synchronize()
    for (_, out), right in zip(calls, expected):
        assert torch.equal(out, right)


@pytest.mark.parametrize("causal", [True, False])
def test_prefill_rows_that_see_nothing_and_padding(causal):
    """Requests without keys, with fewer keys than queries, and buffers with NaN in front of, between and behind the sequences' ends."""
    counts, lengths = [3, 10, 200, 4], [0, 4, 130, 70]
    tokens, keys = 5 + sum(counts) + 9, 3 + sum(lengths) + 200
    q, kv, rope = normal(1, tokens, 2, 192), normal(2, keys, 2, 256), normal(3, keys, 64)
    for tensor, first, last in ((q, 5, 5 + sum(counts)), (kv, 3, 3 + sum(lengths)), (rope, 3, 3 + sum(lengths))):
        tensor[:first] = float("nan")
        tensor[last:] = float("nan")
    check_prefill(q, kv, rope, counts, lengths, 0.07, causal, first=5, first_key=3)


@pytest.mark.parametrize("poison", [float("nan"), float("inf")])
def test_prefill_requests_do_not_see_each_other(poison):
    """A request's values of NaN or infinity stay in that request."""
    counts, lengths = [70, 50, 129], [100, 90, 200]
    q, kv, rope = normal(1, sum(counts), 3, 192), normal(2, sum(lengths), 3, 256), normal(3, sum(lengths), 64)
    arguments = starts(counts), starts(lengths)
    before = latent.latent_prefill(q, kv[..., :128], kv[..., 128:], rope, *arguments, scale=0.07)
    kv[100:190], rope[100:190], q[70:120] = poison, poison, poison
    after = latent.latent_prefill(q, kv[..., :128], kv[..., 128:], rope, *arguments, scale=0.07)
    assert torch.equal(before[:70], after[:70]) and torch.equal(before[120:], after[120:])


@pytest.mark.parametrize("spread", [0.01, 3.0, 12.0])
def test_prefill_flat_and_steep_scores(spread):
    kv, rope = normal(2, 700, 2, 256, dtype=F16, spread=0.5), normal(3, 700, 64, dtype=F16)
    kv *= torch.linspace(0.1, 2.0, 700, device="cuda").view(700, 1, 1).half()
    check_prefill(normal(1, 300, 2, 192, dtype=F16, spread=spread), kv, rope, [300], [700], 0.07)


def test_prefill_strides():
    """Separate buffers, heads in front of tokens, rope keys out of a wider projection, one head of keys for all."""
    counts, lengths = [40, 100], [140, 100]
    q, kv, wide = normal(1, 140, 4, 192), normal(2, 240, 4, 256), normal(3, 240, 576)
    cu = starts(counts), starts(lengths)
    expected = latent.latent_prefill(q, kv[..., :128], kv[..., 128:], wide[:, 512:], *cu, scale=0.07)
    k, v, rope = kv[..., :128].contiguous(), kv[..., 128:].transpose(0, 1).contiguous().transpose(0, 1), wide[:, 512:].contiguous()
    swapped = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(latent.latent_prefill(swapped, k, v, rope, *cu, scale=0.07), expected)
    one = k[:, :1].expand(-1, 4, -1)
    assert torch.equal(latent.latent_prefill(q, one, v, rope, *cu, scale=0.07), latent.latent_prefill(q, one.contiguous(), v, rope, *cu, scale=0.07))


def test_prefill_of_nothing():
    none = normal(0, 0, 2, 128)
    assert latent.latent_prefill(normal(0, 0, 2, 192), none, none, normal(0, 0, 64), i32([0, 0]), i32([0, 0]), scale=1.0).shape == (0, 2, 128)
    out = latent.latent_prefill(normal(0, 3, 2, 192), none, none, normal(0, 0, 64), i32([0, 3]), i32([0, 0]), scale=1.0)
    assert (out == 0).all()


def test_prefill_refusals():
    q, kv, rope, cu = normal(1, 8, 2, 192), normal(2, 8, 2, 256), normal(3, 8, 64), i32([0, 8])
    call = lambda scale=0.1, causal=True, out=None, lse=None, **k: latent.latent_prefill(  # noqa: E731
        *{**dict(q=q, k=kv[..., :128], v=kv[..., 128:], rope=rope, cu_q=cu, cu_k=cu), **k}.values(), scale=scale, causal=causal, out=out, lse=lse)
    call()
    odd = normal(2, 8, 2, 260)
    for message, change in (
        ("scale", dict(scale=0.0)), ("causal", dict(causal=1)), ("192", dict(q=q[..., :128])), ("k: expected", dict(k=kv)), ("v: expected", dict(v=kv[:7, :, :128])),
        ("k_rope", dict(rope=rope[:, :32])), ("16-byte", dict(k=odd[..., 2:130])), ("int32", dict(cu_k=cu.long())), ("shape", dict(cu_k=i32([0]))),
        ("expected torch.bfloat16", dict(rope=rope.half())), ("overlap", dict(out=kv.view(-1)[: 8 * 2 * 128].view(8, 2, 128))), ("lse", dict(lse=normal(1, 8, 2))),
        ("gradient", dict(v=kv[..., 128:].clone().requires_grad_())), ("out", dict(out=normal(1, 8, 2, 256)[..., :128])),
        ("share memory", dict(rope=rope[:1].expand(8, 64))), ("share memory", dict(q=q[:1].expand(8, 2, 192))),
    ):
        with pytest.raises(CompileError, match=message):
            call(**change)


def test_prefill_streams_and_graphs():
    counts, lengths = [150, 1, 70], [150, 300, 700]
    kv, rope, cu = normal(2, sum(lengths), 4, 256), normal(3, sum(lengths), 64), (starts(counts), starts(lengths))
    calls = [normal(10 + i, sum(counts), 4, 192) for i in range(3)]
    run = lambda q: latent.latent_prefill(q, kv[..., :128], kv[..., 128:], rope, *cu, scale=0.07)  # noqa: E731
    expected = [run(q) for q in calls]
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in calls], []
    for _ in range(10):
        for q, stream in zip(calls, streams):
            with torch.cuda.stream(stream):
                outs.append(run(q))
    torch.cuda.synchronize()
    assert all(torch.equal(out, expected[i % 3]) for i, out in enumerate(outs))
    graph, own = torch.cuda.CUDAGraph(), calls[0].clone()
    with torch.cuda.graph(graph):
        out = run(own)
    for want, q in zip(expected, calls):
        own.copy_(q)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


# ---- together ---------------------------------------------------------------------------------------------------------

def test_a_prompt_and_its_next_tokens():
    """A layer as a program runs it: a prompt in expanded form, its rows appended, three more tokens in absorbed form. The latter also in
    expanded form, from the same projections: both are the same function."""
    tokens, more, heads = 150, 3, 16
    total = tokens + more
    latents, rope = normal(1, total, 512, dtype=F16), normal(2, total, 64, dtype=F16)
    down, up = normal(3, heads, 128, 512, spread=512 ** -0.5, dtype=F16), normal(4, heads, 128, 512, spread=512 ** -0.5, dtype=F16)
    projected = normal(5, total, heads, 192, dtype=F16)
    inv_freq = latent.rotary_frequencies(64, scaling="yarn", factor=8.0)
    positions, amplitude, scale = torch.arange(total, device="cuda"), latent.rotary_amplitude(8.0), 192 ** -0.5
    q = latent.rotary(projected, positions, inv_freq, amplitude=amplitude)
    keys = latent.rotary(rope, positions, inv_freq, amplitude=amplitude)
    k, v = torch.einsum("tc,hdc->thd", latents, down), torch.einsum("tc,hdc->thd", latents, up)
    whole = latent.latent_prefill(q, k, v, keys, i32([0, total]), i32([0, total]), scale=scale)
    prompt = latent.latent_prefill(q[:tokens], k[:tokens], v[:tokens], keys[:tokens], i32([0, tokens]), i32([0, tokens]), scale=scale)
    R.within(prompt, whole[:tokens].double(), torch.tensor(2.0 ** -9, device="cuda").double(), "prompt")
    cache = torch.full((3, 64, 1, 576), float("nan"), dtype=F16, device="cuda")
    table = i32([[2, 0, 1]])
    latent.rotary_append(latents[:tokens], rope[:tokens], cache, table, i32([0, tokens]), i32([tokens]), inv_freq, amplitude=amplitude)
    for first, count in ((tokens, 1), (tokens + 1, 2)):
        own = slice(first, first + count)
        latent.rotary_append(latents[own], rope[own], cache, table, i32([0, count]), i32([first + count]), inv_freq, amplitude=amplitude)
        absorbed = torch.empty((count, heads, 576), dtype=F16, device="cuda")
        absorbed[..., :512] = torch.einsum("thd,hdc->thc", projected[own, :, :128], down)
        latent.rotary(projected[own, :, 128:], positions[own], inv_freq, amplitude=amplitude, out=absorbed[..., 512:])
        out = latent.latent_attention(absorbed, cache, table, i32([0, count]), i32([first + count]), scale=scale)
        # five roundings to half (2^-11 each) of queries, keys, values and outputs of magnitude about 1 on the way
        expanded = torch.einsum("thc,hdc->thd", out, up)
        R.within(expanded, whole[own].double(), torch.tensor(2.0 ** -6, device="cuda").double(), f"tokens {first}..")
    assert ops.status()[0] == 0
