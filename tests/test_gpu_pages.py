"""The pages of a cache on a GPU against a plain program on the host: every number, and every byte of the caches."""

import itertools
import random

import pytest
import torch

from ascendflow_b200 import latent, latent8, ops, pages
from ascendflow_b200.diagnostics import CompileError
from tests import latent8_reference as E
from tests import latent_reference as R

pytestmark = pytest.mark.gpu


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# ---- the same on the host ------------------------------------------------------------------------------------------------

def counted(length, page_rows, entries):
    return min(-(-max(length, 0) // page_rows), entries)


def resized(table, counts, lengths, page_rows):
    table, counts = [list(row) for row in table], list(counts)
    for row, length in zip(table, lengths):
        for i in range(len(row)):
            if not 0 <= row[i] < len(counts):
                row[i] = -1
            elif i >= counted(length, page_rows, len(row)):
                counts[row[i]] -= 1
                row[i] = -1
    free = [p for p, count in enumerate(counts) if count == 0]
    for row, length in zip(table, lengths):
        for i in range(counted(length, page_rows, len(row))):
            if row[i] < 0 and free:
                row[i] = free.pop(0)
                counts[row[i]] = 1
    return table, counts


def forked(caches, table, counts, parents, lengths, page_rows):
    """(table, counts, caches) behind the call."""
    caches, entries = [cache.clone() for cache in caches], len(table[0]) if table else 0
    free, rows, seen = [p for p, count in enumerate(counts) if count == 0], [], set()
    for parent in parents:
        row = [-1] * entries
        if 0 <= parent < len(table):
            length = min(max(lengths[parent], 0), entries * page_rows)
            n, rest = counted(length, page_rows, entries), length % page_rows
            row[:n] = [p if 0 <= p < len(counts) else -1 for p in table[parent][:n]]
            if rest and row[n - 1] >= 0 and (parent in seen or counts[row[n - 1]] != 1):
                source, row[n - 1] = row[n - 1], free.pop(0) if free else -1
                for cache in caches if row[n - 1] >= 0 else ():
                    held = -(-rest * cache.shape[1] // page_rows)
                    cache[row[n - 1], :held] = cache[source, :held]
            seen.add(parent)
        rows.append(row)
    counts = [0] * len(counts)
    for p in itertools.chain(*rows):
        if p >= 0:
            counts[p] += 1
    return rows, counts, caches


def compacted(caches, table, counts):
    caches, counts = [cache.clone() for cache in caches], list(counts)
    border = sum(count > 0 for count in counts)
    places = [p if count > 0 else -1 for p, count in enumerate(counts)]
    for source, target in zip([p for p in range(border, len(counts)) if counts[p] > 0], [p for p in range(border) if counts[p] == 0]):
        places[source], counts[target], counts[source] = target, counts[source], 0
        for cache in caches:
            cache[target] = cache[source]
    return [[places[p] if 0 <= p < len(counts) else p for p in row] for row in table], counts, places, caches


def state_of(rng, requests, entries, blocks, page_rows, shared=0.3, empty=0.1):
    """A random table with its counts and lengths: some pages shared, some entries missing."""
    order, table, lengths = rng.sample(range(blocks), blocks), [], []
    for b in range(requests):
        length = rng.choice([0, rng.randrange(entries * page_rows + 1), rng.randrange(entries * page_rows + 1), entries * page_rows])
        row = [-1] * entries
        for i in range(counted(length, page_rows, entries)):
            if table and rng.random() < shared and table[-1][i] >= 0:
                row[i] = table[-1][i]
            elif rng.random() >= empty and order:
                row[i] = order.pop()
        table.append(row)
        lengths.append(length)
    counts = [0] * blocks
    for p in itertools.chain(*table):
        if p >= 0:
            counts[p] += 1
    return table, counts, lengths


def tensor(table, entries):
    return i32(table).reshape(len(table), entries)


def same(got, table, counts, entries):
    assert torch.equal(got[0].cpu(), torch.tensor(table, dtype=torch.int32).reshape(len(table), entries))
    assert torch.equal(got[1].cpu(), torch.tensor(counts, dtype=torch.int32))


def caches_of(seed, blocks, page_rows):
    """Tensors of many types and shapes: odd bytes to a page among them."""
    generator = torch.Generator(device="cuda").manual_seed(seed)

    def bytes_(*shape):
        return torch.randint(0, 256, (blocks, *shape), dtype=torch.uint8, device="cuda", generator=generator)

    return [bytes_(page_rows, 1, 1152).view(torch.bfloat16), bytes_(page_rows, 1, 576).view(E.HELD), bytes_(page_rows).view(E.SCALE), bytes_(page_rows // 16), bytes_(1, 7), bytes_(page_rows, 3),
            bytes_(page_rows // 2, 20).view(torch.int32), bytes_(2, 40000), bytes_(page_rows, 0)]


def equal(a, b):
    return all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a, b))


SIZES = [(1, 1, 1, 64), (3, 5, 12, 64), (7, 33, 100, 128), (40, 9, 300, 16), (5, 300, 900, 1), (300, 40, 3000, 64), (70, 1000, 40000, 64), (1300, 65, 30000, 128), (1, 70000, 70001, 64)]


@pytest.mark.parametrize("size", range(len(SIZES)))
@pytest.mark.parametrize("in_place", [False, True])
def test_resize(size, in_place):
    requests, entries, blocks, page_rows = SIZES[size]
    rng = random.Random(size)
    table, counts, lengths = state_of(rng, requests, entries, blocks, page_rows)
    for step in range(3):
        lengths = [rng.choice([length, length + rng.randrange(9), length - rng.randrange(9), 0, rng.randrange(entries * page_rows + 1)]) for length in lengths]
        lengths = [min(length, entries * page_rows) for length in lengths]
        given = tensor(table, entries), i32(counts)
        got = pages.resize(*given, i32(lengths), page_rows=page_rows, out=given if in_place else None)
        before, table, counts = (table, counts), *resized(table, counts, lengths, page_rows)
        same(got, table, counts, entries)
        if not in_place:
            same(given, *before, entries)  # left as they were
        short = any(p < 0 for row, length in zip(table, lengths) for p in row[: counted(length, page_rows, entries)])
        assert ops.status()[0] == (3 if short else 0)


def test_resize_takes_the_lowest_pages_and_says_who_went_without():
    table, counts = i32([[-1] * 4, [-1] * 4]), i32([0, 1, 0, 0, 1])
    got = pages.resize(table, counts, i32([129, 64]), page_rows=64)
    same(got, [[0, 2, 3, -1], [-1] * 4], [1, 1, 1, 1, 1], 4)
    assert ops.status()[:3] == (3, 1, 0)
    got = pages.resize(*got, i32([0, 100]), page_rows=64)  # what one gives back another has at once
    same(got, [[-1] * 4, [0, 2, -1, -1]], [1, 1, 1, 0, 1], 4)
    got = pages.resize(*got, i32([-5, 257]), page_rows=64)  # behind the table
    assert ops.status()[0] == 1
    same(got, [[-1] * 4, [0, 2, 3, -1]], [1, 1, 1, 1, 1], 4)


@pytest.mark.parametrize("size", range(7))
@pytest.mark.parametrize("children", [0, 1, 6, 64, 1500])
def test_fork(size, children):
    requests, entries, blocks, page_rows = SIZES[size]
    if page_rows < 16:
        page_rows = 16
    rng = random.Random(size * 10 + children)
    table, counts, lengths = state_of(rng, requests, entries, blocks, page_rows)
    parents = [rng.choice([-1, requests, *range(requests)]) if rng.random() < 0.5 else rng.randrange(min(requests, 3)) for _ in range(children)]
    caches = caches_of(size, min(blocks, 300), page_rows) if blocks <= 300 else []
    expected = forked(caches, table, counts, parents, lengths, page_rows)
    got = pages.fork(caches, tensor(table, entries), i32(counts), i32(parents), i32(lengths), page_rows=page_rows)
    same(got, *expected[:2], entries)
    assert equal(caches, expected[2])
    wanted = [r for r in range(children) for p, t in [(parents[r], expected[0][r])] if 0 <= p < requests and (n := counted(lengths[p], page_rows, entries)) and t[n - 1] < 0 <= table[p][n - 1]]
    assert ops.status()[0] == (3 if wanted else 0)


def test_fork_with_counts_in_place_and_lengths_that_do_not_fit():
    table, counts, caches = i32([[4, 1, -1], [2, -1, -1]]), i32([0, 1, 1, 0, 1]), [torch.arange(5 * 8, device="cuda").view(5, 8)]
    out = torch.empty((3, 3), dtype=torch.int32, device="cuda")
    got = pages.fork(caches, table, counts, i32([0, 0, 1]), i32([100, -3]), page_rows=64, out=(out, counts))
    assert got[0] is out and got[1] is counts
    same(got, [[4, 1, -1], [4, 0, -1], [-1, -1, -1]], [1, 1, 0, 0, 2], 3)
    assert torch.equal(caches[0][0, :5], torch.arange(8, 13, device="cuda")) and torch.equal(caches[0][0, 5:], torch.arange(5, 8, device="cuda"))  # 36 rows: five of eight parts
    assert ops.status()[0] == 0
    pages.fork([], table, got[1], i32([0]), i32([193, 0]), page_rows=64)
    assert ops.status()[:3] == (1, 0, 193)


@pytest.mark.parametrize("size", range(7))
@pytest.mark.parametrize("in_place", [False, True])
def test_compact(size, in_place):
    requests, entries, blocks, page_rows = SIZES[size]
    rng = random.Random(size)
    table, counts, _ = state_of(rng, requests, entries, blocks, page_rows)
    for p in rng.sample(range(blocks), blocks // 10):  # pages that somebody else keeps
        counts[p] += 1
    caches = caches_of(size, blocks, 16) if blocks <= 300 else [torch.randint(0, 256, (blocks, 5), dtype=torch.uint8, device="cuda")]
    expected = compacted(caches, table, counts)
    given = tensor(table, entries), i32(counts)
    got = pages.compact(caches, *given, out=given if in_place else None)
    same(got[:2], expected[0], expected[1], entries)
    assert torch.equal(got[2].cpu(), torch.tensor(expected[2], dtype=torch.int32)) and equal(caches, expected[3])
    again = pages.compact(caches, *got[:2])  # nothing to do
    assert torch.equal(again[0], got[0]) and torch.equal(again[1], got[1]) and equal(caches, expected[3]) and ops.status()[0] == 0


def test_compact_of_full_and_empty_caches():
    for counts in ([0] * 70, [1] * 70, [0] * 69 + [2], [2] + [0] * 69):
        cache = torch.arange(70, device="cuda").view(70, 1)
        table = [[p if c else -1 for p, c in enumerate(counts)]]
        expected = compacted([cache], table, counts)
        got = pages.compact([cache], i32(table), i32(counts))
        same(got[:2], expected[0], expected[1], 70)
        assert equal([cache], expected[3])


def test_a_cache_of_millions_of_pages():
    """The marks of its pages take more shared memory than blocks have without asking."""
    blocks = pages.MOST_BLOCKS
    counts = torch.ones(blocks, dtype=torch.int32, device="cuda")
    counts[[5, 4000000, blocks - 1]] = 0
    got = pages.resize(i32([[-1] * 4]), counts, i32([4]), page_rows=1)
    assert got[0].tolist() == [[5, 4000000, blocks - 1, -1]] and ops.status()[0] == 3
    counts.zero_()
    counts[[7, blocks - 1]] = 1
    cache = torch.zeros((blocks, 2), dtype=torch.uint8, device="cuda")
    cache[7], cache[-1] = 3, 4
    table, counts, places = pages.compact([cache], i32([[7, blocks - 1]]), counts)
    assert table.tolist() == [[1, 0]] or table.tolist() == [[0, 1]]
    assert counts[:2].tolist() == [1, 1] and int(counts.sum()) == 2 and cache[:2, 0].tolist() == [3 if p == 7 else 4 for p in sorted((7, blocks - 1), key=lambda p: int(places[p]))]
    with pytest.raises(CompileError):
        pages.resize(i32([[-1]]), torch.zeros(blocks + 1, dtype=torch.int32, device="cuda"), i32([4]), page_rows=1)


@pytest.mark.parametrize("in_place", [False, True])
def test_a_fork_of_many_rows(in_place):
    """More rows than the planning threads; about half of them get a page of their own before there are no more."""
    requests, entries, blocks, page_rows, children = 9, 3, 12000, 16, 20000
    rng = random.Random(77)
    table, counts, lengths = state_of(rng, requests, entries, blocks, page_rows)
    parents = [rng.randrange(-1, requests) for _ in range(children)]
    caches = [torch.randint(0, 256, (blocks, page_rows, 3), dtype=torch.uint8, device="cuda", generator=torch.Generator(device="cuda").manual_seed(7))]
    expected = forked(caches, table, counts, parents, lengths, page_rows)
    given = i32(counts)
    out = (torch.empty((children, entries), dtype=torch.int32, device="cuda"), given) if in_place else None
    got = pages.fork(caches, tensor(table, entries), given, i32(parents), i32(lengths), page_rows=page_rows, out=out)
    same(got, *expected[:2], entries)
    assert equal(caches, expected[2])
    ops.status()


@pytest.mark.parametrize("blocks", [100000, 500000])
@pytest.mark.parametrize("one_in", [1, 2, 5, 40, 3000])
def test_free_pages_lie_close_or_far_apart(blocks, one_in):
    """A large table's wishes are listed out of marks of every density, whole words of free pages and of used ones among them; nothing is left in the end."""
    requests, entries = 90, 1000
    generator = torch.Generator().manual_seed(one_in)
    free = torch.randint(0, one_in, (blocks,), generator=generator) == 0
    free[5000:9000], free[20000:60000] = True, False
    lengths = torch.randint(0, 64 * entries, (requests,), generator=generator, dtype=torch.int32)
    wishes = (torch.arange(entries) < (lengths[:, None] + 63) // 64)
    pages_ = free.nonzero()[:, 0].int()[: int(wishes.sum())]
    expected = torch.full((requests * entries,), -1, dtype=torch.int32)
    expected[wishes.flatten().nonzero()[: len(pages_), 0]] = pages_
    counts = (~free).int()
    got = pages.resize(torch.full((requests, entries), -1, dtype=torch.int32, device="cuda"), counts.cuda(), lengths.cuda(), page_rows=64)
    counts[pages_.long()] = 1
    assert torch.equal(got[0].cpu().flatten(), expected) and torch.equal(got[1].cpu(), counts)
    assert ops.status()[0] == (3 if len(pages_) < int(wishes.sum()) else 0)


def test_many_tensors():
    caches = [torch.full((6, 4, 24), k, dtype=torch.int16, device="cuda") + torch.arange(6, dtype=torch.int16, device="cuda").view(6, 1, 1) for k in range(pages.MOST_CACHES)]
    expected = forked(caches, [[2]], [0, 0, 1, 0, 0, 0], [0, 0, 0], [7], 8)
    got = pages.fork(caches, i32([[2]]), i32([0, 0, 1, 0, 0, 0]), i32([0, 0, 0]), i32([7]), page_rows=8)
    same(got, *expected[:2], 1)
    assert equal(caches, expected[2])
    with pytest.raises(CompileError):
        pages.fork([*caches, caches[0].clone()], i32([[2]]), i32([0] * 6), i32([0]), i32([7]), page_rows=8)


def test_refused_calls():
    table, counts, lengths, cache = i32([[0, -1]]), i32([1, 0, 0]), i32([70]), torch.zeros((3, 64, 16), device="cuda")
    pages.resize(table, counts, lengths, page_rows=64)
    for change in ({"block_table": table.long()}, {"counts": counts.float()}, {"lengths": lengths.cpu()}, {"lengths": i32([1, 2])}, {"page_rows": 0}, {"page_rows": 64.0}, {"page_rows": True},
                   {"out": (table, table.view(-1)[:1])}, {"out": (counts[:2].view(1, 2), counts)}, {"block_table": table.t()}, {"out": (table,)}, {"out": (table, None)}, {"block_table": None},
                   {"lengths": None}):
        with pytest.raises(CompileError):
            pages.resize(**{"block_table": table, "counts": counts, "lengths": lengths, "page_rows": 64, **change})
    parents = i32([0, 0])
    pages.fork([cache], table, counts, parents, lengths, page_rows=64)
    for change in ({"caches": cache}, {"caches": [cache[:2]]}, {"caches": [cache[:, ::2]]}, {"caches": [cache, cache]}, {"caches": [cache.cpu()]}, {"caches": [cache[:, :48].contiguous()]},
                   {"caches": [cache[:, 0, 0].contiguous()]}, {"caches": [counts]}, {"parents": parents.long()}, {"out": (table, counts)}, {"caches": [None]}, {"caches": [torch.zeros((3, 64), device="cuda", requires_grad=True)]}):
        with pytest.raises(CompileError):
            pages.fork(**{"caches": [cache], "block_table": table, "counts": counts, "parents": parents, "lengths": lengths, "page_rows": 64, **change})
    pages.compact([cache], table, counts)
    for change in ({"caches": [cache[:2]]}, {"places": counts}, {"places": torch.empty(3, device="cuda")}, {"counts": i32([[1, 0, 0]])}, {"caches": [cache, cache[1:]]}):
        with pytest.raises(CompileError):
            pages.compact(**{"caches": [cache], "block_table": table, "counts": counts, **change})
    assert ops.status()[0] == 0


def test_captured_and_replayed():
    """A step in a graph that works on the program's own tensors: replays continue where the last one ended. On two streams at the same time."""
    rng, streams, work = random.Random(4), [torch.cuda.Stream() for _ in range(2)], []
    for k, s in enumerate(streams):
        table, counts, lengths = state_of(rng, 30, 20, 400, 64, empty=0.0)
        given, growing = (tensor(table, 20), i32(counts)), i32(lengths)
        cache = torch.randint(0, 256, (400, 64, 32), dtype=torch.uint8, device="cuda")
        other = torch.empty_like(given[0])
        parents = [rng.randrange(30) for _ in range(30)]
        work.append([s, None, given, growing, cache, (table, counts, lengths), parents, i32(parents), other])
    pages.resize(*work[0][2], work[0][3], page_rows=64)
    for item in work:
        s, _, given, growing, cache, _, _, parents, other = item
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            growing.add_(3).clamp_(max=20 * 64)
            pages.resize(*given, growing, page_rows=64, out=given)
            pages.fork([cache], *given, parents, growing, page_rows=64, out=(other, given[1]))
            given[0].copy_(other)
            growing.copy_(growing[parents.long()])
            pages.compact([cache], *given, out=given)
        item[1] = graph
    expected = [[item[4].clone(), *item[5]] for item in work]
    torch.cuda.synchronize()
    for _ in range(4):
        for s, graph, *_ in work:
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for (s, graph, given, growing, cache, _, parents, _, _), (held, table, counts, lengths) in zip(work, expected):
        for _ in range(4):
            lengths = [min(length + 3, 20 * 64) for length in lengths]
            table, counts = resized(table, counts, lengths, 64)
            table, counts, (held,) = forked([held], table, counts, parents, lengths, 64)
            lengths = [lengths[p] for p in parents]
            table, counts, _, (held,) = compacted([held], table, counts)
        same(given, table, counts, 20)
        assert torch.equal(cache, held) and growing.tolist() == lengths


@pytest.mark.parametrize("block", [1, 16, 64])
def test_a_program_that_serves(block):
    """Prompts, steps, samples of a prompt, ends, compaction: a cache in 8 bits whose pages the calls hand out, against rows kept one by one on the host."""
    rng, page_rows, entries, blocks, heads = random.Random(block), 64, 6, 40, 8
    cache = torch.zeros((blocks, page_rows, 1, 576), dtype=torch.uint8, device="cuda").view(E.HELD)
    scales = torch.zeros((blocks, page_rows // block), dtype=torch.uint8, device="cuda").view(E.SCALE)
    inv_freq, generator = latent.rotary_frequencies(64), torch.Generator(device="cuda").manual_seed(7)
    table, counts = i32([[-1] * entries] * 4), i32([0] * blocks)
    rows = [torch.zeros((0, 576), dtype=torch.float64, device="cuda") for _ in range(4)]  # what each request has been given, turned
    for step in range(14):
        if step % 4 == 2:
            parents = [rng.randrange(len(rows)) for _ in range(rng.randrange(2, 6))]
            table, counts = pages.fork([cache, scales], table, counts, i32(parents), i32([len(r) for r in rows]), page_rows=page_rows)
            rows = [rows[p].clone() for p in parents]
        if step % 5 == 3:
            table, counts, _ = pages.compact([cache, scales], table, counts)
            assert not bool((counts[int((counts > 0).sum()) :] > 0).any())
        new = [rng.choice([1, 1, 2, 5, 70 if len(r) < 200 else 1]) for r in rows]
        if step == 8:  # one ends, another begins in its place
            rows[0] = rows[0][:0]
            table, counts = pages.resize(table, counts, i32([len(r) for r in rows]), page_rows=page_rows)
        if step == 11:  # a request goes back a long way, into pages that others share
            rows[1] = rows[1][: len(rows[1]) // 2]
            table, counts = pages.fork([cache, scales], table, counts, i32(list(range(len(rows)))), i32([len(r) for r in rows]), page_rows=page_rows)
        lengths = [len(r) + n for r, n in zip(rows, new)]
        table, counts = pages.resize(table, counts, i32(lengths), page_rows=page_rows)
        tokens = sum(new)
        given = torch.randn((tokens, 576), device="cuda", generator=generator).bfloat16()
        cu = i32([0, *itertools.accumulate(new)])
        latent8.rotary_append8(given[:, :512], given[:, 512:], cache, scales, table, cu, i32(lengths), inv_freq)
        q = torch.randn((tokens, heads, 576), device="cuda", generator=generator).bfloat16()
        out = latent8.latent_attention8(q, cache, scales, table, cu, i32(lengths), scale=0.04)
        assert ops.status()[0] == 0
        wide, token = E.values(cache, scales), 0
        for b, (n, length) in enumerate(zip(new, lengths)):
            turned = R.turn(given[token : token + n, 512:], torch.arange(length - n, length, device="cuda"), inv_freq, "interleaved")
            rows[b] = torch.cat([rows[b], torch.cat([given[token : token + n, :512].double(), turned], 1)])
            own = wide[table[b, : -(-length // page_rows)].long()].view(-1, 576)[:length]
            # rounded once to 2^-4, and subnormal numbers (below 2^-6 of a scale of at most 2^-6) by half a step of theirs for every growth
            assert ((own - rows[b]).abs() <= 2.0 ** -4 * rows[b].abs() + 2.0 ** -11).all()
            seen = torch.arange(length, device="cuda") < (length - n + 1 + torch.arange(n, device="cuda"))[:, None]
            expected, _, error, _ = R.attention(q[token : token + n], own[None], own[None, :, :512], seen, 0.04)
            R.within(out[token : token + n], expected, error, f"step {step}, request {b}")
            token += n
        flat = [p for p in table.flatten().tolist() if p >= 0]
        assert counts.tolist() == [flat.count(p) for p in range(blocks)]


@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_a_compiled_step_is_the_eager_one(backend):
    def step(cache, scales, table, counts, lengths, parents, rows, q, cu, inv_freq):
        table, counts = pages.resize(table, counts, lengths, page_rows=64)
        latent8.rotary_append8(rows[:, :512], rows[:, 512:], cache, scales, table, cu, lengths, inv_freq)
        out = latent8.latent_attention8(q, cache, scales, table, cu, lengths, scale=0.04)
        table, counts = pages.fork([cache, scales], table, counts, parents, lengths, page_rows=64)
        return out, *pages.compact([cache, scales], table, counts)

    generator = torch.Generator(device="cuda").manual_seed(1)
    rows, q = (torch.randn(shape, device="cuda", generator=generator).bfloat16() for shape in ((3, 576), (3, 8, 576)))
    results = []
    for compiled in (False, True):
        cache = torch.zeros((9, 64, 1, 576), dtype=torch.uint8, device="cuda").view(E.HELD)
        scales = torch.zeros((9, 4), dtype=torch.uint8, device="cuda").view(E.SCALE)
        torch._dynamo.reset()
        call = torch.compile(step, backend=backend, fullgraph=True) if compiled else step
        got = call(cache, scales, i32([[8, -1, -1], [3, -1, -1]]), i32([0, 0, 0, 1, 0, 0, 0, 0, 1]), i32([66, 1]), i32([0, 0, 1, 0]), rows, q, i32([0, 2, 3]), latent.rotary_frequencies(64))
        results.append([cache.view(torch.uint8), scales.view(torch.uint8), *got])
    assert all(torch.equal(a, b) for a, b in zip(*results)) and ops.status()[0] == 0
