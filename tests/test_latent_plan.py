"""How the absorbed attention call is dealt to blocks, on the CPU and from the kernel's source (`latent_plan.cpp`): every chunk that a tile's rows see is some
block's, once; what several blocks have of a tile is found again by the kernel that adds it up."""

import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest

ROOT = Path(__file__).resolve().parents[1]
ROWS, CHUNK = 64, 64


def plan_text(source):
    constants = source[source.index("constexpr int kRows = 64"):source.index("constexpr uint32_t kColumnsQ")]
    piece = source[source.index("// What a block does next"):source.index("template <int kWidth>\nstruct Layout")]
    bars = source[source.index("enum Bar {"):source.index("__device__ __forceinline__ bool warp_wait(")]
    plan = source[source.index("// A request's tiles and what they cost"):source.index("// Everybody's way through the pieces.")]
    text = constants + piece + bars + plan
    assert "asm" not in text
    return text


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("no C++ compiler")
    folder = tmp_path_factory.mktemp("plan")
    (folder / "plan.inc").write_text(plan_text((ROOT / "ascendflow_b200/csrc/latent_attention.cu").read_text()))
    subprocess.run(["g++", "-std=c++17", "-O2", "-w", f"-I{folder}", str(ROOT / "tests/latent_plan.cpp"), "-o", str(folder / "plan")], check=True)

    def run(blocks, heads, counts, lengths, pages, page_rows):
        cu = np.concatenate([[0], np.cumsum(counts)])
        words = np.concatenate([[blocks, heads, len(counts), pages, page_rows, cu[-1]], cu, lengths]).astype(np.int32)
        result = subprocess.run([folder / "plan"], input=words.tobytes(), capture_output=True, timeout=600)
        assert result.returncode == 0, result.stderr.decode()
        words, at, pieces, records = np.frombuffer(result.stdout, dtype=np.int64), 0, [], []
        for _ in range(blocks):
            own = []
            while words[at + 7] >= 0:
                own.append(dict(zip(("row", "rows", "request", "token", "head", "base", "length", "first", "last", "slot"), words[at : at + 10].tolist())))
                at += 10
            records.append(dict(zip(("row", "rows", "head", "last", "empty"), words[at + 10 : at + 15].tolist())))
            at += 15
            pieces.append(own)
        assert at == len(words)
        return pieces, records
    return run


def check(plan, blocks, heads, counts, lengths, pages=1 << 20, page_rows=64):
    pieces, records = plan(blocks, heads, counts, lengths, pages, page_rows)
    found = {}
    for block, own in enumerate(pieces):
        for piece in own:
            found.setdefault(piece["row"], []).append((block, piece))
    capacity, begin, loads = pages * page_rows, 0, [sum(p["last"] - p["first"] for p in own) for own in pieces]
    for request, (count, length) in enumerate(zip(counts, lengths)):
        length = max(length, 0)
        for start in range(0, count * heads, ROWS):
            rows = min(ROWS, count * heads - start)
            seen = min(max(length - count + (start + rows - 1) // heads + 1, 0), capacity + 1)
            chunks, row = -(-seen // CHUNK), begin * heads + start
            parts = found.pop(row)
            at = 0
            for block, piece in parts:
                assert (piece["rows"], piece["request"], piece["token"], piece["head"]) == (rows, request, start // heads, start % heads)
                assert piece["base"] == length - count + 1 and piece["length"] == min(length, capacity + 1)
                assert piece["first"] == at and (piece["last"] > at or chunks == 0)
                at = piece["last"]
            assert at == chunks
            if len(parts) == 1:
                assert parts[0][1]["slot"] == -1
                continue
            first, last = parts[0][0], parts[-1][0]
            assert records[first] | {"empty": 0} == dict(row=row, rows=rows, head=start % heads, last=records[first]["last"], empty=0)
            # what is added up: slot 2 i + 1 of the first, slots 2 i of those up to `last` that have not said that theirs is empty
            members = [first] + [i for i in range(first + 1, records[first]["last"] + 1) if not records[i]["empty"]]
            assert members == [block for block, _ in parts] and records[first]["last"] >= last
            assert [piece["slot"] for _, piece in parts] == [2 * first + 1] + [2 * block for block, _ in parts[1:]]
        begin += count
    assert not found
    for block, record in enumerate(records):  # nobody else leads
        assert record["last"] < 0 or any(piece["slot"] == 2 * block + 1 for piece in pieces[block])
    return loads


@pytest.mark.parametrize("blocks,heads,counts,lengths", [
    (148, 64, [1], [8192]), (148, 64, [1], [1]), (148, 64, [6] * 32, [16384] * 32), (148, 64, [1] * 100, [400] * 100), (148, 64, [1] * 64, [32768] * 64),
    (148, 16, [5, 1, 0, 4, 2], [50011, 4023, 700, 0, 16978]), (7, 1, [300], [300]), (148, 65, [0, 0, 0], [5, 5, 5]), (20, 128, [3, 1], [2, 100000]), (148, 64, [500], [500]),
    (132, 64, [2] * 75, [640] * 75), (1, 24, [9, 1], [3000, 10]),
])
def test_every_chunk_is_some_blocks_once(plan, blocks, heads, counts, lengths):
    check(plan, blocks, heads, counts, lengths)


def test_random_batches(plan):
    rng = np.random.default_rng(5)
    for _ in range(25):
        requests, blocks, heads = int(rng.choice([1, 3, 30, 90])), int(rng.choice([1, 5, 24, 37])), int(rng.choice([1, 5, 16, 64, 65, 128]))
        counts = rng.choice([0, 1, 1, 2, 6, 40, 200], requests).tolist()
        lengths = (rng.random(requests) ** 3 * rng.choice([50, 3000, 200000])).astype(int).tolist()
        lengths[0] = int(rng.choice([-4, 0, lengths[0]]))
        check(plan, blocks, heads, counts, lengths, pages=int(rng.choice([1 << 20, 20])), page_rows=int(rng.choice([64, 128])))


def test_more_requests_than_a_block_has_threads(plan):
    rng = np.random.default_rng(6)
    for requests in (512, 513, 1100):
        counts = rng.choice([0, 1, 1, 3], requests).tolist()
        counts[-1] = 70
        check(plan, 9, 16, counts, (rng.random(requests) * 900).astype(int).tolist())


def test_stretches_are_even_and_tiles_side_by_side(plan):
    loads = check(plan, 148, 64, [1] * 64, [32768] * 64)
    assert max(loads) <= sum(loads) / 148 + 1
    # 32 requests of six tiles on 144 blocks: at every time the six blocks that work on a request are at the same chunk
    pieces, _ = plan(148, 64, [6] * 32, [16384] * 32, 1 << 20, 64)
    assert [len(own) for own in pieces[144:]] == [0] * 4
    for block in range(24):
        ways = [[(p["request"], p["first"], p["last"]) for p in pieces[block + 24 * tile]] for tile in range(6)]
        assert all(way == ways[0] for way in ways)
    # one tile for each of 100 blocks: none is shared
    pieces, _ = plan(148, 64, [1] * 100, [400] * 100, 1 << 20, 64)
    assert sorted(len(own) for own in pieces) == [0] * 48 + [1] * 100


@pytest.mark.parametrize("heads,count,requests,length,stretch", [(64, 1, 8, 8192, 18), (64, 1, 3, 8192, 49), (64, 1, 32, 2048, 4), (16, 2, 16, 8192, 9), (64, 6, 4, 8192, 6), (64, 1, 1, 8192, 64)])
def test_tiles_alike_have_blocks_of_their_own(plan, heads, count, requests, length, stretch):
    loads = check(plan, 148, heads, [count] * requests, [length] * requests)
    pieces, _ = plan(148, heads, [count] * requests, [length] * requests, 1 << 20, 64)
    tiles = requests * -(-heads * count // ROWS)
    assert [len(own) for own in pieces] == [1] * (tiles * stretch) + [0] * (148 - tiles * stretch)
    assert max(loads) == -(-(-(-length // CHUNK)) // stretch)


@pytest.mark.parametrize("requests,seed", [(2, 0), (12, 2), (33, 4), (60, 5), (148, 7)])
def test_ragged_tiles_have_blocks_of_their_own(plan, requests, seed):
    rng = np.random.default_rng(seed)
    lengths = rng.integers(1000, 9000, requests).tolist()
    loads = check(plan, 148, 64, [1] * requests, lengths)
    pieces, _ = plan(148, 64, [1] * requests, lengths, 1 << 20, 64)
    if requests <= 60:  # (with more of them a block of their own for each would be too long a stretch)
        assert max(len(own) for own in pieces) == 1
    # no stretch is longer than the mean by more than ten chunks, rounding, or a whole tile that is not worth sharing
    assert max(loads) <= sum(loads) / 148 + 10 + 2 or max(len(own) for own in pieces) <= 2
    check(plan, 148, 64, [1] * requests, [0] * (requests - 1) + [9000])
    check(plan, 148, 16, [1] * requests, lengths)
    check(plan, 148, 16, [1] * (requests - 1) + [400], lengths)  # (a request's tiles differ)
