"""Operators around a latent cache held in 8 bits, and around the pages of a cache, as a serving program calls them, and their plain forms.

  append     a step's new rows, their rope part turned on the way, into the paged cache in 8 bits with a scale per block of rows
  attention  of a step's queries over that cache (one row per token is key and value of all heads)
  resize     pages for requests that grew, pages given back by those that ended or were cut
  fork       rows of the block table continued by any number of others (samples, beams), the partly filled page copied
  compact    the pages in use moved to the front of the cache

A case gives sizes and options only. Lengths, which request continues which and which pages are in use follow from the case (so the work of a
pass does), everything else (contents, which page is whose) from the seed.
"""

import math
import random

import numpy as np
import torch

own = False

VALUES, ROPE = 512, 64  # value features of a latent row; its turned features, where it has any
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def _rows_case(kind, requests, queries, context, **options):
    # queries, context: the longest request's new tokens and its length including them
    # ragged: requests of different lengths, as continuous batching makes them; block: rows that share a scale
    case = {"kind": kind, "requests": requests, "queries": queries, "context": context, "heads": 64, "dtype": "bf16", "ragged": False, "width": 576,
            "page": 128, "block": 1, "layout": "interleaved", "sinks": False, "lse": False}
    case.update(options)
    return case


def _pages_case(kind, requests, context, **options):
    # requests: rows of the block table; beams: neighbours that share what they have in common; layers: caches that the pages are of
    # held: e4m3 (a cache of bytes and its scales) or bf16; fill: share of the pages in use
    case = {"kind": kind, "requests": requests, "context": context, "beams": 1, "layers": 1, "held": "e4m3", "page": 128, "fill": 0.8}
    case.update(options)
    return case


def listed():
    return [
        # New rows of a decode batch of requests of different ages, five drafts each.
        _rows_case("append", 64, 6, 8192, ragged=True, layout="half", page=64, block=16, name="append8_64x6"),
        # New rows of a prefill chunk.
        _rows_case("append", 1, 8192, 32768, block=64, name="append8_8k"),
        # One user, one token: what an interactive session waits for between two tokens.
        _rows_case("attention", 1, 1, 8192, block=64, name="decode8_1x1_8k"),
        # An ordinary large decode batch: the cache is read once and nothing else counts.
        _rows_case("attention", 64, 1, 32768, name="decode8_64x1_32k"),
        # Draft verification (five drafts and one token): products count as much as bytes.
        _rows_case("attention", 32, 6, 16384, block=64, lse=True, name="decode8_32x6_16k"),
        # A quarter of the heads (heads shared out over four devices), rows of 512, sinks, half, odd lengths.
        _rows_case("attention", 23, 5, 50011, heads=16, dtype="f16", ragged=True, width=512, page=64, block=16, sinks=True, name="ragged8_23_f16_h16"),
        # A small batch between two steps: most requests keep their pages.
        _pages_case("resize", 16, 4096, page=64, name="resize_16"),
        # A large batch of long contexts: the whole table is looked through.
        _pages_case("resize", 1024, 131072, page=64, name="resize_1024"),
        # Four prompts with four beams each.
        _pages_case("fork", 16, 2048, beams=4, page=64, name="fork_16"),
        # A batch of beams over the layers of a group: what is copied counts.
        _pages_case("fork", 512, 4096, beams=8, layers=8, held="bf16", name="fork_512"),
        # A small cache.
        _pages_case("compact", 8, 1024, page=64, name="compact_8"),
        # Caches of several layers of which a fifth has been given back.
        _pages_case("compact", 96, 8192, layers=4, name="compact_96"),
    ]


def _log(rng, low, high):
    """A whole number, spread evenly over the logarithm."""
    return min(high, max(low, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    kind = rng.choice(["append", "append", "attention", "attention", "attention", "attention", "resize", "resize", "fork", "fork", "compact", "compact"])
    page = rng.choice([64, 128])
    if kind in ("resize", "fork", "compact"):
        options = {"page": page, "held": rng.choice(["e4m3", "bf16"]), "fill": rng.choice([0.5, 0.8, 0.95])}
        if kind == "resize":
            requests = _log(rng, 1, 1024)
            return _pages_case(kind, requests, _log(rng, 100, 131072), **options)
        options["layers"] = _log(rng, 1, 8)
        if kind == "fork":
            options["beams"] = rng.choice([1, 2, 4, 8])
            requests = options["beams"] * _log(rng, 1, 512 // options["beams"])
            return _pages_case(kind, requests, _log(rng, 10, 4096), **options)
        requests = _log(rng, 1, 96)
        # no more bytes than the largest listed case
        return _pages_case(kind, requests, _log(rng, 100, min(65536, 4 * 96 * 8192 // (2 * options["layers"] * requests))), **options)
    options = {"heads": rng.choice([64, 64, 128, 16, 8, 24, 1]), "dtype": rng.choice(["bf16", "bf16", "f16"]), "ragged": rng.random() < 0.5, "page": page,
               "block": rng.choice([1, 1, 2, 16, 32, 64, 64]), "layout": rng.choice(["interleaved", "half"]), "width": rng.choice([576, 576, 512])}
    if kind == "append":
        requests = _log(rng, 1, 128)
        queries = _log(rng, 1, 8192 // requests)
        return _rows_case(kind, requests, queries, _log(rng, queries, max(queries, 262144 // requests)), **options)
    options["sinks"], options["lse"] = rng.random() < 0.3, rng.random() < 0.5
    requests, queries = _log(rng, 1, 128), _log(rng, 1, 8)
    context = _log(rng, 300, 131072)
    if rng.random() < 0.2:  # a chunk of a prompt
        requests, queries = _log(rng, 1, 4), _log(rng, 9, 500)
    # no more rows and products than the largest listed cases
    context = max(queries, min(context, 64 * 32768 // requests, 32 * 6 * 64 * 16384 // (requests * queries * options["heads"])))
    return _rows_case(kind, requests, queries, context, **options)


def _own_rng(case):
    """A generator that follows from the case."""
    return random.Random(" ".join("%s=%s" % (key, case[key]) for key in sorted(case) if key != "name"))


def _lengths(case):
    """New tokens and whole length of every request. The first is the longest; in a ragged call about half of the
    others bring one token and the rest several."""
    counts, lengths = [case["queries"]], [case["context"]]
    rng = _own_rng(case)
    for _ in range(case["requests"] - 1):
        if case["ragged"]:
            counts.append(1 if rng.random() < 0.5 else _log(rng, 1, case["queries"]))
            lengths.append(_log(rng, min(max(counts[-1], 64), case["context"]), case["context"]))
        else:
            counts.append(case["queries"])
            lengths.append(case["context"])
    return counts, lengths


def _pool(case):
    """What the case says of a cache's pages: lengths now, lengths to come (resize), who continues whom (fork), how many first pages a request shares
    with its neighbour in front, pages of the cache, and which of them are in use."""
    rng, page, requests, beams = _own_rng(case), case["page"], case["requests"], case["beams"]
    lengths, later, parents, shared = [], [], [], []
    for b in range(requests):
        if b % beams:
            lengths.append(lengths[-1])
        else:
            lengths.append(case["context"] if b == 0 else _log(rng, max(1, case["context"] // 16), case["context"]))
        fate = rng.random()
        if fate < 0.1:  # ended, or not begun
            later.append(0)
        elif fate < 0.2:
            later.append(lengths[-1])
            lengths[-1] = 0 if case["kind"] == "resize" and b else lengths[-1]
        elif fate < 0.3:  # drafts that were not taken
            later.append(max(0, lengths[-1] - rng.randrange(1, 8)))
        else:
            later.append(min(case["context"], lengths[-1] + rng.randrange(1, 8)))
        parents.append(b - b % beams + rng.randrange(beams) if beams > 1 else (b if fate < 0.8 else rng.randrange(requests)))
        neighbour = b > 0 and (b % beams or case["kind"] == "resize" and b % 4 == 1)
        shared.append(min(lengths[b], lengths[b - 1]) // page // (1 if b % beams else 2) if neighbour else 0)
    used = sum(-(-length // page) - s for length, s in zip(lengths, shared))
    if case["kind"] == "compact":
        blocks = max(used + 1, int(used / case["fill"]))
    else:  # room for all that may be wanted
        blocks = used + sum(-(-length // page) for length in later) // 8 + requests + 8
        blocks = max(blocks, int(blocks / case["fill"]) if case["kind"] == "fork" else sum(-(-length // page) for length in later) + 8)
    return lengths, later, parents, shared, blocks, sorted(rng.sample(range(blocks), used))


def _copies(case):
    """(request that continues, rows of its last page) for everyone but the first to continue a request with a partly filled page."""
    lengths, _, parents, _, _, _ = _pool(case)
    seen, found = set(), []
    for child, parent in enumerate(parents):
        rest = lengths[parent] % case["page"]
        if parent in seen and rest:
            found.append((child, rest))
        seen.add(parent)
    return found


def _normal(shape, dtype, generator):
    return torch.randn(shape, dtype=dtype, device="cuda", generator=generator)


def _offsets(counts):
    return torch.tensor([0] + counts, device="cuda").cumsum(0).to(torch.int32)


def _exponents(most):
    """Least k with most <= 448 * 2^k (whole numbers from -127 to 127)."""
    mantissa, exponent = torch.frexp(most)
    return (exponent - 9 + (mantissa > 0.875)).clamp(-127, 127).masked_fill(most == 0, -127)


def _scales(exponents):
    return (exponents + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _held(pages, case, generator):
    """A cache of rows in 8 bits, and its scales. Rows differ in size, as those of real caches do."""
    page, block, width = case["page"], case.get("block", 1), case.get("width", VALUES + ROPE)
    cache = torch.empty((pages, page, 1, width), dtype=torch.float8_e4m3fn, device="cuda")
    scales = torch.empty((pages, page // block), dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 27) // (page * width))
    for first in range(0, pages, step):
        rows = _normal((min(step, pages - first), page // block, block, width), torch.float32, generator)
        rows *= torch.exp(0.3 * _normal((*rows.shape[:3], 1), torch.float32, generator))
        exponents = _exponents(rows.abs().amax((2, 3)))
        scales[first : first + step] = (exponents + 127).to(torch.uint8)
        cache[first : first + step] = torch.ldexp(rows, -exponents[:, :, None, None]).to(torch.float8_e4m3fn).view(-1, page, 1, width)
    return cache, scales.view(torch.float8_e8m0fnu)


def _prepare_pages(case, seed, generator):
    lengths, later, parents, shared, blocks, used = _pool(case)
    page, entries = case["page"], -(-case["context"] // case["page"]) + 1
    mine = np.array(used, dtype=np.int32)
    np.random.default_rng(seed).shuffle(mine)
    table, at = np.full((len(lengths), entries), -1, dtype=np.int32), 0
    for b, length in enumerate(lengths):
        n = -(-length // page)
        table[b, : shared[b]] = table[b - 1, : shared[b]]
        table[b, shared[b] : n] = mine[at : at + n - shared[b]]
        at += n - shared[b]
    counts = np.bincount(table[table >= 0], minlength=blocks)
    state = {"case": case, "table": torch.from_numpy(table).cuda(), "counts": torch.from_numpy(counts.astype(np.int32)).cuda(), "used": len(used),
             "lengths": torch.tensor(later if case["kind"] == "resize" else lengths, dtype=torch.int32, device="cuda")}
    if case["kind"] == "resize":
        return state
    state["parents"] = torch.tensor(parents, dtype=torch.int32, device="cuda")
    state["caches"] = []
    for _ in range(case["layers"]):
        if case["held"] == "e4m3":
            state["caches"] += _held(blocks, {"page": page, "block": 16}, generator)
        else:
            state["caches"].append(_normal((blocks, page, 1, VALUES + ROPE), torch.bfloat16, generator))
    return state


def prepare(case, seed):
    generator = torch.Generator(device="cuda")
    generator.manual_seed(seed)
    if case["kind"] in ("resize", "fork", "compact"):
        return _prepare_pages(case, seed, generator)
    counts, lengths = _lengths(case)
    dtype, tokens, width, page = TYPES[case["dtype"]], sum(counts), case["width"], case["page"]
    state = {"case": case, "most_queries": max(counts), "most_keys": max(lengths), "cu_seqlens_q": _offsets(counts),
             "seqused_kv": torch.tensor(lengths, dtype=torch.int32, device="cuda")}
    pages = -(-case["context"] // page)
    used = [-(-length // page) for length in lengths]
    order = torch.randperm(sum(used), device="cuda", generator=generator).to(torch.int32)
    index = torch.arange(pages, device="cuda")
    first = torch.tensor([0] + used, device="cuda").cumsum(0)
    places = first[:-1, None] + index
    state["block_table"] = torch.where(index < torch.tensor(used, device="cuda")[:, None], order[places.clamp(max=sum(used) - 1)], -1).to(torch.int32)
    state["cache"], state["scales"] = _held(sum(used), case, generator)
    if case["kind"] == "append":
        state["inv_freq"] = 10000.0 ** -(torch.arange(ROPE // 2, dtype=torch.float64, device="cuda") / (ROPE // 2))
        size = torch.exp(0.3 * _normal((tokens, 1), torch.float32, generator))
        state["latent"] = (_normal((tokens, width - ROPE), torch.float32, generator) * size).to(dtype)
        state["projected"] = (_normal((tokens, width), torch.float32, generator) * size).to(dtype)  # rope is its last part
        return state
    state["q"] = _normal((tokens, case["heads"], width), dtype, generator)
    state["scale"] = 192 ** -0.5
    state["sinks"] = _normal((case["heads"],), torch.float32, generator) if case["sinks"] else None
    return state


def _request_of(state, tokens):
    """Request and place of every token."""
    cu = state["cu_seqlens_q"].long()
    tokens = torch.arange(tokens, device="cuda")
    request = torch.searchsorted(cu[1:].contiguous(), tokens, right=True)
    return request, tokens - cu[request]


def _plain_append(state):
    case, latent, cache = state["case"], state["latent"], state["cache"]
    page, block, width = case["page"], case["block"], case["width"]
    request, place = _request_of(state, len(latent))
    position = state["seqused_kv"].long()[request] - state["cu_seqlens_q"].long().diff()[request] + place
    row = state["block_table"].long()[request, position // page] * page + position % page
    angle = position.double()[:, None] * state["inv_freq"]
    cos, sin = angle.cos().float(), angle.sin().float()
    rope = state["projected"][:, -ROPE:].float()
    if case["layout"] == "half":
        a, b = rope[:, : ROPE // 2], rope[:, ROPE // 2 :]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    else:
        a, b = rope[:, 0::2], rope[:, 1::2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    rows = torch.cat([latent.float(), turned], 1)
    # scales: of every block the greatest of what its new rows need and, where older rows precede them, of what it has
    old = state["scales"].view(torch.uint8).view(-1).int() - 127
    nothing = torch.full_like(old, -128)
    need = nothing.scatter_reduce(0, row // block, _exponents(rows.abs().amax(1)), "amax")
    begin = torch.full_like(old, block).scatter_reduce(0, row // block, (row % block).int(), "amin")  # first new row of the block
    new = torch.where(need == -128, old, torch.where(begin > 0, torch.maximum(old, need), need))
    shift = torch.where(need == -128, 0, old - new)[:, None, None]
    older = torch.arange(block, device="cuda") < begin[:, None]
    held = cache.view(-1, block, width)
    held.copy_(torch.where(older[..., None] & (shift != 0), torch.ldexp(held.float(), shift), held.float()).to(cache.dtype))
    cache.view(-1, width).view(torch.uint8)[row] = torch.ldexp(rows, -new[row // block][:, None]).to(cache.dtype).view(torch.uint8)
    state["scales"].view(torch.uint8).view(-1).copy_(new + 127)
    return {"cache": cache, "scales": state["scales"]}


def _plain_attention(state):
    case, q, table, heads = state["case"], state["q"], state["block_table"].long(), state["case"]["heads"]
    request, place = _request_of(state, len(q))
    count, most = state["cu_seqlens_q"].long().diff(), state["most_queries"]
    padded = torch.zeros((len(count), most, heads, q.shape[-1]), device="cuda")
    padded[request, place] = q.float()
    held = state["cache"].view(torch.uint8)[table.clamp(min=0)].view(state["cache"].dtype).float()  # [B, pages, page, 1, width]
    size = state["scales"].view(torch.uint8)[table.clamp(min=0)].view(state["scales"].dtype).float()
    rows = held.view(*size.shape, case["block"], -1).mul_(size[..., None, None]).view(len(count), -1, q.shape[-1])[:, : state["most_keys"]]
    scores = (padded.view(len(count), most * heads, -1) @ rows.transpose(1, 2)).mul_(state["scale"])
    end = state["seqused_kv"].long()[:, None] - count[:, None] + torch.arange(most, device="cuda") + 1
    seen = torch.arange(rows.shape[1], device="cuda") < end.repeat_interleave(heads, 1)[..., None]
    scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    if state["sinks"] is not None:
        top = torch.maximum(top, state["sinks"].repeat(most)[None, :, None])
    top = top.masked_fill(top == -math.inf, 0.0)
    weights = scores.sub_(top).exp_()
    total = weights.sum(-1, keepdim=True)
    if state["sinks"] is not None:
        total = total + (state["sinks"].repeat(most)[None, :, None] - top).exp()
    out = weights @ rows[..., :VALUES] / total.masked_fill(total == 0, 1.0)
    lse = (total.log() + top).view(len(count), most, heads)
    return {"out": out.view(len(count), most, heads, VALUES)[request, place].to(q.dtype), "lse": lse[request, place] if case["lse"] else None}


def _in_order(flags, values, places):
    """`values` where `flags`, in order, in the first of `places` places; behind them the last again (zeros where there is none)."""
    rank = flags.long().cumsum(0) - 1
    found = torch.zeros(places + 1, dtype=torch.long, device="cuda").scatter_(0, torch.where(flags, rank, places).clamp(max=places), values)
    last = flags.sum().clamp(max=places) - 1
    return found[torch.minimum(torch.arange(places, device="cuda"), last.clamp(min=0))] * (last >= 0)


def _plain_resize(state):
    table, counts, page = state["table"].long(), state["counts"].long(), state["case"]["page"]
    blocks, entries = len(counts), table.shape[1]
    wanted = torch.arange(entries, device="cuda") < ((state["lengths"].long().clamp(min=0) + page - 1) // page)[:, None]
    have = (table >= 0) & (table < blocks)
    counts = counts.scatter_add(0, torch.where(have, table, 0).view(-1), -(have & ~wanted).long().view(-1))
    free = counts == 0
    lacking = (wanted & ~have).view(-1)
    rank = lacking.long().cumsum(0) - 1
    given = lacking & (rank < free.sum())
    numbers = _in_order(free, torch.arange(blocks, device="cuda"), blocks)
    page_of = torch.where(given, numbers[rank.clamp(0, blocks - 1)], -1).view_as(table)
    counts = counts.scatter_add(0, page_of.clamp(min=0).view(-1), given.long())
    return {"table": torch.where(wanted & have, table, page_of).int(), "counts": counts.int()}


def _plain_fork(state):
    table, counts, page = state["table"].long(), state["counts"].long(), state["case"]["page"]
    blocks, entries, children = len(counts), table.shape[1], len(state["parents"])
    parents = state["parents"].long()
    inside = (parents >= 0) & (parents < len(table))
    parents = parents.clamp(0, len(table) - 1)
    length = (state["lengths"].long().clamp(0, entries * page)[parents]) * inside
    index = torch.arange(entries, device="cuda")
    rows = torch.where(index < ((length + page - 1) // page)[:, None], table[parents], -1)
    rows = torch.where((rows >= 0) & (rows < blocks), rows, -1)
    order = torch.arange(children, device="cuda")
    first = torch.full((len(table) + 1,), children, device="cuda").scatter_reduce(0, torch.where(inside, parents, len(table)), order, "amin")
    tail = (length // page).clamp(max=entries - 1)[:, None]  # the partly filled page's entry
    source = rows.gather(1, tail)[:, 0]
    wanting = inside & (first[parents] != order) & (length % page > 0) & (source >= 0)
    free = counts == 0
    rank = wanting.long().cumsum(0) - 1
    given = wanting & (rank < free.sum())
    target = torch.where(given, _in_order(free, torch.arange(blocks, device="cuda"), children)[rank.clamp(min=0)], -1)
    rows = rows.scatter(1, tail, torch.where(wanting, target, source)[:, None])
    had = (table >= 0) & (table < blocks)
    counts = counts.scatter_add(0, torch.where(had, table, 0).view(-1), -had.long().view(-1))
    counts = counts.scatter_add(0, rows.clamp(min=0).view(-1), (rows >= 0).long().view(-1))
    source, target, filled = (_in_order(given, v, children) for v in (source, target, length % page))
    for cache in state["caches"]:
        held = cache.view(torch.uint8)  # (bytes, whatever the type)
        each = page // held.shape[1]
        keep = (torch.arange(held.shape[1], device="cuda") * each < filled[:, None]).view(children, -1, *(1,) * (held.dim() - 2))
        held[target] = torch.where(keep, held[source], held[target])
    return {"table": rows.int(), "counts": counts.int(), "caches": state["caches"]}


def _plain_compact(state):
    table, counts, caches = state["table"].long(), state["counts"].long(), state["caches"]
    blocks, most = len(counts), max(1, min(state["used"], len(counts) - state["used"]))
    numbers, used = torch.arange(blocks, device="cuda"), counts > 0
    border = used.sum()
    source = _in_order(used & (numbers >= border), numbers, most)
    target = _in_order(~used & (numbers < border), numbers, most)
    places = torch.where(used, numbers, -1).scatter(0, source, torch.where(used[source], target, -1))
    moved = torch.where(places >= 0, places, blocks)
    counts = torch.zeros(blocks + 1, dtype=torch.long, device="cuda").scatter(0, moved, counts)[:blocks]
    for cache in caches:
        held = cache.view(torch.uint8)
        held[target] = held[source]
    renumbered = torch.where((table >= 0) & (table < blocks), places[table.clamp(0, blocks - 1)], table)
    return {"table": renumbered.int(), "counts": counts.int(), "places": places.int(), "caches": caches}


def _call(state):
    """The framework's operators."""
    from ascendflow_b200 import latent8, pages

    case, kind = state["case"], state["case"]["kind"]
    if kind == "append":
        latent8.rotary_append8(state["latent"], state["projected"][:, -ROPE:], state["cache"], state["scales"], state["block_table"], state["cu_seqlens_q"],
                               state["seqused_kv"], state["inv_freq"], layout=case["layout"])
        return {"cache": state["cache"], "scales": state["scales"]}
    if kind == "attention":
        lse = torch.empty(state["q"].shape[:2], dtype=torch.float32, device="cuda") if case["lse"] else None
        out = latent8.latent_attention8(state["q"], state["cache"], state["scales"], state["block_table"], state["cu_seqlens_q"], state["seqused_kv"],
                                        scale=state["scale"], sinks=state["sinks"], lse=lse)
        return {"out": out, "lse": lse}
    if kind == "resize":
        table, counts = pages.resize(state["table"], state["counts"], state["lengths"], page_rows=case["page"])
        return {"table": table, "counts": counts}
    if kind == "fork":
        table, counts = pages.fork(state["caches"], state["table"], state["counts"], state["parents"], state["lengths"], page_rows=case["page"])
        return {"table": table, "counts": counts, "caches": state["caches"]}
    table, counts, places = pages.compact(state["caches"], state["table"], state["counts"])
    return {"table": table, "counts": counts, "places": places, "caches": state["caches"]}


def run(state):
    if own:
        return _call(state)
    return {"append": _plain_append, "attention": _plain_attention, "resize": _plain_resize, "fork": _plain_fork, "compact": _plain_compact}[state["case"]["kind"]](state)


def work(case):
    if case["kind"] in ("resize", "fork", "compact"):
        lengths, _, parents, _, blocks, used = _pool(case)
        entries = 4 * len(lengths) * (-(-case["context"] // case["page"]) + 1)
        row = case["layers"] * (2 * (VALUES + ROPE) if case["held"] == "bf16" else VALUES + ROPE)
        if case["kind"] == "fork":
            scales = case["layers"] / 16 if case["held"] == "e4m3" else 0
            rows = sum(rest for _, rest in _copies(case))
            return {"bytes": 2 * entries + 8 * blocks + 8 * len(lengths) + int(2 * rows * (row + scales)), "flops": 0}
        if case["kind"] == "resize":
            return {"bytes": 2 * entries + 8 * blocks + 4 * len(lengths), "flops": 0}
        scales = case["layers"] * case["page"] // 16 if case["held"] == "e4m3" else 0
        moves = sum(number >= len(used) for number in used)
        return {"bytes": 2 * entries + 12 * blocks + 2 * moves * (case["page"] * row + scales), "flops": 0}
    counts, lengths = _lengths(case)
    tokens, width, heads = sum(counts), case["width"], case["heads"]
    tables = 4 * (2 * len(counts) + 1)
    pages = 4 * sum(-(-length // case["page"]) for length in lengths)
    if case["kind"] == "append":
        written = -(-max(counts) // case["page"]) + 1  # page numbers read per request, at most
        return {"bytes": 3 * tokens * width + -(-tokens // case["block"]) + tables + min(pages, 4 * written * len(counts)) + 4 * ROPE, "flops": 3 * tokens * ROPE}
    # (query, key) pairs that are not masked
    pairs = sum(n * (length - n) + n * (n + 1) // 2 for n, length in zip(counts, lengths))
    lse = 4 * tokens * heads if case["lse"] else 0
    return {"bytes": sum(lengths) * width + sum(-(-length // case["block"]) for length in lengths) + 2 * tokens * heads * (width + VALUES) + lse + tables + pages,
            "flops": 2 * pairs * heads * (width + VALUES)}


# ---- from the definitions, in 64 bits -------------------------------------------------------------------------------------


def _exact_append(state):
    """Request by request, block by block."""
    case = state["case"]
    page, block, layout = case["page"], case["block"], case["layout"]
    cache, scales = state["cache"].double(), state["scales"].double()
    cu, lengths = state["cu_seqlens_q"].tolist(), state["seqused_kv"].tolist()
    if sum(-(-(end - begin) // block) + 1 for begin, end in zip(cu, cu[1:])) > 4096:
        return None
    for b, length in enumerate(lengths):
        count, at = cu[b + 1] - cu[b], cu[b]
        first = length - count
        positions = torch.arange(first, length, device="cuda", dtype=torch.float64)
        rope = state["projected"][at : at + count, -ROPE:].double()
        half = ROPE // 2
        pairs = torch.complex(rope[:, :half], rope[:, half:]) if layout == "half" else torch.view_as_complex(rope.reshape(count, half, 2).contiguous())
        turned = pairs * torch.polar(torch.ones_like(pairs.real), positions[:, None] * state["inv_freq"])
        turned = torch.cat([turned.real, turned.imag], -1) if layout == "half" else torch.view_as_real(turned).flatten(-2)
        rows = torch.cat([state["latent"][at : at + count].double(), turned], 1)
        most = rows.abs().amax(1).tolist()
        pages = state["block_table"][b].tolist()
        while first < length:
            stop = min(length, (first // block + 1) * block)
            need = max(most[first - (length - count) : stop - (length - count)])
            size = 2.0 ** max(-127, math.ceil(math.log2(need / 448)))
            number, place = pages[first // page], first % page
            begin = place // block * block
            if begin < place:
                had = scales[number, place // block].item()
                size = max(size, had)
                cache[number, begin:place, 0] *= had / size
            scales[number, place // block] = size
            cache[number, place : place + stop - first, 0] = rows[first - (length - count) : stop - (length - count)] / size
            first = stop
    return {"cache": cache, "scales": scales}


def _exact_attention(state):
    case, outs, lses, token = state["case"], [], [], 0
    cu, lengths = state["cu_seqlens_q"].tolist(), state["seqused_kv"].tolist()
    for b, length in enumerate(lengths):
        n = cu[b + 1] - cu[b]
        pages = state["block_table"][b, : -(-length // case["page"])].long()
        held = state["cache"].view(torch.uint8)[pages].view(state["cache"].dtype).double().view(-1, case["width"])
        size = state["scales"].view(torch.uint8)[pages].view(state["scales"].dtype).double().view(-1)
        rows = (held * size.repeat_interleave(case["block"])[:, None])[:length]
        ends = torch.arange(length - n + 1, length + 1, device="cuda")
        step = max(1, (1 << 28) // (length * case["heads"]))
        for i in range(0, n, step):
            q = state["q"][token + i : token + min(n, i + step)].double()
            scores = torch.einsum("nhd,ld->nhl", q, rows) * state["scale"]
            scores = torch.where(torch.arange(length, device="cuda") < ends[i : i + step, None, None], scores, -math.inf)
            if state["sinks"] is not None:
                scores = torch.cat([scores, state["sinks"].double()[None, :, None].expand(len(q), -1, 1)], -1)
            lses.append(torch.logsumexp(scores, -1))
            outs.append(torch.einsum("nhl,le->nhe", torch.softmax(scores, -1)[..., :length], rows[:, :VALUES]))
        token += n
    return {"out": torch.cat(outs), "lse": torch.cat(lses) if case["lse"] else None}


def _exact_pages(state):
    """Page by page, on the host."""
    case, kind, page = state["case"], state["case"]["kind"], state["case"]["page"]
    table, counts, lengths = state["table"].tolist(), state["counts"].tolist(), state["lengths"].tolist()
    if kind == "resize":
        wanted = [-(-length // page) for length in lengths]
        for row, n in zip(table, wanted):
            for i in range(n, len(row)):
                if row[i] >= 0:
                    counts[row[i]] -= 1
                    row[i] = -1
        free = iter([p for p, count in enumerate(counts) if count == 0])
        for row, n in zip(table, wanted):
            for i in range(n):
                if row[i] < 0:
                    row[i] = next(free)
                    counts[row[i]] = 1
        return {"table": torch.tensor(table), "counts": torch.tensor(counts)}
    caches = [cache.double() for cache in state["caches"]]
    if kind == "fork":
        free = iter([p for p, count in enumerate(counts) if count == 0])
        rows, seen = [], set()
        for parent in state["parents"].tolist():
            n, rest = -(-lengths[parent] // page), lengths[parent] % page
            row = table[parent][:n] + [-1] * (len(table[parent]) - n)
            if parent in seen and rest:
                row[n - 1] = next(free)
                for cache in caches:
                    held = -(-rest * cache.shape[1] // page)
                    cache[row[n - 1], :held] = cache[table[parent][n - 1], :held]
            seen.add(parent)
            rows.append(row)
        counts = np.bincount([p for row in rows for p in row if p >= 0], minlength=len(counts))
        return {"table": torch.tensor(rows), "counts": torch.from_numpy(counts), "caches": caches}
    border = sum(count > 0 for count in counts)
    places = [p if count > 0 else -1 for p, count in enumerate(counts)]
    for source, target in zip([p for p in range(border, len(counts)) if counts[p] > 0], [p for p in range(border) if counts[p] == 0]):
        places[source] = target
        counts[target], counts[source] = counts[source], 0
        for cache in caches:
            cache[target] = cache[source]
    table = [[places[p] if p >= 0 else p for p in row] for row in table]
    return {"table": torch.tensor(table), "counts": torch.tensor(counts), "places": torch.tensor(places), "caches": caches}


def exact(case, seed):
    state = prepare(case, seed)
    return {"append": _exact_append, "attention": _exact_attention}.get(case["kind"], _exact_pages)(state)
