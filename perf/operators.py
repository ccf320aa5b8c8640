"""Operators around dense latent attention, as a serving program calls them, and their plain forms.

  rotary   the queries' rope part, rotated out of a projection into the buffer that attention reads
  append   a step's new rows into the paged latent cache, their rope part rotated on the way
  absorbed attention of a step's queries over the paged latent cache (one row per token is key and value)
  expanded attention of prompts with keys and values per head and one shared rope key per token

A case gives sizes and options only. Request lengths follow from the case (so the work of a pass does), everything
else (contents, page permutations, positions) from the seed.
"""

import math
import random

import torch

own = False

VALUES, ROPE, NOPE = 512, 64, 128  # value features of a latent row; rope features; features per head without rope
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def _case(kind, requests, queries, context, **options):
    # queries, context: the longest request's new tokens and its length including them
    # ragged: requests of different lengths, as continuous batching makes them
    # layout: pairs of neighbours ("interleaved") or of halves ("half"); scaled: frequencies for contexts eight times the trained one
    # width: features of a cache row; sinks: a logit per head in the denominator; lse: also the log of the denominator
    case = {"kind": kind, "requests": requests, "queries": queries, "context": context, "heads": 64, "dtype": "bf16", "ragged": False,
            "layout": "interleaved", "scaled": False, "width": 576, "page": 128, "sinks": False, "lse": False, "causal": True}
    case.update(options)
    return case


def listed():
    return [
        # One user's next token: the rope part of 64 heads.
        _case("rotary", 1, 1, 8192, name="rotary_1x1"),
        # Draft verification for 128 requests far into their contexts: pairs of halves, scaled frequencies.
        _case("rotary", 128, 6, 131072, layout="half", scaled=True, dtype="f16", name="rotary_128x6"),
        # A prefill chunk.
        _case("rotary", 1, 8192, 32768, scaled=True, name="rotary_8k"),
        # New rows of a decode batch of requests of different ages.
        _case("append", 64, 6, 8192, ragged=True, layout="half", page=64, name="append_64x6"),
        # New rows of a prefill chunk.
        _case("append", 1, 8192, 32768, scaled=True, name="append_8k"),
        # One user, one token: what an interactive session waits for between two tokens.
        _case("absorbed", 1, 1, 8192, name="decode_1x1_8k"),
        # An ordinary large decode batch: the cache is read once and nothing else counts.
        _case("absorbed", 64, 1, 32768, name="decode_64x1_32k"),
        # Draft verification (five drafts and one token): products count as much as bytes.
        _case("absorbed", 32, 6, 16384, lse=True, name="decode_32x6_16k"),
        # A quarter of the heads (heads shared out over four devices), rows of 512, sinks, half, odd lengths.
        _case("absorbed", 23, 5, 50011, heads=16, dtype="f16", ragged=True, width=512, page=64, sinks=True, name="ragged_23_f16_h16"),
        # A whole prompt.
        _case("expanded", 1, 8192, 8192, lse=True, name="prefill_8k_8k"),
        # The next chunk of a long prompt, 16 heads.
        _case("expanded", 1, 2048, 16384, heads=16, dtype="f16", name="prefill_2k_16k_f16"),
        # Prompts and chunks of odd lengths in one call.
        _case("expanded", 17, 1500, 2011, ragged=True, name="prefill_ragged_17"),
    ]


def _log(rng, low, high):
    """A whole number, spread evenly over the logarithm."""
    return min(high, max(low, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    kind = rng.choice(["rotary", "append", "absorbed", "absorbed", "absorbed", "expanded", "expanded"])
    heads = rng.choice([64, 64, 128, 16, 8, 24, 1])
    options = {"heads": heads, "dtype": rng.choice(["bf16", "bf16", "f16"]), "ragged": rng.random() < 0.5, "page": rng.choice([64, 128]),
               "layout": rng.choice(["interleaved", "half"]), "scaled": rng.random() < 0.5, "lse": rng.random() < 0.5}
    if kind in ("rotary", "append"):
        requests = _log(rng, 1, 128)
        queries = _log(rng, 1, 8192 // requests)
        context = _log(rng, queries, 131072 if kind == "rotary" else max(queries, 262144 // requests))
        if kind == "rotary":
            options["heads"] = min(heads, 64)
        else:
            options["width"] = rng.choice([512, 576])
    elif kind == "absorbed":
        options["width"], options["sinks"] = rng.choice([576, 576, 512]), rng.random() < 0.3
        requests, queries = _log(rng, 1, 128), _log(rng, 1, 8)
        context = _log(rng, 300, 131072)
        if rng.random() < 0.2:  # a chunk of a prompt
            requests, queries = _log(rng, 1, 4), _log(rng, 9, 500)
        # no more rows and products than the largest listed cases
        context = max(queries, min(context, 64 * 32768 // requests, 32 * 6 * 64 * 16384 // (requests * queries * heads)))
    else:
        options["causal"] = rng.random() < 0.8
        requests, queries = _log(rng, 1, 24), _log(rng, 1, 4096)
        queries = min(queries, 16384 // requests)
        context = _log(rng, queries, max(queries, 16384 // requests))
        heads = options["heads"] = min(heads, max(1, 8192 * 4096 * 64 // (requests * queries * context)))
    return _case(kind, requests, queries, context, **options)


def _lengths(case):
    """New tokens and whole length of every request. The first is the longest; in a ragged call about half of the
    others bring one token and the rest several."""
    counts, lengths = [case["queries"]], [case["context"]]
    rng = random.Random("%d %d %d" % (case["requests"], case["queries"], case["context"]))
    for _ in range(case["requests"] - 1):
        if case["ragged"]:
            counts.append(1 if rng.random() < 0.5 else _log(rng, 1, case["queries"]))
            lengths.append(_log(rng, min(max(counts[-1], 64), case["context"]), case["context"]))
        else:
            counts.append(case["queries"])
            lengths.append(case["context"])
    return counts, lengths


def _inverse_frequencies(case):
    """Radians per position of every pair, in 64 bits. Scaled: pairs that turn less than once within the trained 4096 positions
    are slowed down eightfold, those that turn more than 32 times are left, the ones between are interpolated."""
    half = ROPE // 2
    exponent = torch.arange(half, dtype=torch.float64, device="cuda") / half
    plain = 10000.0 ** -exponent
    if not case["scaled"]:
        return plain

    def pair_of(turns):
        return half * math.log(4096 / (turns * 2 * math.pi)) / math.log(10000.0)

    low, high = max(math.floor(pair_of(32.0)), 0), min(math.ceil(pair_of(1.0)), half - 1)
    ramp = ((torch.arange(half, dtype=torch.float64, device="cuda") - low) / (high - low)).clamp(0, 1)
    return plain * (1 - ramp) + plain / 8 * ramp


def _normal(shape, dtype, generator):
    return torch.randn(shape, dtype=dtype, device="cuda", generator=generator)


def _offsets(counts):
    return torch.tensor([0] + counts, device="cuda").cumsum(0).to(torch.int32)


def prepare(case, seed):
    generator = torch.Generator(device="cuda")
    generator.manual_seed(seed)
    counts, lengths = _lengths(case)
    kind, dtype, heads, tokens = case["kind"], TYPES[case["dtype"]], case["heads"], sum(counts)
    state = {"case": case, "most_queries": max(counts), "most_keys": max(lengths), "cu_seqlens_q": _offsets(counts),
             "seqused_kv": torch.tensor(lengths, dtype=torch.int32, device="cuda"),
             "amplitude": 0.1 * math.log(8.0) + 1.0 if case["scaled"] else 1.0}
    if kind in ("rotary", "append"):
        state["inv_freq"] = _inverse_frequencies(case)
    if kind == "rotary":
        count = torch.tensor(counts, device="cuda")
        request = torch.repeat_interleave(torch.arange(len(counts), device="cuda"), count)
        first = torch.tensor(lengths, device="cuda") - count - state["cu_seqlens_q"][:-1]
        state["positions"] = (torch.arange(tokens, device="cuda") + first[request]).to(torch.int32)
        state["projected"] = _normal((tokens, heads, NOPE + ROPE), dtype, generator)  # rope is its last part
        state["q"] = _normal((tokens, heads, VALUES + ROPE), dtype, generator)  # what attention reads: the rope goes to its last part
        return state
    if kind == "expanded":
        state["cu_seqlens_k"] = _offsets(lengths)
        state["q"] = _normal((tokens, heads, NOPE + ROPE), dtype, generator)
        state["kv"] = _normal((sum(lengths), heads, 2 * NOPE), dtype, generator)  # one projection: keys, then values
        state["k_rope"] = _normal((sum(lengths), ROPE), dtype, generator)
        return state
    width, page = case["width"], case["page"]
    pages = -(-case["context"] // page)
    used = [-(-length // page) for length in lengths]
    order = torch.randperm(sum(used), device="cuda", generator=generator).to(torch.int32)
    index = torch.arange(pages, device="cuda")
    first = torch.tensor([0] + used, device="cuda").cumsum(0)
    places = first[:-1, None] + index
    state["block_table"] = torch.where(index < torch.tensor(used, device="cuda")[:, None], order[places.clamp(max=sum(used) - 1)], -1).to(torch.int32)
    state["cache"] = _normal((sum(used), page, 1, width), dtype, generator)
    if kind == "append":
        state["latent"] = _normal((tokens, width - ROPE), dtype, generator)
        state["projected"] = _normal((tokens, width), dtype, generator)  # rope is its last part
        return state
    state["q"] = _normal((tokens, heads, width), dtype, generator)
    state["scale"] = 192 ** -0.5
    state["sinks"] = _normal((heads,), torch.float32, generator) if case["sinks"] else None
    return state


def _rotated(x, positions, state):
    """Plain rotation of `x` [T, ..., ROPE] in 32 bits, angles in 64."""
    angle = positions.double()[:, None] * state["inv_freq"]
    shape = (len(positions),) + (1,) * (x.dim() - 2) + (ROPE // 2,)
    cos, sin = (angle.cos() * state["amplitude"]).float().view(shape), (angle.sin() * state["amplitude"]).float().view(shape)
    x = x.float()
    if state["case"]["layout"] == "half":
        a, b = x[..., : ROPE // 2], x[..., ROPE // 2 :]
        return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)


def _request_of(state):
    """Request and place of every token."""
    cu = state["cu_seqlens_q"].long()
    tokens = torch.arange(state["q" if "q" in state else "latent"].shape[0], device="cuda")
    request = torch.searchsorted(cu[1:].contiguous(), tokens, right=True)
    return request, tokens - cu[request]


def _plain_append(state):
    cache, table, page = state["cache"], state["block_table"].long(), state["case"]["page"]
    request, place = _request_of(state)
    count = state["cu_seqlens_q"].long().diff()
    position = state["seqused_kv"].long()[request] - count[request] + place
    row = table[request, position // page] * page + position % page
    rope = _rotated(state["projected"][:, -ROPE:], position, state)
    cache.view(-1, cache.shape[-1])[row] = torch.cat([state["latent"].float(), rope], 1).to(cache.dtype)
    return cache


def _softmax_values(scores, mask, values, sinks):
    """Softmax over the last axis where `mask`, times `values`: (out, log of the denominator), in the type of the scores. Rows without keys give zeros."""
    scores.masked_fill_(~mask, -math.inf)
    most = scores.amax(-1, keepdim=True)
    if sinks is not None:
        most = torch.maximum(most, sinks)
    most = most.masked_fill(most == -math.inf, 0.0)
    weights = scores.sub_(most).exp_()
    total = weights.sum(-1, keepdim=True)
    empty = total == 0
    if sinks is not None:
        total = total + (sinks - most).exp()
    out = weights @ values / total.masked_fill(total == 0, 1.0)
    return out.masked_fill(empty, 0.0), (total.log() + most).squeeze(-1)


def _plain_absorbed(state):
    q, cache, table, heads = state["q"], state["cache"], state["block_table"].long(), state["case"]["heads"]
    request, place = _request_of(state)
    count, most = state["cu_seqlens_q"].long().diff(), state["most_queries"]
    padded = torch.zeros((len(count), most, heads, q.shape[-1]), device="cuda")
    padded[request, place] = q.float()
    rows = cache.float()[table.clamp(min=0)].view(len(count), -1, q.shape[-1])[:, : state["most_keys"]]
    scores = (padded.view(len(count), most * heads, -1) @ rows.transpose(1, 2)).mul_(state["scale"])
    end = state["seqused_kv"].long()[:, None] - count[:, None] + torch.arange(most, device="cuda") + 1
    mask = torch.arange(rows.shape[1], device="cuda") < end.repeat_interleave(heads, 1)[..., None]
    sinks = state["sinks"].repeat(most)[None, :, None] if state["sinks"] is not None else None
    out, lse = _softmax_values(scores, mask, rows[..., :VALUES], sinks)
    return {"out": out.view(len(count), most, heads, VALUES)[request, place].to(q.dtype),
            "lse": lse.view(len(count), most, heads)[request, place] if state["case"]["lse"] else None}


def _plain_expanded(state):
    q, kv, case = state["q"], state["kv"], state["case"]
    request, place = _request_of(state)
    count, length = state["cu_seqlens_q"].long().diff(), state["seqused_kv"].long()
    most, keys = state["most_queries"], state["most_keys"]
    padded = torch.zeros((len(count), most, case["heads"], q.shape[-1]), device="cuda")
    padded[request, place] = q.float()
    index = torch.arange(keys, device="cuda")
    row = (state["cu_seqlens_k"].long()[:-1, None] + index).clamp(max=kv.shape[0] - 1)
    row = torch.where(index < length[:, None], row, 0)
    k, v = kv[row].float().split(NOPE, -1)
    rope = state["k_rope"][row].float()
    scores = padded[..., :NOPE].transpose(1, 2) @ k.permute(0, 2, 3, 1)
    scores.add_(padded[..., NOPE:].transpose(1, 2) @ rope.transpose(1, 2)[:, None])
    scores.mul_((NOPE + ROPE) ** -0.5)
    end = length[:, None] - count[:, None] + torch.arange(most, device="cuda") + 1 if case["causal"] else length[:, None].expand(-1, most)
    out, lse = _softmax_values(scores, (index < end[..., None])[:, None], v.transpose(1, 2), None)
    return {"out": out.transpose(1, 2)[request, place].to(q.dtype), "lse": lse.transpose(1, 2)[request, place] if case["lse"] else None}


def _call(state):
    """The framework's operators."""
    from ascendflow_b200 import latent

    case, kind = state["case"], state["case"]["kind"]
    if kind == "rotary":
        latent.rotary(state["projected"][..., NOPE:], state["positions"], state["inv_freq"], layout=case["layout"],
                      amplitude=state["amplitude"], out=state["q"][..., VALUES:])
        return state["q"][..., VALUES:]
    if kind == "append":
        return latent.rotary_append(state["latent"], state["projected"][:, -ROPE:], state["cache"], state["block_table"], state["cu_seqlens_q"],
                                    state["seqused_kv"], state["inv_freq"], layout=case["layout"], amplitude=state["amplitude"])
    lse = torch.empty(state["q"].shape[:2], dtype=torch.float32, device="cuda") if case["lse"] else None
    if kind == "absorbed":
        out = latent.latent_attention(state["q"], state["cache"], state["block_table"], state["cu_seqlens_q"], state["seqused_kv"],
                                      scale=state["scale"], sinks=state["sinks"], lse=lse)
    else:
        out = latent.latent_prefill(state["q"], state["kv"][..., :NOPE], state["kv"][..., NOPE:], state["k_rope"], state["cu_seqlens_q"],
                                    state["cu_seqlens_k"], scale=(NOPE + ROPE) ** -0.5, causal=case["causal"], lse=lse)
    return {"out": out, "lse": lse}


def run(state):
    if own:
        return _call(state)
    kind = state["case"]["kind"]
    if kind == "rotary":
        out = state["q"][..., VALUES:]
        out.copy_(_rotated(state["projected"][..., NOPE:], state["positions"], state))
        return out
    return {"append": _plain_append, "absorbed": _plain_absorbed, "expanded": _plain_expanded}[kind](state)


def work(case):
    counts, lengths = _lengths(case)
    kind, heads, tokens = case["kind"], case["heads"], sum(counts)
    tables = 4 * (2 * len(counts) + 1)
    if kind == "rotary":
        values = tokens * heads * ROPE
        return {"bytes": 4 * values + 4 * tokens + 4 * ROPE, "flops": 3 * values}
    pages = 4 * sum(-(-length // case["page"]) for length in lengths)
    if kind == "append":
        written = -(-max(counts) // case["page"]) + 1  # page numbers read per request, at most
        return {"bytes": 4 * tokens * case["width"] + tables + min(pages, 4 * written * len(counts)) + 4 * ROPE, "flops": 3 * tokens * ROPE}
    # (query, key) pairs that are not masked
    if case["causal"]:
        pairs = sum(n * (length - n) + n * (n + 1) // 2 for n, length in zip(counts, lengths))
    else:
        pairs = sum(n * length for n, length in zip(counts, lengths))
    lse = 4 * tokens * heads if case["lse"] else 0
    if kind == "absorbed":
        width = case["width"]
        return {"bytes": 2 * sum(lengths) * width + 2 * tokens * heads * (width + VALUES) + lse + tables + pages,
                "flops": 2 * pairs * heads * (width + VALUES)}
    return {"bytes": 2 * sum(lengths) * (heads * 2 * NOPE + ROPE) + 2 * tokens * heads * (2 * NOPE + ROPE) + lse + tables,
            "flops": 2 * pairs * heads * (2 * NOPE + ROPE)}


def _exact_rotation(x, angle, amplitude, layout):
    """The pairs as complex numbers, turned."""
    x = x.double()
    half = ROPE // 2
    pairs = torch.complex(x[..., :half], x[..., half:]) if layout == "half" else torch.view_as_complex(x.reshape(*x.shape[:-1], half, 2).contiguous())
    turned = pairs * torch.polar(torch.full_like(angle, amplitude), angle)
    return torch.cat([turned.real, turned.imag], -1) if layout == "half" else torch.view_as_real(turned).flatten(-2)


def _exact_attention(q, k, v, scale, ends, sinks):
    """One request, one block of queries: q [n, H, D], k [H or 1, L, D], v [H or 1, L, E], query i sees keys below ends[i]."""
    scores = torch.einsum("nhd,hld->hnl", q, k.expand(q.shape[1], -1, -1)) * scale
    scores = torch.where(torch.arange(k.shape[1], device="cuda") < ends[:, None], scores, torch.full_like(scores, -math.inf))
    if sinks is not None:
        scores = torch.cat([scores, sinks.double()[:, None, None].expand(-1, len(q), 1)], -1)
    lse = torch.logsumexp(scores, -1)
    weights = torch.softmax(scores, -1).masked_fill((ends <= 0)[:, None], 0.0)[..., : k.shape[1]]
    return torch.einsum("hnl,hle->nhe", weights, v.expand(q.shape[1], -1, -1)), lse.T


def exact(case, seed):
    state = prepare(case, seed)
    counts, lengths = _lengths(case)
    kind = case["kind"]
    if kind == "rotary":
        angle = state["positions"].double()[:, None, None] * state["inv_freq"]
        return _exact_rotation(state["projected"][..., NOPE:], angle, state["amplitude"], case["layout"])
    if kind == "append":
        cache = state["cache"].double()
        token = 0
        for b, (n, length) in enumerate(zip(counts, lengths)):
            positions = torch.arange(length - n, length, device="cuda")
            rope = _exact_rotation(state["projected"][token : token + n, -ROPE:], positions.double()[:, None] * state["inv_freq"],
                                   state["amplitude"], case["layout"])
            page = state["block_table"][b].long()[positions // case["page"]]
            cache[page, positions % case["page"], 0] = torch.cat([state["latent"][token : token + n].double(), rope], 1)
            token += n
        return cache
    outs, lses, token, first = [], [], 0, 0
    for b, (n, length) in enumerate(zip(counts, lengths)):
        q = state["q"][token : token + n].double()
        if kind == "absorbed":
            pages = state["block_table"][b, : -(-length // case["page"])].long()
            k = state["cache"][pages].double().view(1, -1, case["width"])[:, :length]
            v, scale = k[..., :VALUES], state["scale"]
        else:
            kv = state["kv"][first : first + length].double().transpose(0, 1)
            rope = state["k_rope"][first : first + length].double().expand(case["heads"], -1, -1)
            k, v, scale = torch.cat([kv[..., :NOPE], rope], -1), kv[..., NOPE:], (NOPE + ROPE) ** -0.5
        ends = torch.arange(length - n + 1, length + 1, device="cuda") if case["causal"] else torch.full((n,), length, device="cuda")
        step = max(1, (1 << 28) // (length * case["heads"]))
        for i in range(0, n, step):
            out, lse = _exact_attention(q[i : i + step], k, v, scale, ends[i : i + step], state.get("sinks"))
            outs.append(out)
            lses.append(lse)
        token, first = token + n, first + length
    return {"out": torch.cat(outs), "lse": torch.cat(lses) if case["lse"] else None}
