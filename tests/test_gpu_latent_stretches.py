"""Long contexts whose outputs show every stretch of the keys: each 64 of them have values in a feature of their own, all positive, so that one stretch that is
left out, taken twice or read from another place changes the output by far more than roundings may."""

import pytest
import torch

from ascendflow_b200 import latent, ops
from tests import latent_reference as R

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16
STRETCH = 64


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def marked(dtype, keys, features, seed, shift=0):
    """[keys, features]: row i has a value from 0.5 to 1.5 in feature i / 64 + shift alone (features repeat where there are more stretches)."""
    generator = torch.Generator(device="cuda").manual_seed(seed)
    values = torch.zeros((keys, features), device="cuda")
    index = torch.arange(keys, device="cuda")
    values[index, (index // STRETCH + shift) % features] = torch.rand(keys, device="cuda", generator=generator) + 0.5
    return values.to(dtype)


def check(out, q, k, v, scale, ends):
    """out [n, H, E] of q [n, H, D], k and v [H or 1, L, .], query i sees keys below ends[i]. Scores are at most about 1, sums of 64 products at most.

    Allowed: what `latent_reference.attention` allows for scores, exponentials and roundings of weights and output (its roundings are relative to sums of
    magnitudes, which are the outputs themselves here), weights being about as large as the row's greatest; and FP32 sums of terms of one sign, 16
    keys at a time, each addition off by 2^-23 of the sum."""
    length, q, k, v = k.shape[1], q.double().transpose(0, 1), k.double(), v.double()
    scores = (scale * q @ k.transpose(1, 2)).masked_fill(torch.arange(length, device="cuda") >= ends[:, None], -torch.inf)
    weights = torch.softmax(scores, -1)
    expected, step = weights @ v, R.HALF_STEP[out.dtype]
    magnitude = scale * (q.abs() @ k.abs().transpose(1, 2)).amax()
    relative = step * (1 + step) + 2 * 64 * 2.0 ** -24 * magnitude + 2.0 ** -18 + 2 * length / 16 * 2.0 ** -23
    error = relative * expected
    error = error + step * (expected + error) + (2.0 ** -24 if out.dtype == F16 else 2.0 ** -133)
    R.within(out.transpose(0, 1), expected, error)
    # Every stretch that a row sees whole can be told from none.
    count = length // STRETCH
    parts = (weights * v.sum(-1)[:, None])[..., : count * STRETCH].unflatten(-1, (count, STRETCH)).sum(-1)  # [H, n, stretches]
    owner = v[:, : count * STRETCH : STRETCH].argmax(-1)[:, None].expand(*parts.shape)
    whole = ends[:, None] >= STRETCH * torch.arange(1, count + 1, device="cuda")
    assert (parts > 4 * error.gather(-1, owner))[whole.expand(*parts.shape)].all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,queries,lengths", [(64, 1, [70001]), (16, 3, [40000]), (64, 2, [9000, 4000, 8777]), (9, 1, [12000, 11900, 500, 11000]), (64, 1, [3000] * 40), (3, 50, [5000])])
def test_absorbed(dtype, heads, queries, lengths):
    pages = [-(-length // 128) for length in lengths]
    order = torch.randperm(sum(pages), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).int()
    table = torch.full((len(lengths), max(pages)), -1, dtype=torch.int32, device="cuda")
    cache = torch.full((sum(pages), 128, 1, 576), float("nan"), dtype=dtype, device="cuda")
    rows, first = [], 0
    generator = torch.Generator(device="cuda").manual_seed(2)
    for b, (length, count) in enumerate(zip(lengths, pages)):
        own = torch.cat([marked(dtype, length, 512, b, shift=7 * b), (torch.randn((length, 64), device="cuda", generator=generator) * 0.25).to(dtype)], 1)
        table[b, :count] = order[first : first + count]
        padded = torch.full((count * 128, 576), float("nan"), dtype=dtype, device="cuda")
        padded[:length] = own
        cache[table[b, :count].long()] = padded.view(count, 128, 1, 576)
        rows.append(own)
        first += count
    q = torch.zeros((queries * len(lengths), heads, 576), device="cuda")
    q[..., 512:] = torch.randn((*q.shape[:2], 64), device="cuda", generator=generator) * 0.25
    q = q.to(dtype)
    cu = i32([queries * b for b in range(len(lengths) + 1)])
    out = latent.latent_attention(q, cache, table, cu, i32(lengths), scale=0.1)
    assert ops.status()[0] == 0
    for b, own in enumerate(rows):
        part = slice(queries * b, queries * (b + 1))
        ends = torch.arange(lengths[b] - queries + 1, lengths[b] + 1, device="cuda")
        # (queries see the decisive features alone)
        check(out[part], q[part, :, 512:], own[None, :, 512:], own[None, :, :512], 0.1, ends)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,counts,lengths", [(1, [1], [20000]), (16, [3], [5000]), (5, [300], [4001]), (2, [257, 1, 130], [2000, 5000, 7001]), (74, [2], [1664]), (75, [2], [1664]), (80, [130], [3000]), (3, [700], [700])])
def test_expanded(dtype, causal, heads, counts, lengths):
    generator = torch.Generator(device="cuda").manual_seed(3)
    keys = sum(lengths)
    q = (torch.randn((sum(counts), heads, 192), device="cuda", generator=generator) * 0.25).to(dtype)
    q[..., :128] = 0  # scores by the rope part alone
    kv = torch.empty((keys, heads, 256), dtype=dtype, device="cuda")
    kv[..., :128] = torch.randn((keys, heads, 128), device="cuda", generator=generator).to(dtype)
    rope = (torch.randn((keys, 64), device="cuda", generator=generator) * 0.25).to(dtype)
    first = 0
    for b, length in enumerate(lengths):
        for head in range(heads):
            kv[first : first + length, head, 128:] = marked(dtype, length, 128, 10 * b + head, shift=5 * head + b)
        first += length
    starts = [i32([sum(n[:b]) for b in range(len(n) + 1)]) for n in (counts, lengths)]
    out = latent.latent_prefill(q, kv[..., :128], kv[..., 128:], rope, *starts, scale=0.1, causal=causal)
    assert ops.status()[0] == 0
    token = first = 0
    for n, length in zip(counts, lengths):
        part, keys_of = slice(token, token + n), slice(first, first + length)
        ends = torch.arange(length - n + 1, length + 1, device="cuda") if causal else torch.full((n,), length, device="cuda")
        check(out[part], q[part, :, 128:], rope[keys_of][None], kv[keys_of, :, 128:].transpose(0, 1), 0.1, ends)
        token, first = token + n, first + length
