"""The operators around dense latent attention from their definitions, in 64 bits, and what their roundings allow."""

import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def turn(x, positions, inv_freq, layout, amplitude=1.0, inverse=False):
    """x [T, ..., 2 P] in 64 bits, turned."""
    x, pairs = x.double(), len(inv_freq)
    angle = positions.double()[:, None] * inv_freq.double() * (-1 if inverse else 1)
    angle = angle.view(len(positions), *(1,) * (x.dim() - 2), pairs)
    out = torch.empty_like(x)
    first, second = (slice(0, pairs), slice(pairs, None)) if layout == "half" else (slice(0, None, 2), slice(1, None, 2))
    out[..., first] = amplitude * (x[..., first] * angle.cos() - x[..., second] * angle.sin())
    out[..., second] = amplitude * (x[..., first] * angle.sin() + x[..., second] * angle.cos())
    return out


def turn_tolerance(x, expected, pairs, amplitude=1.0):
    """Half a step of the output's type; in FP32 two products, one sum, cosine, sine and amplitude to a few units of 2^-24, an angle to 2^-24 of half a turn."""
    size = amplitude * x.double().abs()[..., -2 * pairs:].amax(-1, keepdim=True)
    return HALF_STEP[x.dtype] * expected.abs() + 16 * 2.0 ** -24 * size


def append(latent, rope, cache, table, counts, lengths, inv_freq, layout, amplitude=1.0):
    """The cache after the append, in 64 bits; rows without a legal page are left out."""
    cache = cache.double().clone()
    blocks, page_rows, _, _ = cache.shape
    token = 0
    for b, (n, length) in enumerate(zip(counts, lengths)):
        for j in range(n):
            position = length - n + j
            if 0 <= position // page_rows < table.shape[1] and 0 <= int(table[b, position // page_rows]) < blocks:
                turned = turn(rope[token : token + 1], torch.tensor([position], device=rope.device), inv_freq, layout, amplitude)[0]
                cache[int(table[b, position // page_rows]), position % page_rows, 0] = torch.cat([latent[token].double(), turned])
            token += 1
    return cache


def attention(q, k, v, seen, scale, sinks=None):
    """One request: q [n, H, D], k and v [H or 1, L, ...] in storage types, seen [n, L] truth values. (out, lse, allowed error of out, of lse).

    Allowed: the output's half step; every weight rounded by half a step to the storage type in front of the second product; scores summed in
    FP32 (their error moves weight and denominator alike), exponentials and sums to 2^-18. All but the first scale with the
    weighted sum of the values' magnitudes.
    """
    step, features = HALF_STEP[q.dtype], q.shape[2]
    q, k, v = q.double().transpose(0, 1), k.double(), v.double()
    scores = scale * q @ k.transpose(1, 2)
    magnitude = scale * q.abs() @ k.abs().transpose(1, 2)
    scores = scores.masked_fill(~seen, -torch.inf)
    if k.shape[1]:
        score_error = features * 2.0 ** -24 * magnitude.masked_fill(~seen, 0.0).amax(-1, keepdim=True)
        most = scores.amax(-1, keepdim=True)
    else:
        score_error, most = torch.zeros_like(q[..., :1]), torch.full_like(q[..., :1], -torch.inf)
    if sinks is not None:
        most = torch.maximum(most, sinks.double()[:, None, None])
    most = most.masked_fill(most == -torch.inf, 0.0)
    weights = torch.exp(scores - most)
    total = weights.sum(-1, keepdim=True)
    empty = total == 0
    if sinks is not None:
        total = total + torch.exp(sinks.double()[:, None, None] - most)
    weights = weights / total.masked_fill(total == 0, 1.0)
    out = (weights @ v).masked_fill(empty, 0.0)
    size = weights @ v.abs()
    error = (step * (1 + step) + 2 * score_error + 2.0 ** -18) * size
    error = error + step * (out.abs() + error)
    # what is below the storage type's normal range is off by its smallest step
    error = error + (2.0 ** -24 if step == 2.0 ** -11 else 2.0 ** -133) + (2.0 ** -25 * v.abs().amax() * k.shape[1] if step == 2.0 ** -11 and k.shape[1] else 0.0)
    lse = (total.log() + most).squeeze(-1)
    lse_error = (score_error + 2.0 ** -18).squeeze(-1) + 2.0 ** -22 * lse.nan_to_num(0, 0, 0).abs()
    return out.transpose(0, 1), lse.transpose(0, 1), error.transpose(0, 1), lse_error.transpose(0, 1)


def within(actual, expected, allowed, label=""):
    actual = actual.double()
    same = (actual == expected)  # infinities
    off = (actual - expected).abs()
    bad = ~(same | (off <= allowed))
    assert not bad.any(), (f"{label}: {int(bad.sum())} of {bad.numel()} values outside, first at {bad.nonzero()[0].tolist()}: "
                           f"{actual[bad][0].item()} for {expected[bad][0].item()}, allowed {allowed.expand_as(off)[bad][0].item()}")
