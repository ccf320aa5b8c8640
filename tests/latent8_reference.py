"""A latent cache held in 8 bits from its definitions, in 64 bits."""

import math

import torch

from tests import latent_reference as R

HELD, SCALE = torch.float8_e4m3fn, torch.float8_e8m0fnu
MOST = 448.0


def scales_of(scale_bytes):
    """What bytes stand for, in 64 bits."""
    e = scale_bytes.view(torch.uint8).long()
    return torch.where(e == 255, math.nan, (e - 127 + 1023 << 52).view(torch.float64))


def values(cache, scales):
    """What a cache stands for [BLOCKS, PAGE_ROWS, 1, W], in 64 bits."""
    block = cache.shape[1] // scales.shape[1]
    return cache.float().double() * scales_of(scales).repeat_interleave(block, 1)[..., None, None]


def rounded(x):
    """To the nearest e4m3 number (finite, of at most 448)."""
    return x.to(torch.float32).to(HELD)


def append(latent, rope, cache, scales, table, counts, lengths, inv_freq, layout, amplitude=1.0):
    """For every block that gets rows: (page, block of the page, first row, rows in 64 bits, allowed error of these, the greatest magnitude, scale byte and older rows' numbers
    before). Rows without a legal page are left out."""
    blocks, page_rows, _, _ = cache.shape
    per_scale = page_rows // scales.shape[1]
    found, token = [], 0
    for b, (n, length) in enumerate(zip(counts, lengths)):
        start = length - n
        if n:
            positions = torch.arange(start, length, device=rope.device)
            turned = R.turn(rope[token : token + n], positions, inv_freq, layout, amplitude)
            rows = torch.cat([latent[token : token + n].double(), turned], 1)
            if latent.dtype == torch.float16:
                rows = torch.where(rows.isfinite(), rows.clamp(-61440, 61440), rows)
            size = amplitude * rope[token : token + n].double().abs().amax(-1, keepdim=True)
            error = torch.cat([torch.zeros_like(latent[token : token + n].double()), (16 * 2.0 ** -24 * size).expand_as(turned)], 1)
            first = max(start, 0)
            while first < length:
                last = min(length, (first // per_scale + 1) * per_scale)
                column = first // page_rows
                page = int(table[b, column]) if column < table.shape[1] else -1
                if 0 <= page < blocks:
                    place = first % page_rows
                    block = place // per_scale
                    older = cache[page, block * per_scale : place, 0].clone()
                    byte = int(scales.view(torch.uint8)[page, block])
                    own = slice(first - start, last - start)
                    found.append((page, block, place, rows[own], error[own], rows[own].abs().max().item(), byte, older))
                first = last
        token += n
    return found


def check_append(found, cache, scales):
    """The cache and scales behind the call against `found`; returns the bytes of everything else, to be compared with what was there."""
    per_scale = cache.shape[1] // scales.shape[1]
    bytes_, numbers = scales.view(torch.uint8), cache.float().double()
    for page, block, place, rows, error, most, had, older in found:
        byte = int(bytes_[page, block])
        begins = place % per_scale == 0
        if not math.isfinite(most):
            assert byte == 255
            continue
        slack = error.max().item()
        least = [max(0, 127 + math.ceil(math.log2(m / MOST))) if m > 0 else 0 for m in (max(most - slack, 0), most + slack)]
        allowed = {e if begins else max(e, had) for e in least}
        assert byte in allowed, (page, block, byte, allowed)
        scale = 2.0 ** (byte - 127)
        if older.numel():
            assert torch.equal(cache[page, block * per_scale : place, 0].float(), rounded(older.float() * 2.0 ** (had - byte)).float())
        held = numbers[page, place : place + len(rows), 0] * scale
        # half a step: 2^-4 of the value, or of the smallest normal number
        R.within(held, rows, 2.0 ** -4 * rows.abs().clamp(min=2.0 ** -6 * scale) + error + 2.0 ** -126, (page, block))
    return found
