"""Small weights beside a dominant one: what most keys have in rows whose first key takes nearly all of the weight."""

import math

import pytest
import torch

from ascendflow_b200 import latent, ops
from tests import latent_reference as R

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16
SCALE = 0.125


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def peaked(dtype, keys, features, gap, seed):
    """One feature that decides the score of `keys` rows, and values: the first row above the others by about `gap` binades and without value, the others' values about 1."""
    generator = torch.Generator(device="cuda").manual_seed(seed)
    decides = (torch.rand(keys, device="cuda", generator=generator) - 0.5) * 0.5
    decides[0] = gap * math.log(2.0) / SCALE
    values = torch.rand((keys, features), device="cuda", generator=generator) + 0.5
    values[0] = 0
    return decides.to(dtype), values.to(dtype)


def check(out, dtype, decides, values, q):
    """Scores are single products, exact in FP32, and one product by the scale's (2^-24 of up to 64 binades; twice, since the reference has one too). Weights
    are rounded to the storage type by half a step or, where they are small, by 2^-25 (half) or 2^-134 (bfloat16) of a unit that
    is at most 2^-6 of the row's greatest weight (what a first reference leaves); exponentials to 2^-18; FP32 sums are of terms of one sign, 16 keys at a time at least, each addition off by 2^-23
    of the sum, once for the values and once for the denominator; the output by half a step."""
    score = SCALE * q.double() * decides.double()
    weights = torch.exp(score - score.amax())
    total, values = weights.sum(), values.double()
    step, least = R.HALF_STEP[dtype], 2.0 ** -25 if dtype == F16 else 2.0 ** -134
    expected = (weights @ values) / total
    error = (step + 2.0 ** -16 + 2.0 ** -18 + 2 * len(decides) / 16 * 2.0 ** -23) * (weights @ values.abs()) / total + least * 2.0 ** -6 * values.abs().sum(0) / total
    error = error + step * (expected.abs() + error) + least
    R.within(out, expected.expand(out.shape), error, "values")
    # What is tested for can be seen: small weights off by a thirtieth, all the same way, lie outside.
    assert (expected / 30 > error).any()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("gap", [14.6, 18.3, 22.4, 25.7])
@pytest.mark.parametrize("keys,heads,requests", [(700, 64, 1), (8192, 64, 1), (8192, 5, 40), (70001, 16, 1)])
def test_absorbed(dtype, gap, keys, heads, requests):
    decides, values = peaked(dtype, keys, 512, gap, keys)
    pages = -(-keys // 64)
    cache = torch.zeros((pages, 64, 1, 576), dtype=dtype, device="cuda")
    cache.view(-1, 576)[:keys, :512], cache.view(-1, 576)[:keys, 570] = values, decides
    q = torch.zeros((requests, heads, 576), dtype=dtype, device="cuda")
    q[..., 570] = 1
    table = torch.arange(pages, dtype=torch.int32, device="cuda").expand(requests, -1).contiguous()
    out = latent.latent_attention(q, cache, table, i32(list(range(requests + 1))), i32([keys] * requests), scale=SCALE)
    check(out, dtype, decides, values, torch.ones((), device="cuda"))
    assert ops.status()[0] == 0


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("gap", [14.6, 18.3, 22.4, 25.7])
@pytest.mark.parametrize("keys,heads,queries", [(700, 2, 1), (8192, 2, 3), (8192, 80, 1), (40000, 3, 130)])
def test_expanded(dtype, gap, keys, heads, queries):
    """Whole items and such that are cut."""
    decides, values = peaked(dtype, keys, 128, gap, keys)
    kv = torch.zeros((keys, heads, 256), dtype=dtype, device="cuda")
    kv[..., 128:], kv[..., 77] = values[:, None], decides[:, None]
    q = torch.zeros((queries, heads, 192), dtype=dtype, device="cuda")
    q[..., 77] = 1
    rope = torch.zeros((keys, 64), dtype=dtype, device="cuda")
    out = latent.latent_prefill(q, kv[..., :128], kv[..., 128:], rope, i32([0, queries]), i32([0, keys]), scale=SCALE, causal=False)
    check(out, dtype, decides, values, torch.ones((), device="cuda"))
    assert ops.status()[0] == 0
