"""IEEE half held to what its smallest numbers cost. A row's unit is at most 2^-6 of its greatest weight (what a first reference leaves, later ones more), so
a weight is off by at most 2^-25 units, 2^-31 of the greatest, besides its half step; the denominator is no less than the greatest weight. `latent_reference.attention` allows
2^-25 of the greatest value for every key instead, which for long contexts is more than bfloat16 is allowed."""

import pytest
import torch

from tests import latent_reference as R
from tests.test_gpu_latent import check_attention, check_prefill, normal, paged

pytestmark = pytest.mark.gpu
F16 = torch.float16


@pytest.fixture(autouse=True)
def narrow(monkeypatch):
    wide = R.attention

    def attention(q, k, v, seen, scale, sinks=None):
        out, lse, error, lse_error = wide(q, k, v, seen, scale, sinks)
        if k.shape[1]:
            error = error - 2.0 ** -25 * v.double().abs().amax() * k.shape[1] + 2.0 ** -31 * v.double().abs().sum(1).amax()
        return out, lse, error, lse_error

    monkeypatch.setattr(R, "attention", attention)


@pytest.mark.parametrize("spread", [0.05, 1.0, 8.0])
@pytest.mark.parametrize("heads,counts,lengths", [(64, [1], [70001]), (16, [3], [40000]), (5, [1] * 9, [9000 - 700 * b for b in range(9)]), (64, [6, 1, 0, 40], [500, 3000, 7, 2000])])
def test_absorbed(spread, heads, counts, lengths):
    cache, table = paged(1, lengths, 576, 64, F16)
    check_attention(normal(2, sum(counts), heads, 576, dtype=F16, spread=spread), cache, table, counts, lengths, 192 ** -0.5)


@pytest.mark.parametrize("spread", [0.05, 1.0, 8.0])
@pytest.mark.parametrize("heads,counts,lengths", [(1, [1], [20000]), (16, [3], [5000]), (4, [1000], [3333]), (2, [257, 0, 1, 130], [2000, 5000, 1, 7001]), (75, [2], [1664])])
def test_expanded(spread, heads, counts, lengths):
    q, kv, rope = (normal(i, *shape, dtype=F16) for i, shape in enumerate([(sum(counts), heads, 192), (sum(lengths), heads, 256), (sum(lengths), 64)]))
    check_prefill(q * spread, kv, rope, counts, lengths, 192 ** -0.5)
