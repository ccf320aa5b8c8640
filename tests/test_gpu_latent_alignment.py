"""Tensors that begin 16 bytes behind a 32-byte boundary, which is all the alignment that the calls around dense latent attention ask for."""

import pytest
import torch

from ascendflow_b200 import latent, ops

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def shifted(tensor):
    """The same values, contiguous and 16 bytes behind a 32-byte boundary; 24 entries of 7 around them."""
    entries = 16 // tensor.element_size()
    buffer = torch.full((tensor.numel() + 4 * entries,), 7.0, dtype=tensor.dtype, device="cuda")
    out = buffer[entries : entries + tensor.numel()].view(tensor.shape)
    out.copy_(tensor)
    assert out.is_contiguous() and (out.data_ptr() % 32 == 16 or out.numel() == 0)
    return out, buffer


def normal(seed, *shape, dtype=BF16):
    return torch.randn(shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(dtype)


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def same(call, shape, dtype):
    """A call writes the same bits into a shifted output as into one of its own, and nothing beside it."""
    out, buffer = shifted(torch.zeros(shape, dtype=dtype, device="cuda"))
    assert torch.equal(call(out=out), call(out=None)) and ops.status()[0] == 0
    entries = 16 // out.element_size()
    assert (buffer[:entries] == 7).all() and (buffer[entries + out.numel() :] == 7).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("counts,lengths,heads", [([1], [1], 1), ([130, 3], [200, 3], 3), ([257], [257], 150), ([3], [5000], 5), ([300], [3000], 2), ([2], [0], 4)])
def test_expanded(dtype, counts, lengths, heads):
    """Items that are whole, that are cut, and of rows that see nothing."""
    tokens, keys = sum(counts), sum(lengths)
    q, k, v, rope = (shifted(normal(i, *shape, dtype=dtype))[0] for i, shape in enumerate([(tokens, heads, 192), (keys, heads, 128), (keys, heads, 128), (keys, 64)]))
    cu = [i32([sum(n[:b]) for b in range(len(n) + 1)]) for n in (counts, lengths)]
    same(lambda out: latent.latent_prefill(q, k, v, rope, *cu, scale=0.07, out=out), (tokens, heads, 128), dtype)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("lengths,heads", [([1, 0], 5), ([300, 200], 64), ([9000, 4000], 16)])
def test_absorbed(dtype, lengths, heads):
    """Tiles that are whole and that are shared."""
    pages = [-(-max(length, 1) // 64) for length in lengths]
    cache, q = shifted(normal(1, sum(pages), 64, 1, 576, dtype=dtype))[0], shifted(normal(2, 2, heads, 576, dtype=dtype))[0]
    table = torch.zeros((2, max(pages)), dtype=torch.int32, device="cuda")
    table[0, : pages[0]] = torch.arange(pages[0])
    table[1, : pages[1]] = pages[0] + torch.arange(pages[1])
    same(lambda out: latent.latent_attention(q, cache, table, i32([0, 1, 2]), i32(lengths), scale=0.07, out=out), (2, heads, 512), dtype)


@pytest.mark.parametrize("dtype", [BF16, F16, torch.float32])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_rotary(dtype, layout):
    x, inv_freq = shifted(normal(1, 5, 3, 192, dtype=dtype))[0], latent.rotary_frequencies(64)
    same(lambda out: latent.rotary(x, i32([1, 2, 3, 4, 5]), inv_freq, layout=layout, out=out), x.shape, dtype)


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_append(layout):
    rows, rope, inv_freq = shifted(normal(1, 3, 512))[0], normal(2, 3 * 64 + 1)[1:].view(3, 64), latent.rotary_frequencies(64)  # (rope: any address)
    cache = normal(3, 2, 64, 1, 576)
    own, buffer = shifted(cache)
    for target in (own, cache):
        latent.rotary_append(rows, rope, target, i32([[1, 0]]), i32([0, 3]), i32([70]), inv_freq, layout=layout)
    assert torch.equal(own, cache) and (buffer[:8] == 7).all() and (buffer[8 + own.numel() :] == 7).all()
