"""How the calls around dense latent attention treat what they are given: places in the cache, numbers, versions, tangents, empty and very wide calls, threads."""

import threading

import numpy as np
import pytest
import torch

from ascendflow_b200 import latent, ops
from ascendflow_b200.diagnostics import CompileError
from tests import latent_reference as R

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def normal(seed, *shape, dtype=BF16):
    return torch.randn(shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(dtype)


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("starts,counts", [([0, 5], [3]), ([0, 2, 7], [2, 1]), ([-4, 2, 3], [2, 1]), ([-9, -1, 1 << 30], [0, 3])])
def test_append_puts_rows_where_attention_reads_them(starts, counts):
    """Offsets outside of the tokens are clamped: the last rows of a request are its last tokens, for the append as for the attention call behind it."""
    lengths = [130, 70][: len(counts)]
    rows, rope, inv_freq = normal(1, 3, 512), normal(2, 3, 64), latent.rotary_frequencies(64)
    cache, table = normal(3, 6, 64, 1, 576), i32([[4, 0, 2], [1, 3, 5]][: len(counts)])
    expected = R.append(rows, rope, cache, table, counts, lengths, inv_freq, "interleaved")
    clamped = cache.clone()
    ops.status()
    latent.rotary_append(rows, rope, cache, table, i32(starts), i32(lengths), inv_freq)
    assert ops.status()[0] == 0
    R.within(cache, expected, R.HALF_STEP[BF16] * expected.abs() + 16 * 2.0 ** -24 * 8, "cache")
    latent.rotary_append(rows, rope, clamped, table, i32([min(max(s, 0), 3) for s in starts]), i32(lengths), inv_freq)
    assert torch.equal(cache, clamped)


def test_numbers_are_taken_or_refused_alike_by_all_calls():
    """Real numbers of any kind are taken, whether or not the call stays in native code; tensors and texts are not."""
    q, kv, rope, cu = normal(1, 4, 2, 192), normal(2, 4, 2, 256), normal(3, 4, 64), i32([0, 4])
    cache, table, seq, inv_freq = normal(4, 1, 64, 1, 576), i32([[0]]), i32([20]), latent.rotary_frequencies(64)
    absorbed, rows = normal(5, 4, 2, 576), normal(6, 4, 512)
    calls = {
        "scale": (lambda n: latent.latent_prefill(q, kv[..., :128], kv[..., 128:], rope, cu, cu, scale=n), lambda n: latent.latent_attention(absorbed, cache, table, cu, seq, scale=n)),
        "amplitude": (lambda n: latent.rotary(q, i32([1, 2, 3, 4]), inv_freq, amplitude=n), lambda n: latent.rotary_append(rows, rope, cache, table, cu, seq, inv_freq, amplitude=n)),
    }
    for name, group in calls.items():
        for call in group:
            expected = call(0.5).clone()
            for number in (np.float32(0.5), np.float64(0.5), np.float16(0.5)):
                assert torch.equal(call(number), expected)
            assert torch.equal(call(1), call(np.int64(1)))
            for wrong in (torch.tensor(0.5), torch.tensor(0.5, device="cuda"), np.array(0.5), "0.5", None, 10 ** 400, float("nan"), float("inf"), 1e39):
                with pytest.raises(CompileError, match=name):
                    call(wrong)


@pytest.mark.parametrize("name", ["np.float32(0.5)", "torch.tensor(0.5)"])
def test_the_first_call_of_a_process_takes_what_others_take(name):
    import subprocess
    import sys
    from pathlib import Path

    program = """
import numpy as np, torch
from ascendflow_b200 import latent
q, kv, cu = torch.randn((4, 2, 192), device="cuda").half(), torch.randn((4, 2, 256), device="cuda").half(), torch.tensor([0, 4], dtype=torch.int32, device="cuda")
for _ in range(2):
    try:
        latent.latent_prefill(q, kv[..., :128], kv[..., 128:], q[:, 0, 128:], cu, cu, scale=NUMBER)
        print("taken")
    except Exception as error:
        print(type(error).__name__)
    latent.latent_prefill(q, kv[..., :128], kv[..., 128:], q[:, 0, 128:], cu, cu, scale=0.5)
""".replace("NUMBER", name)
    result = subprocess.run([sys.executable, "-c", program], cwd=Path(__file__).resolve().parents[1], capture_output=True, text=True, timeout=120)
    assert result.stdout.split() == ["taken" if "np" in name else "CompileError"] * 2, result.stderr[-2000:]


def written_by(name, target):
    """A call that writes `target`."""
    if name == "rotary":
        return lambda: latent.rotary(target, i32([1, 2, 3, 4]), latent.rotary_frequencies(64), out=target)
    cache, table, cu, seq = normal(4, 1, 64, 1, 576), i32([[0]]), i32([0, 4]), i32([20])
    if name == "append":
        return lambda: latent.rotary_append(normal(1, 4, 512), normal(2, 4, 64), target, table, cu, seq, latent.rotary_frequencies(64))
    if name.startswith("attention"):
        q = normal(3, 4, 2, 576)
        return lambda: latent.latent_attention(q, cache, table, cu, seq, scale=0.1, **{name.split()[1]: target})
    q, kv = normal(3, 4, 2, 192), normal(5, 4, 2, 256)
    return lambda: latent.latent_prefill(q, kv[..., :128], kv[..., 128:], q[:, 0, 128:], cu, cu, scale=0.1, **{name.split()[1]: target})


TARGETS = [("rotary", (4, 2, 64), BF16), ("append", (1, 64, 1, 576), BF16), ("attention out", (4, 2, 512), BF16), ("attention lse", (4, 2), torch.float32),
           ("prefill out", (4, 2, 128), BF16), ("prefill lse", (4, 2), torch.float32)]


@pytest.mark.parametrize("name,shape,dtype", TARGETS)
def test_writes_count_the_version_up(name, shape, dtype):
    """So that autograd sees that a tensor which it keeps has changed; tensors made in inference mode have no version."""
    target = normal(7, *shape, dtype=dtype)
    call = written_by(name, target)
    call()
    before = target._version
    call()
    assert target._version == before + 1
    leaf = normal(8, *shape, dtype=dtype).requires_grad_()
    product = leaf * target  # keeps target
    with torch.no_grad():
        call()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.sum().backward()
    with torch.inference_mode():
        written_by(name, normal(7, *shape, dtype=dtype))()


@pytest.mark.parametrize("name,shape,dtype", TARGETS)
def test_tensors_with_a_tangent_are_refused(name, shape, dtype):
    import torch.autograd.forward_ad as forward

    with forward.dual_level():
        target = forward.make_dual(normal(7, *shape, dtype=dtype), normal(8, *shape, dtype=dtype))
        with pytest.raises(CompileError, match="gradient"):
            written_by(name, target)()
    written_by(name, normal(7, *shape, dtype=dtype))()


def test_calls_of_nothing_with_odd_strides():
    """What has no entries has no alignment: empty batches out of odd projections, rows that are rope alone."""
    inv_freq = latent.rotary_frequencies(64)
    assert latent.rotary(normal(1, 3, 2, 100)[:0, :, 1:65], i32([]), inv_freq).shape == (0, 2, 64)
    assert latent.rotary(normal(1, 3, 2, 100)[:, :0, 1:65], i32([1, 2, 3]), inv_freq).shape == (3, 0, 64)
    cache, rope = normal(2, 2, 64, 1, 64), normal(3, 3, 64)
    for latents in (normal(4, 3, 0), normal(4, 3, 7)[:, 3:3], normal(4, 3, 64)[:, :0]):
        own = cache.clone()
        latent.rotary_append(latents, rope, own, i32([[1, 0]]), i32([0, 3]), i32([70]), inv_freq)
        expected = R.append(latents, rope, cache, i32([[1, 0]]), [3], [70], inv_freq, "interleaved")
        R.within(own, expected, R.HALF_STEP[BF16] * expected.abs() + 16 * 2.0 ** -24 * 8)
    latent.rotary_append(normal(4, 3, 519)[:0, 1:513], rope[:0], normal(2, 2, 64, 1, 576), i32([[1, 0]]), i32([0, 0]), i32([70]), inv_freq)


def test_rotary_of_the_widest_tokens():
    """As many heads and features as the call takes: 2^29 features of one token."""
    x = torch.zeros((1, 65536, 8192), dtype=BF16, device="cuda")
    x[0, ::4099] = normal(1, 16, 8192)
    out = latent.rotary(x, i32([12345]), latent.rotary_frequencies(64))
    some = latent.rotary(x[:, ::4099].contiguous(), i32([12345]), latent.rotary_frequencies(64))
    assert torch.equal(out[:, ::4099], some)
    out[0, ::4099] = 0
    assert not out.any()


def test_calls_of_several_threads_at_once():
    """Each on a stream of its own; scratch memory and reports are a call's own."""
    lengths = [3000, 50, 700]
    cache, table, cu, seq = normal(1, 70, 64, 1, 576), torch.arange(63 * 3, dtype=torch.int32, device="cuda").view(3, 63) % 70, i32([0, 2, 3, 6]), i32(lengths)
    kv, rope, cu_k = normal(2, 9000, 2, 256), normal(3, 9000, 64), i32([0, 3000, 4000, 9000])
    queries = [normal(10 + i, 6, 64, 576) for i in range(4)]

    def both(q):
        out = latent.latent_attention(q, cache, table, cu, seq, scale=0.07)
        prompt = latent.rotary(q[:, :2, :192], i32([1, 2, 3, 4, 5, 6]), frequencies)
        return out, latent.latent_prefill(prompt, kv[..., :128], kv[..., 128:], rope, cu, cu_k, scale=0.07)

    frequencies = latent.rotary_frequencies(64)
    expected = [both(q) for q in queries]
    torch.cuda.synchronize()
    found, failed = [[] for _ in queries], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(25):
                    found[i].append(both(queries[i]))
                torch.cuda.current_stream().synchronize()
                assert ops.status()[0] == 0
        except BaseException as error:  # noqa: BLE001
            failed.append(error)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(queries))]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    assert not failed, failed
    for own, (out, prompt) in zip(found, expected):
        assert len(own) == 25 and all(torch.equal(a, out) and torch.equal(b, prompt) for a, b in own)
