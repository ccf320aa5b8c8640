"""Operators around dense latent attention where there is no device: their refusals, and the frequencies."""

import ctypes
import math

import pytest
import torch

from ascendflow_b200 import latent
from ascendflow_b200.build import library_path
from ascendflow_b200.diagnostics import CompileError


def i32(*shape, device="cpu"):
    return torch.zeros(shape, dtype=torch.int32, device=device)


def bf16(*shape, device="cpu"):
    return torch.zeros(shape, dtype=torch.bfloat16, device=device)


@pytest.mark.parametrize("device", ["cpu", "meta"])
def test_tensors_elsewhere_are_refused(device):
    i = lambda *shape: i32(*shape, device=device)  # noqa: E731
    b = lambda *shape: bf16(*shape, device=device)  # noqa: E731
    frequencies = torch.ones(32, dtype=torch.float64, device=device)
    calls = [
        lambda: latent.rotary(b(2, 4, 64), i(2), frequencies),
        lambda: latent.rotary_append(b(2, 512), b(2, 64), b(4, 64, 1, 576), i(1, 4), i(2), i(1), frequencies),
        lambda: latent.latent_attention(b(2, 4, 576), b(4, 64, 1, 576), i(1, 4), i(2), i(1), scale=0.1),
        lambda: latent.latent_prefill(b(2, 4, 192), b(3, 4, 128), b(3, 4, 128), b(3, 64), i(2), i(2), scale=0.1),
    ]
    for call in calls:
        with pytest.raises(CompileError, match="CUDA tensor"):
            call()


def test_what_is_no_tensor_or_no_choice_is_refused():
    frequencies = torch.ones(32, dtype=torch.float64)
    with pytest.raises(CompileError, match="layout"):
        latent.rotary(bf16(2, 4, 64), i32(2), frequencies, layout="thirds")
    with pytest.raises(CompileError, match="layout"):
        latent.rotary_append(bf16(2, 512), bf16(2, 64), bf16(4, 64, 1, 576), i32(1, 4), i32(2), i32(1), frequencies, layout=None)
    with pytest.raises(CompileError, match="Torch tensor"):
        latent.rotary([1.0], i32(2), frequencies)
    with pytest.raises(CompileError, match="Torch tensor"):
        latent.latent_attention(None, None, None, None, None, scale=1.0)
    with pytest.raises(CompileError, match="scale"):
        latent.latent_attention(bf16(2, 4, 576), None, None, None, None, scale=math.inf)
    with pytest.raises(CompileError, match="scale"):
        latent.latent_prefill(bf16(2, 4, 192), None, None, None, None, None, scale=0)
    with pytest.raises(CompileError, match="amplitude"):
        latent.rotary(bf16(2, 4, 64), i32(2), frequencies, amplitude=math.nan)


def test_frequencies():
    plain = latent.rotary_frequencies(64, device="cpu")
    assert plain.dtype == torch.float64 and plain.shape == (32,)
    assert plain[0] == 1 and abs(plain[16].item() - 0.01) < 1e-15  # 10000 ** -(1/2)
    assert torch.equal(latent.rotary_frequencies(64, scaling="linear", factor=4.0, device="cpu"), plain / 4)
    grown = latent.rotary_frequencies(64, scaling="ntk", factor=8.0, device="cpu")
    assert grown[0] == 1 and abs(grown[-1] / (plain[-1] / 8) - 1) < 1e-12
    # 4096 positions: pair i turns 4096 * 10000 ** (-i / 32) / (2 pi) times: 32 times at i = 10.47, once at i = 22.5
    ramped = latent.rotary_frequencies(64, scaling="yarn", factor=8.0, device="cpu")
    assert torch.equal(ramped[:11], plain[:11]) and torch.allclose(ramped[23:], plain[23:] / 8, rtol=1e-15)
    assert ((ramped[11:23] < plain[11:23]) & (ramped[11:23] > plain[11:23] / 8)).all()
    assert latent.rotary_amplitude(1.0) == 1.0 and abs(latent.rotary_amplitude(math.e) - 1.1) < 1e-12
    for wrong in (dict(dims=63), dict(dims=64, base=1.0), dict(dims=64, factor=0.5), dict(dims=64, scaling="other"),
                  dict(dims=64, scaling="yarn", beta_slow=0.0)):
        with pytest.raises(CompileError):
            latent.rotary_frequencies(**wrong, device="cpu")


class PrefillCall(ctypes.Structure):
    _fields_ = [("type", ctypes.c_int32), ("causal", ctypes.c_int32), *((name, ctypes.c_void_p) for name in (
        "q", "k", "v", "k_rope", "cu_seqlens_q", "cu_seqlens_k", "out", "lse", "workspace", "status")), *((name, ctypes.c_int64) for name in (
            "q_token", "q_head", "k_token", "k_head", "v_token", "v_head", "rope_token", "batches", "tokens", "keys", "heads")), ("scale", ctypes.c_double)]


def test_workspace_of_the_expanded_call():
    """Calls of few items and many keys want one, others do not; a call without the one that it wants is refused before anything is launched."""
    library = ctypes.CDLL(str(library_path()))
    size = ctypes.c_uint64()

    def wanted(batches, tokens, keys, heads):
        call = PrefillCall(batches=batches, tokens=tokens, keys=keys, heads=heads)
        assert library.workspace_size_latent_prefill(ctypes.byref(size), ctypes.byref(call)) == 0
        return size.value

    slot = 256 * 128 * 4 + 256 * 8
    for few in ((1, 1, 1537, 1), (1, 512, 16384, 16), (3, 3, 9000, 16), (1, 256, 5000, 66), (2, 257, 5000, 22)):
        assert wanted(*few) > 0 and wanted(*few) % slot == 0
    for other in ((1, 1, 1408, 1), (1, 0, 16384, 1), (0, 0, 16384, 1), (1, 2048, 16384, 16), (1, 1, 5000, 1000), (400, 400, 10 ** 6, 1), (1, 8192, 8192, 64)):
        assert wanted(*other) == 0
    assert library.workspace_size_latent_prefill(None, ctypes.byref(PrefillCall())) == -1 and library.workspace_size_latent_prefill(ctypes.byref(size), None) == -1
    for wrong in (dict(heads=-1), dict(heads=65536), dict(tokens=-1), dict(keys=-1), dict(batches=-1)):
        assert library.workspace_size_latent_prefill(ctypes.byref(size), ctypes.byref(PrefillCall(**wrong))) == -1
    call = PrefillCall(type=1, batches=1, tokens=2, keys=5000, heads=2, scale=1.0, status=64)
    for workspace in (None, 16):
        call.workspace = workspace
        assert library.launch_latent_prefill(None, ctypes.byref(call)) == -1
