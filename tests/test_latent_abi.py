"""The C functions of the operators around dense latent attention refuse addresses and strides that their kernels cannot take, before anything is enqueued."""

import ctypes

import pytest

from ascendflow_b200.build import library_path


def structure(halves, pointers, words):
    fields = [(name, ctypes.c_int32) for name in halves] + [(name, ctypes.c_void_p) for name in pointers] + [(name, ctypes.c_int64) for name in words]
    return type("Call", (ctypes.Structure,), {"_fields_": [*fields, ("scale", ctypes.c_double)]})


Append = structure(["type", "layout"], ["latent", "rope", "cache", "block_table", "cu_seqlens_q", "seqused_kv", "inv_freq", "status"],
                   ["latent_token", "rope_token", "batches", "tokens", "pages", "blocks", "page_rows", "width", "pairs"])
Attention = structure(["type", "reserved"], ["q", "cache", "block_table", "cu_seqlens_q", "seqused_kv", "sinks", "out", "lse", "workspace", "status"],
                      ["batches", "tokens", "heads", "width", "pages", "blocks", "page_rows"])
Prefill = structure(["type", "causal"], ["q", "k", "v", "k_rope", "cu_seqlens_q", "cu_seqlens_k", "out", "lse", "workspace", "status"],
                    ["q_token", "q_head", "k_token", "k_head", "v_token", "v_head", "rope_token", "batches", "tokens", "keys", "heads"])
# (a batch of no requests: a call that is accepted enqueues nothing either)
CALLS = {
    "launch_latent_append": Append(type=1, latent=64, rope=66, cache=64, status=64, latent_token=512, rope_token=64, tokens=2, pages=1, blocks=1, page_rows=64, width=576, pairs=32, scale=1.0),
    "launch_latent_attention": Attention(type=1, q=64, cache=64, out=64, status=64, tokens=2, heads=4, width=576, pages=1, blocks=1, page_rows=64, scale=1.0),
    "launch_latent_prefill": Prefill(type=1, q=64, k=64, v=64, k_rope=64, out=64, status=64, q_token=384, q_head=192, k_token=256, k_head=128, v_token=256, v_head=128, rope_token=64,
                                     tokens=2, keys=2, heads=2, scale=1.0),
}


@pytest.mark.parametrize("name,pointers,strides", [
    ("launch_latent_append", ["latent", "cache"], ["latent_token"]),
    ("launch_latent_attention", ["q", "cache", "out"], []),
    ("launch_latent_prefill", ["q", "k", "v", "k_rope", "out"], ["q_token", "q_head", "k_token", "k_head", "v_token", "v_head", "rope_token"]),
])
def test_addresses_and_strides(name, pointers, strides):
    launch, call = getattr(ctypes.CDLL(str(library_path())), name), CALLS[name]
    assert launch(None, ctypes.byref(call)) == 0
    for field, wrong in [(field, 64 + off) for field in pointers for off in (2, 8)] + [(field, off) for field in strides for off in (1, 4, 204)]:
        right = getattr(call, field)
        setattr(call, field, wrong)
        assert launch(None, ctypes.byref(call)) == -1, field
        setattr(call, field, right)
    assert launch(None, ctypes.byref(call)) == 0


Rotary = structure(["type", "layout", "inverse", "positions64"], ["x", "out", "positions", "inv_freq"], ["x_token", "x_head", "out_token", "out_head", "tokens", "heads", "features", "pairs"])


def test_amplitudes():
    """Finite in FP32 (the field behind the whole numbers)."""
    library, append = ctypes.CDLL(str(library_path())), CALLS["launch_latent_append"]
    rotary = Rotary(type=1, x=64, out=64, x_token=64, x_head=64, out_token=64, out_head=64, tokens=0, heads=1, features=64, pairs=32)
    for amplitude, expected in ((1.0, 0), (-3.4e38, 0), (0.0, 0), (3.5e38, -1), (-1e39, -1), (float("inf"), -1), (float("nan"), -1)):
        rotary.scale = append.scale = amplitude
        assert library.launch_latent_rotary(None, ctypes.byref(rotary)) == expected, amplitude
        assert library.launch_latent_append(None, ctypes.byref(append)) == expected, amplitude
    append.scale = 1.0


@pytest.mark.parametrize("name", ["launch_latent_attention", "launch_latent_prefill"])
def test_scales(name):
    launch, call = getattr(ctypes.CDLL(str(library_path())), name), CALLS[name]
    for scale, expected in ((1.0, 0), (1e-30, 0), (1e30, 0), (0.0, -1), (-1.0, -1), (1e-40, -1), (1e39, -1), (float("inf"), -1), (float("nan"), -1)):
        call.scale = scale
        assert launch(None, ctypes.byref(call)) == expected, scale
    call.scale = 1.0
