"""The registered ops of the operators around dense latent attention on a GPU: the functions' results, errors and graphs."""

import pytest
import torch

from ascendflow_b200 import latent, ops
from ascendflow_b200.diagnostics import CompileError

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def normal(seed, *shape, dtype=BF16):
    return torch.randn(shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(dtype)


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


@pytest.fixture
def layer():
    """What a layer's step has in hand."""
    return dict(projected=normal(1, 5, 16, 192), rows=normal(2, 5, 512), rope=normal(3, 5, 64), cache=normal(4, 6, 64, 1, 576), table=i32([[4, 0, 2], [1, 3, 5]]), cu=i32([0, 2, 5]),
                lengths=i32([130, 70]), positions=i32([128, 129, 67, 68, 69]), absorbed=normal(5, 5, 16, 576), kv=normal(6, 200, 16, 256), k_rope=normal(7, 200, 64),
                cu_k=i32([0, 130, 200]), inv_freq=latent.rotary_frequencies(64))


def step(s):
    """Turn, append, attend; a prompt in expanded form; queries turned in place."""
    q = s["absorbed"] * 1.0
    latent.rotary(s["projected"][..., 128:], s["positions"], s["inv_freq"], out=q[..., 512:])
    cache = latent.rotary_append(s["rows"], s["rope"], s["cache"], s["table"], s["cu"], s["lengths"], s["inv_freq"])
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)
    out = latent.latent_attention(q, cache, s["table"], s["cu"], s["lengths"], scale=0.07, sinks=s["sinks"], lse=lse)
    prompt = s["projected"] + 0.0
    latent.rotary(prompt, s["positions"], s["inv_freq"], layout="half", out=prompt)
    whole = latent.latent_prefill(prompt, s["kv"][..., :128], s["kv"][..., 128:], s["k_rope"], s["cu"], s["cu_k"], scale=0.07)
    return q, cache, out, lse, prompt, whole


@pytest.mark.parametrize("sinks", [False, True])
@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_a_compiled_step_is_the_eager_one(layer, sinks, backend):
    layer["sinks"] = normal(8, 16, dtype=torch.float32) if sinks else None
    before = layer["cache"].clone()
    expected = [t.clone() for t in step(layer)]
    layer["cache"].copy_(before)
    torch._dynamo.reset()
    found = torch.compile(step, backend=backend, fullgraph=True)(layer)
    assert all(torch.equal(a, b) for a, b in zip(found, expected))
    assert torch.equal(layer["cache"], expected[1]) and not torch.equal(before, expected[1])
    assert ops.status()[0] == 0


def test_dispatch_modes_see_calls_with_tensors_of_memory(layer):
    from torch.fx.experimental.proxy_tensor import make_fx

    layer["sinks"] = None
    before = layer["cache"].clone()
    expected = [t.clone() for t in step(layer)]
    layer["cache"].copy_(before)
    names = list(layer)
    graph = make_fx(lambda *values: step(dict(zip(names, values))))(*layer.values())
    assert sum("ascendflow" in str(node.target) for node in graph.graph.nodes) == 5
    for _ in range(2):  # what was traced does it again
        layer["cache"].copy_(before)
        assert all(torch.equal(a, b) for a, b in zip(graph(*layer.values()), expected))


def test_ops_do_what_the_functions_do(layer):
    s, call = layer, torch.ops.ascendflow_b200
    out, lse = torch.empty((5, 16, 512), dtype=BF16, device="cuda"), torch.empty((5, 16), device="cuda")
    call.latent_attention(s["absorbed"], s["cache"], s["table"], s["cu"], s["lengths"], 0.07, None, out, lse)
    again = torch.empty_like(lse)
    assert torch.equal(out, latent.latent_attention(s["absorbed"], s["cache"], s["table"], s["cu"], s["lengths"], scale=0.07, lse=again)) and torch.equal(lse, again)
    turned = torch.empty_like(s["projected"])
    call.rotary(s["projected"], s["positions"], s["inv_freq"], True, False, 1.25, turned)
    assert torch.equal(turned, latent.rotary(s["projected"], s["positions"], s["inv_freq"], layout="half", amplitude=1.25))
    version = turned._version
    call.rotary(s["projected"], s["positions"], s["inv_freq"], True, False, 1.25, turned)
    assert turned._version == version + 1


def test_registrations_hold_together(layer):
    """Schemas (what is mutated and what is not), fake kernels and autograd, as torch checks them."""
    s, call, f32 = layer, torch.ops.ascendflow_b200, dict(dtype=torch.float32, device="cuda")
    out = torch.zeros((5, 16, 512), dtype=BF16, device="cuda")
    prompt = s["projected"], s["kv"][..., :128], s["kv"][..., 128:], s["k_rope"], s["cu"], s["cu_k"], 0.07, True, torch.zeros((5, 16, 128), dtype=BF16, device="cuda")
    for op, arguments in (
        (call.rotary, (s["projected"], s["positions"], s["inv_freq"], False, True, 1.0, torch.zeros_like(s["projected"]))),
        (call.latent_append, (s["rows"], s["rope"], s["cache"], s["table"], s["cu"], s["lengths"], s["inv_freq"], True, 1.0)),
        (call.latent_attention, (s["absorbed"], s["cache"], s["table"], s["cu"], s["lengths"], 0.07, None, out, None)),
        (call.latent_attention, (s["absorbed"], s["cache"], s["table"], s["cu"], s["lengths"], 0.07, torch.zeros(16, **f32), out, torch.zeros((5, 16), **f32))),
        (call.latent_prefill, (*prompt, None)),
        (call.latent_prefill, (*prompt, torch.zeros((5, 16), **f32))),
    ):
        torch.library.opcheck(op.default, arguments, test_utils=("test_schema", "test_autograd_registration", "test_faketensor"))


def test_refused_calls_raise_the_front_ends_error(layer):
    s, call = layer, torch.ops.ascendflow_b200
    out = torch.empty((5, 16, 512), dtype=BF16, device="cuda")
    for message, wrong in (
        ("scale", lambda: call.latent_attention(s["absorbed"], s["cache"], s["table"], s["cu"], s["lengths"], -1.0, None, out, None)),
        ("lse", lambda: call.latent_attention(s["absorbed"], s["cache"], s["table"], s["cu"], s["lengths"], 0.1, None, out, out)),
        ("amplitude", lambda: call.rotary(s["projected"], s["positions"], s["inv_freq"], False, False, 1e39, s["projected"])),
        ("int32", lambda: call.latent_append(s["rows"], s["rope"], s["cache"], s["table"].long(), s["cu"], s["lengths"], s["inv_freq"], False, 1.0)),
        ("192", lambda: call.latent_prefill(s["absorbed"], s["kv"][..., :128], s["kv"][..., 128:], s["k_rope"], s["cu"], s["cu_k"], 0.1, True, s["absorbed"], None)),
    ):
        with pytest.raises(CompileError, match=message):
            wrong()
    with pytest.raises(RuntimeError, match="no gradient"):
        call.latent_attention(s["absorbed"].requires_grad_(), s["cache"], s["table"], s["cu"], s["lengths"], 0.1, None, out, None)


@pytest.mark.parametrize("entry", ["function", "op"])
def test_the_first_call_of_a_process(entry):
    """As a function or as an op, with a rule violated or not."""
    import subprocess
    import sys
    from pathlib import Path

    program = """
import torch
from ascendflow_b200 import latent
q, kv, cu = torch.randn((4, 2, 192), device="cuda").half(), torch.randn((4, 2, 256), device="cuda").half(), torch.tensor([0, 4], dtype=torch.int32, device="cuda")
for scale in (-1.0, 0.5, -1.0, 0.5):
    out = torch.zeros((4, 2, 128), device="cuda").half()
    try:
        if "ENTRY" == "op":
            torch.ops.ascendflow_b200.latent_prefill(q, kv[..., :128], kv[..., 128:], q[:, 0, 128:], cu, cu, scale, True, out, None)
        else:
            latent.latent_prefill(q, kv[..., :128], kv[..., 128:], q[:, 0, 128:], cu, cu, scale=scale, out=out)
        print("taken" if out.any() else "nothing")
    except Exception as error:
        print(type(error).__name__)
""".replace("ENTRY", entry)
    result = subprocess.run([sys.executable, "-c", program], cwd=Path(__file__).resolve().parents[1], capture_output=True, text=True, timeout=120)
    assert result.stdout.split() == ["CompileError", "taken"] * 2, result.stderr[-2000:]
