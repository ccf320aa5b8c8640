"""The registered ops of the operators around dense latent attention where there is no device: tracing, versions, and no gradient."""

import pytest
import torch

from ascendflow_b200 import host, latent

NAMES = ["rotary", "latent_append", "latent_attention", "latent_prefill"]


def make(name, device, written=None):
    """Arguments of the op, the positions of what it writes, and those of floating inputs."""
    b = lambda *shape: torch.zeros(shape, dtype=torch.bfloat16, device=device)  # noqa: E731
    i = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=device)  # noqa: E731
    f = lambda *shape, dtype=torch.float32: torch.zeros(shape, dtype=dtype, device=device)  # noqa: E731
    if name == "rotary":
        return [b(2, 4, 64), i(2), f(32, dtype=torch.float64), False, True, 1.5, b(2, 4, 64)], [6], [0]
    if name == "latent_append":
        return [b(2, 512), b(2, 64), b(4, 64, 1, 576), i(1, 4), i(2), i(1), f(32, dtype=torch.float64), True, 1.0], [2], [0, 1]
    if name == "latent_attention":
        return [b(2, 4, 576), b(4, 64, 1, 576), i(1, 4), i(2), i(1), 0.1, f(4), b(2, 4, 512), f(2, 4)], [7, 8], [0, 1, 6]
    return [b(2, 4, 192), b(3, 4, 128), b(3, 4, 128), b(3, 64), i(2), i(2), 0.1, True, b(2, 4, 128), f(2, 4)], [8, 9], [0, 1, 2, 3]


def op(name):
    return getattr(torch.ops.ascendflow_b200, name)


@pytest.mark.parametrize("name", NAMES)
def test_outputs_count_as_mutated(name):
    arguments, written, _ = make(name, "meta")
    before = [t._version for t in arguments if isinstance(t, torch.Tensor)]
    op(name)(*arguments)
    after = [t._version for t in arguments if isinstance(t, torch.Tensor)]
    expected = [int(place in written) for place, t in enumerate(arguments) if isinstance(t, torch.Tensor)]
    assert [b - a for a, b in zip(before, after)] == expected
    with torch.inference_mode():
        op(name)(*make(name, "meta")[0])
    if name in NAMES[2:]:  # optional tensors
        arguments[-1] = None
        op(name)(*arguments)


@pytest.mark.parametrize("name", NAMES)
def test_what_wants_a_gradient_is_refused(name):
    for place in make(name, "meta")[2]:
        arguments = make(name, "meta")[0]
        arguments[place].requires_grad_()
        with pytest.raises(RuntimeError, match="no gradient"):
            op(name)(*arguments)
        with torch.no_grad():
            op(name)(*arguments)

        def loss(factor):
            call, written, _ = make(name, "meta")
            call[place] = call[place] * factor
            op(name)(*call)
            return call[written[0]].sum()

        with pytest.raises(RuntimeError):
            torch.func.grad(loss)(torch.ones((), dtype=arguments[place].dtype, device="meta"))


CALLS = {
    "rotary": lambda a: latent.rotary(a[0], a[1], a[2], layout="half", inverse=True, amplitude=a[5]),
    "rotary in place": lambda a: latent.rotary(a[0], a[1], a[2], out=a[0]),
    "latent_append": lambda a: latent.rotary_append(*a[:7], amplitude=a[8]),
    "latent_attention": lambda a: latent.latent_attention(*a[:5], scale=a[5], sinks=a[6], lse=a[8]),
    "latent_prefill": lambda a: latent.latent_prefill(*a[:6], scale=a[6], causal=False),
}
SHAPES = {"rotary": (2, 4, 64), "rotary in place": (2, 4, 64), "latent_append": (4, 64, 1, 576), "latent_attention": (2, 4, 512), "latent_prefill": (2, 4, 128)}


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_functions_are_traced_as_one_graph(call, backend):
    torch._dynamo.reset()
    graphs = []

    def keep(graph, inputs):
        graphs.append(graph)
        return graph if backend == "eager" else torch._dynamo.lookup_backend(backend)(graph, inputs)

    def step(arguments):
        return CALLS[call](arguments)

    out = torch.compile(step, backend=keep, fullgraph=True)(make(call.split()[0], "meta")[0])
    assert out.shape == SHAPES[call] and out.dtype == torch.bfloat16 and out.device.type == "meta"
    assert len(graphs) == 1 and [node.target for node in graphs[0].graph.nodes if "ascendflow" in str(node.target)] == [op(call.split()[0])]


@pytest.mark.parametrize("name", NAMES)
def test_what_wants_a_gradient_is_refused_while_a_graph_is_traced(name):
    torch._dynamo.reset()
    arguments, _, floating = make(name, "meta")
    arguments[floating[0]].requires_grad_()
    with pytest.raises(Exception, match="no gradient"):
        torch.compile(lambda a: CALLS[name](a), backend="aot_eager", fullgraph=True)(arguments)


@pytest.mark.parametrize("call", CALLS)
def test_fake_tensors(call):
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        out = CALLS[call](make(call.split()[0], "cpu")[0])
        assert out.shape == SHAPES[call] and out.dtype == torch.bfloat16


@pytest.mark.parametrize("call", CALLS)
def test_dispatch_modes_see_the_call(call):
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils._python_dispatch import TorchDispatchMode

    arguments = make(call.split()[0], "meta")[0]
    graph = make_fx(lambda *tensors: CALLS[call](list(tensors)))(*arguments)
    assert op(call.split()[0]).default in [node.target for node in graph.graph.nodes]
    seen = []

    class Look(TorchDispatchMode):
        def __torch_dispatch__(self, function, types, args=(), kwargs=None):
            seen.append(function)
            return function(*args, **(kwargs or {}))

    with Look():
        CALLS[call](arguments)
    assert op(call.split()[0]).default in seen


@pytest.mark.parametrize("name", NAMES)
def test_the_stand_in_registers_the_same_schemas(name):
    """What the package defines where the native module cannot be had."""
    schema = next(s for s in host.LATENT_SCHEMAS if s.startswith(name + "("))
    assert torch._C.parse_schema("ascendflow_b200::" + schema) == op(name).default._schema


def test_imports_and_traces_where_the_native_module_cannot_be_built(tmp_path):
    import os
    import shutil
    import subprocess
    import sys
    from pathlib import Path

    root = Path(__file__).resolve().parents[1]
    shutil.copytree(root / "ascendflow_b200", tmp_path / "ascendflow_b200", ignore=shutil.ignore_patterns("lib", "__pycache__"))
    shutil.copytree(root / "include", tmp_path / "include")
    program = """
import torch
from ascendflow_b200 import latent
from ascendflow_b200.diagnostics import CompileError
b, i = (lambda *shape, d="meta", t=t: torch.zeros(shape, dtype=t, device=d) for t in (torch.bfloat16, torch.int32))
torch.ops.ascendflow_b200.latent_attention(b(2, 4, 576), b(4, 64, 1, 576), i(1, 4), i(2), i(1), 0.1, None, b(2, 4, 512), None)
try:
    latent.latent_attention(b(2, 4, 576), b(4, 64, 1, 576), i(1, 4), i(2), i(1), scale=0.1)
except CompileError as error:
    assert "CUDA tensor" in str(error)
    print("refused")
from ascendflow_b200 import ops
"""
    result = subprocess.run([sys.executable, "-c", program], cwd=tmp_path, capture_output=True, text=True,
                            env=dict(os.environ, CXX="/bin/false", PYTHONPATH=str(tmp_path)))
    assert result.stdout.strip() == "refused" and result.returncode == 0, result.stderr[-2000:]
