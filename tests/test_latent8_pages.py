"""The operators on a latent cache held in 8 bits and on a cache's pages where there is no device: refusals, the C entries, the registered ops."""

import ctypes

import pytest
import torch

from ascendflow_b200 import host, latent8, pages
from ascendflow_b200.build import library_path
from ascendflow_b200.diagnostics import CompileError

HELD, SCALE = torch.float8_e4m3fn, torch.float8_e8m0fnu


def make(name, device):
    """Arguments of the op, the positions of what it writes, and those of floating inputs."""
    b = lambda *shape: torch.zeros(shape, dtype=torch.bfloat16, device=device)  # noqa: E731
    i = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=device)  # noqa: E731
    u = lambda t, *shape: torch.zeros(shape, dtype=torch.uint8, device=device).view(t)  # noqa: E731
    if name == "latent_append8":
        return [b(2, 512), b(2, 64), u(HELD, 4, 64, 1, 576), u(SCALE, 4, 4), i(1, 4), i(2), i(1), torch.zeros(32, dtype=torch.float64, device=device), True, 1.0], [2, 3], [0, 1]
    if name == "latent_attention8":
        return [b(2, 4, 576), u(HELD, 4, 64, 1, 576), u(SCALE, 4, 4), i(1, 4), i(2), i(1), 0.1, torch.zeros(4, device=device), b(2, 4, 512), torch.zeros((2, 4), device=device)], [8, 9], [0, 7]
    if name == "pages_resize":
        return [i(2, 3), i(5), i(2), 64, i(2, 3), i(5)], [4, 5], []
    if name == "pages_fork":
        return [[b(5, 64, 8), u(SCALE, 5, 4)], i(2, 3), i(5), i(4), i(2), 64, i(4, 3), i(5)], [6, 7], []
    return [[b(5, 64, 8), u(SCALE, 5, 4)], i(2, 3), i(5), i(2, 3), i(5), i(5)], [3, 4, 5], []


CALLS = {
    "latent_append8": lambda a: latent8.rotary_append8(*a[:8], amplitude=a[9])[0],
    "latent_attention8": lambda a: latent8.latent_attention8(*a[:6], scale=a[6], sinks=a[7], lse=a[9]),
    "pages_resize": lambda a: pages.resize(*a[:3], page_rows=a[3])[0],
    "pages_fork": lambda a: pages.fork(*a[:5], page_rows=a[5])[0],
    "pages_compact": lambda a: pages.compact(*a[:3])[2],
}
SHAPES = {"latent_append8": (4, 64, 1, 576), "latent_attention8": (2, 4, 512), "pages_resize": (2, 3), "pages_fork": (4, 3), "pages_compact": (5,)}


def op(name):
    return getattr(torch.ops.ascendflow_b200, name)


def tensors(arguments):
    return [t for a in arguments for t in (a if isinstance(a, list) else [a]) if isinstance(t, torch.Tensor)]


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("device", ["cpu", "meta"])
def test_tensors_elsewhere_are_refused(name, device):
    with pytest.raises(CompileError, match="CUDA tensor"):
        CALLS[name](make(name, device)[0])


def test_what_is_no_tensor_or_no_choice_is_refused():
    append, attention, fork = (make(name, "cpu")[0] for name in ("latent_append8", "latent_attention8", "pages_fork"))
    for call in (lambda: latent8.rotary_append8(*append[:8], layout="both"), lambda: latent8.rotary_append8(*append[:8], amplitude=float("inf")), lambda: latent8.latent_attention8(None, *attention[1:6], scale=1.0),
                 lambda: latent8.latent_attention8(*attention[:6], scale=0.0), lambda: pages.resize(None, *fork[2:4], page_rows=64), lambda: pages.resize(fork[1], fork[2], fork[4], page_rows=0),
                 lambda: pages.resize(fork[1], fork[2], fork[4], page_rows=64, out=fork[1]), lambda: pages.fork(fork[0][0], *fork[1:5], page_rows=64),
                 lambda: pages.fork(*fork[:3], None, fork[4], page_rows=64), lambda: pages.compact(None, *fork[1:3])):
        with pytest.raises(CompileError):
            call()


@pytest.mark.parametrize("name", CALLS)
def test_outputs_count_as_mutated(name):
    arguments, written, _ = make(name, "meta")
    expected = [int(place in written or isinstance(a, list)) for place, a in enumerate(arguments) for t in (a if isinstance(a, list) else [a]) if isinstance(t, torch.Tensor)]
    before = [t._version for t in tensors(arguments)]
    op(name)(*arguments)
    assert [t._version - v for t, v in zip(tensors(arguments), before)] == expected


@pytest.mark.parametrize("name", CALLS)
def test_what_wants_a_gradient_is_refused(name):
    places = make(name, "meta")[2]
    for place in places or [None]:
        arguments = make(name, "meta")[0]
        if place is None:
            if not isinstance(arguments[0], list):
                continue
            arguments[0][0].requires_grad_()
        else:
            arguments[place].requires_grad_()
        with pytest.raises(RuntimeError, match="no gradient"):
            op(name)(*arguments)
        with torch.no_grad():
            op(name)(*arguments)


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_functions_are_traced_as_one_graph(name, backend):
    torch._dynamo.reset()
    graphs = []

    def keep(graph, inputs):
        graphs.append(graph)
        return graph if backend == "eager" else torch._dynamo.lookup_backend(backend)(graph, inputs)

    out = torch.compile(lambda a: CALLS[name](a), backend=keep, fullgraph=True)(make(name, "meta")[0])
    assert out.shape == SHAPES[name] and out.device.type == "meta"
    assert len(graphs) == 1 and [node.target for node in graphs[0].graph.nodes if "ascendflow" in str(node.target)] == [op(name)]


@pytest.mark.parametrize("name", CALLS)
def test_fake_tensors(name):
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        assert CALLS[name](make(name, "cpu")[0]).shape == SHAPES[name]


@pytest.mark.parametrize("name", CALLS)
def test_the_stand_in_registers_the_same_schemas(name):
    schema = next(s for s in (*host.LATENT_SCHEMAS, *host.PAGES_SCHEMAS) if s.startswith(name + "("))
    assert torch._C.parse_schema("ascendflow_b200::" + schema) == op(name).default._schema


# ---- the C entries -------------------------------------------------------------------------------------------------------

def structure(name, halves, pointers, words, last=()):
    fields = [(f, ctypes.c_int32) for f in halves] + [(f, ctypes.c_void_p) for f in pointers] + [(f, ctypes.c_int64) for f in words] + list(last)
    return type(name, (ctypes.Structure,), {"_fields_": fields})


DOUBLE = [("scale", ctypes.c_double)]
Append = structure("Append", ["type", "layout"], ["latent", "rope", "cache", "block_table", "cu_seqlens_q", "seqused_kv", "inv_freq", "status"],
                   ["latent_token", "rope_token", "batches", "tokens", "pages", "blocks", "page_rows", "width", "pairs"], DOUBLE)
Attention = structure("Attention", ["type", "reserved"], ["q", "cache", "block_table", "cu_seqlens_q", "seqused_kv", "sinks", "out", "lse", "workspace", "status"],
                      ["batches", "tokens", "heads", "width", "pages", "blocks", "page_rows"], DOUBLE)
Append8 = type("Append8", (ctypes.Structure,), {"_fields_": [("call", Append), ("scales", ctypes.c_void_p), ("block_rows", ctypes.c_int64)]})
Attention8 = type("Attention8", (ctypes.Structure,), {"_fields_": [("call", Attention), ("scales", ctypes.c_void_p), ("block_rows", ctypes.c_int64)]})
Pages = structure("Pages", [], ["table_in", "table_out", "counts_in", "counts_out", "lengths", "workspace", "status"], ["requests", "entries", "blocks", "page_rows"])
Tensor = structure("Tensor", [], ["memory"], ["page_bytes", "rows"])
Fork = type("Fork", (ctypes.Structure,), {"_fields_": [("call", Pages), ("parents", ctypes.c_void_p), ("tensors", ctypes.POINTER(Tensor)), ("children", ctypes.c_int64), ("tensor_count", ctypes.c_int64)]})
Compact = type("Compact", (ctypes.Structure,), {"_fields_": [("call", Pages), ("places", ctypes.c_void_p), ("tensors", ctypes.POINTER(Tensor)), ("tensor_count", ctypes.c_int64)]})


@pytest.mark.parametrize("name,call,changes", [
    ("launch_latent_append8", Append8(Append(type=1, latent=64, rope=66, cache=64, status=64, latent_token=512, rope_token=64, tokens=2, pages=1, blocks=1, page_rows=64, width=576, pairs=32, scale=1.0), 64, 16),
     {"type": [2, -1], "latent": [66, 72], "cache": [72], "latent_token": [513, 4], "width": [568, 48, 65552], "pairs": [4, 12, 136], "page_rows": [32, 96, 0], "tokens": [-1], "batches": [-1], "pages": [-1, 1 << 31],
      "blocks": [-1, 1 << 31], "scale": [float("nan"), 1e39], "status": [None], "block_rows": [0, 3, 128, -1]}),
    ("launch_latent_attention8", Attention8(Attention(type=1, q=64, cache=64, out=64, status=64, tokens=2, heads=4, width=576, pages=1, blocks=1, page_rows=64, scale=1.0), 64, 16),
     {"type": [2, -1], "q": [66], "cache": [72], "out": [72], "width": [64, 1024], "heads": [0], "page_rows": [32, 96], "tokens": [-1, 1 << 30], "batches": [-1], "pages": [-1], "blocks": [-1], "scale": [0.0, float("nan")],
      "block_rows": [0, 3, 128, -1]}),
])
def test_entries_for_rows_in_8_bits_refuse(name, call, changes):
    """(A batch of no requests: a call that is accepted enqueues nothing either.)"""
    launch = getattr(ctypes.CDLL(str(library_path())), name)
    assert launch(None, ctypes.byref(call)) == 0 and launch(None, None) == -1
    for field, values in changes.items():
        own = call if hasattr(call, field) else call.call
        right = getattr(own, field)
        for wrong in values:
            setattr(own, field, wrong)
            assert launch(None, ctypes.byref(call)) == -1, (field, wrong)
        setattr(own, field, right)
    assert launch(None, ctypes.byref(call)) == 0


def test_entries_for_pages_refuse():
    library, tensor = ctypes.CDLL(str(library_path())), Tensor(64, 64, 4)
    table = Pages(requests=0, entries=3, blocks=5, page_rows=64, counts_in=64, counts_out=64)
    calls = {"resize": table, "fork": Fork(table, 64, ctypes.pointer(tensor), 0, 1), "compact": Compact(Pages(requests=0, entries=3, blocks=0, page_rows=64), 64, ctypes.pointer(tensor), 1)}
    size = ctypes.c_uint64()
    for name, call in calls.items():
        launch, workspace, common = getattr(library, "launch_pages_" + name), getattr(library, "workspace_size_pages_" + name), call if name == "resize" else call.call
        assert launch(None, ctypes.byref(call)) == 0 and launch(None, None) == -1 and workspace(None, ctypes.byref(call)) == -1 and workspace(ctypes.byref(size), None) == -1
        for field, values in {"requests": [-1, 1 << 31, 1 << 30], "entries": [-1, 1 << 31], "blocks": [-1, (1 << 23) + 1], "page_rows": [0, -1, 1 << 31]}.items():
            right = getattr(common, field)
            for wrong in values:
                setattr(common, field, wrong)
                assert launch(None, ctypes.byref(call)) == -1 and workspace(ctypes.byref(size), ctypes.byref(call)) == -1, (name, field, wrong)
            setattr(common, field, right)
        # something to do, and no workspace or status
        common.requests, common.blocks = 2, 5
        assert launch(None, ctypes.byref(call)) == -1
        assert workspace(ctypes.byref(size), ctypes.byref(call)) == 0 and size.value >= 16
        common.workspace = 64
        assert launch(None, ctypes.byref(call)) == -1
        common.workspace, common.status = 72, 64
        assert launch(None, ctypes.byref(call)) == -1
        if name == "resize":
            continue
        common.workspace = 64
        for change in ({"rows": 0}, {"rows": 5}, {"rows": 128}, {"page_bytes": -4}, {"page_bytes": 6}):
            own = Tensor(64, 64, 4)
            for field, value in change.items():
                setattr(own, field, value)
            call.tensors = ctypes.pointer(own)
            assert launch(None, ctypes.byref(call)) == -1, change
        call.tensors = None
        assert launch(None, ctypes.byref(call)) == -1
        call.tensors, call.tensor_count = ctypes.pointer(tensor), 129
        assert launch(None, ctypes.byref(call)) == -1
