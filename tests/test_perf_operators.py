"""The operators of perf/operators.py through the library run on torch's current stream, each
stream with a handle of its own: the choice on the CPU, and passes on two streams and in a graph."""
import importlib.util
import os

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture()
def ops():
    spec = importlib.util.spec_from_file_location("operators_under_test", os.path.join(ROOT, "perf", "operators.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    module.own = True
    return module


def test_a_handle_for_every_stream(ops, monkeypatch):
    from rtatblas_amd import native

    class Handle:
        def __init__(self, stream):
            self.stream = stream

    now = []
    monkeypatch.setattr(ops.torch.cuda, "current_device", lambda: now[-1][0])
    monkeypatch.setattr(ops.torch._C, "_cuda_getCurrentRawStream", lambda device: now[-1][1] if device == now[-1][0] else None)
    monkeypatch.setattr(native, "Handle", Handle)
    seen = {}
    for on in [(0, 0), (0, 64), (0, 0), (1, 0), (0, 64), (1, 64)]:
        now.append(on)
        h = ops._handle()[1]
        assert h.stream == on[1]
        assert seen.setdefault(on, h) is h
    assert len({id(h) for h in seen.values()}) == 4


CASES = [
    {"op": "fwd", "tokens": 70, "inp": 264, "out": 200, "dtype": "bf16", "act": "gelu", "wt": "nk", "residual": True, "aux": True, "pad": 0},
    {"op": "bwd", "tokens": 300, "inp": 130, "out": 257, "dtype": "f16", "act": "silu", "wt": "nk", "grads": "f16", "pad": 1},
    {"op": "dact", "tokens": 64, "inp": 128, "out": 512, "dtype": "bf16", "act": "relu", "pad": 0},
    {"op": "orth", "rows": 200, "cols": 150, "batch": 2, "dtype": "f32", "steps": 3, "pad": 0}]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=lambda c: c["op"])
def test_passes_follow_the_current_stream(ops, case):
    """The same bits on the default stream, on another whose inputs are still being written when the
    pass is called, and from a graph captured there and replayed on new inputs."""
    import torch

    def same(a, b):
        assert a.keys() == b.keys()
        for k in a:
            assert (a[k] is None) == (b[k] is None) and (a[k] is None or torch.equal(a[k], b[k])), k

    first, second = ops.prepare(case, 1), ops.prepare(case, 2)
    want = [{k: v if v is None else v.clone() for k, v in ops.run(s).items()} for s in (first, second)]
    torch.cuda.synchronize()

    def fill(state, source):
        for k, v in state.items():
            if isinstance(v, torch.Tensor):
                v.copy_(source[k])

    side, state = torch.cuda.Stream(), ops.prepare(case, 3)
    busy = torch.zeros(1 << 26, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for source, w in ((first, want[0]), (second, want[1])):
            for _ in range(4):
                busy.add_(1.0)
            fill(state, source)
            got = ops.run(state)
            side.synchronize()
            same(got, w)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = ops.run(state)
    for source, w in ((first, want[0]), (second, want[1]), (first, want[0])):
        fill(state, source)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        same(got, w)
        ops.run(state)
        torch.cuda.synchronize()
        same(got, w)
    for h in ops._handles.values():
        h.close()
