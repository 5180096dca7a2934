"""Row operators with a workspace: calls, streams and captured graphs whose work overlaps keep theirs apart."""
import pytest
import torch

pytestmark = pytest.mark.gpu

WORKERS = 3


def _inputs(k):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(k)
    rand = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    ids = (rand(20000) ** 4 * 3).long().clamp_(max=499)  # with runs of many groups
    return {"g": rand(20000, 72), "ids": ids, "x": rand(3000, 700).bfloat16(), "dy": rand(3000, 700).bfloat16(), "long": rand(20, 30001),
            "dlong": rand(20, 30001)}


def _calls(pkg, s):
    _, m, r = pkg.layernorm(s["x"], stats=True)
    y, ml, rl = pkg.layernorm(s["long"], stats=True)
    return [pkg.embedding_backward(s["g"], s["ids"], 500), *pkg.layernorm_backward(s["dy"], s["x"], m, r), y, ml, rl,
            *pkg.layernorm_backward(s["dlong"], s["long"], ml, rl)]


def _sizes(pkg, s):
    rows, code = pkg.rows, pkg.rows._TYPES
    return [rows._embedding_workspace_size(code[torch.float32], 72, 20000, code[torch.float32], 500),
            rows._workspace_size("b200ppLayerNormBackwardWorkspace", code[torch.bfloat16], 700, 3000),
            rows._workspace_size("b200ppLayerNormWorkspace", code[torch.float32], 30001, 20),
            rows._workspace_size("b200ppLayerNormBackwardWorkspace", code[torch.float32], 30001, 20)]


def test_captured_graphs_keep_their_workspaces_apart(pkg):
    inputs = [_inputs(k) for k in range(WORKERS)]
    assert all(n > 0 for n in _sizes(pkg, inputs[0]))
    want = [_calls(pkg, s) for s in inputs]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in inputs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(_calls(pkg, s))
    streams = [torch.cuda.Stream() for _ in inputs]
    for _ in range(20):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for got, w in zip(outs, want) for a, b in zip(got, w))


def test_streams_keep_their_workspaces_apart(pkg):
    inputs = [_inputs(k) for k in range(WORKERS)]
    want = [_calls(pkg, s) for s in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in inputs]
    got = [[] for _ in inputs]
    for _ in range(5):
        for k, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[k].append(_calls(pkg, inputs[k]))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for calls, w in zip(got, want) for call in calls for a, b in zip(call, w))
