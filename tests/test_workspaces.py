"""The amax workspaces: one per stream, and one of its own for every captured
call.  On CPU with a fake of torch.cuda; on the GPU with two graphs at once."""
import importlib
import os
import sys
import types

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
import __graft_entry__ as graft  # noqa: E402

graft.import_package()
ops = importlib.import_module("nvfp4_b200.ops")


def test_captured_calls_share_none(monkeypatch):
    state = types.SimpleNamespace(stream=11, capturing=False)
    monkeypatch.setattr(ops, "_WS", {})
    monkeypatch.setattr(torch.cuda, "current_stream", lambda d: types.SimpleNamespace(cuda_stream=state.stream))
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: state.capturing)
    dev = torch.device("cpu")
    state.capturing = True
    captured = [ops.workspace(dev) for _ in range(3)]          # the stream's first calls are captured ones
    state.capturing = False
    eager = ops.workspace(dev)
    assert eager is ops.workspace(dev)                         # a stream keeps its own
    state.capturing = True
    captured += [ops.workspace(dev) for _ in range(3)]
    state.capturing, state.stream = False, 12
    other = ops.workspace(dev)
    everyone = captured + [eager, other]
    assert len({t.data_ptr() for t in everyone}) == len(everyone)
    assert all((t == 0).all() and t.numel() == 2 for t in everyone)


@pytest.mark.gpu
def test_two_graphs_at_once(pkg):
    """Global scales of different tensors, captured one after the other, replayed at once."""
    xs = [(torch.randn(4096, 4096, device="cuda") * s).to(torch.bfloat16) for s in (1, 100)]
    ref = [pkg.ops.global_scale(x) for x in xs]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append([pkg.ops.global_scale(x) for _ in range(8)])
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for rep in range(20):
        for o in outs:
            for v in o:
                v.zero_()
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for o, r in zip(outs, ref):
            assert all(torch.equal(v, r) for v in o), rep
    assert all(torch.equal(pkg.ops.global_scale(x), r) for x, r in zip(xs, ref))
