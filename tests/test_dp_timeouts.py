"""A reduce-scatter that does not complete in time, on CPU with a fake of the
failing call: the wait raises, and the bucket is free for the next step's."""
import importlib
import os
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
import __graft_entry__ as graft  # noqa: E402

graft.import_package()
dp = importlib.import_module("nvfp4_b200.dp")


class Work:
    def __init__(self, fails):
        self.fails = fails

    def wait(self, timeout=None):
        if self.fails:
            raise RuntimeError("timed out")


@pytest.fixture
def opt(monkeypatch):
    monkeypatch.setattr(dp.dist, "get_world_size", lambda pg: 2)
    monkeypatch.setattr(dp.dist, "get_rank", lambda pg: 0)
    fails = []

    def scatter(out, full, op, group, async_op):
        out.copy_(full[:out.numel()])
        return Work(fails.pop(0))

    monkeypatch.setattr(dp.dist, "reduce_scatter_tensor", scatter)
    opt = dp.ShardedBucketOptimizer(None, {"a": 40}, "cpu")
    opt.fails = fails
    return opt


@pytest.mark.parametrize("first", ["update", "wait_grads"])
def test_bucket_is_free_after_a_wait_that_raises(opt, first):
    n = opt.padded_len("a")
    param, seen = torch.zeros(n, dtype=torch.bfloat16), []
    step = lambda **kw: opt.update("a", param, lambda p, g, m, v: seen.append(g.clone()), gather=False, **kw)
    opt.fails[:] = [True, False]
    opt.reduce_scatter("a", torch.ones(n, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="timed out"):
        step(timeout_s=1) if first == "update" else opt.wait_grads("a", timeout_s=1)
    assert not seen
    with pytest.raises(RuntimeError, match="no reduce-scatter in flight"):
        step()                                         # what timed out is gone
    opt.reduce_scatter("a", torch.full((n,), 2.0, dtype=torch.bfloat16))
    opt.wait_grads("a")
    step()
    assert len(seen) == 1 and (seen[0] == 2).all()
