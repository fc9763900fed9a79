"""Clipping by the global gradient norm under ZeRO-1, on CPU with gloo ranks:
the trainer's host logic (wait for every bucket's shard, sum the ranks' sums
of squares, one factor for all) with plain stand-ins for the two kernels."""
import importlib
import math
import os
import sys
import traceback
import types

import pytest
import torch
import torch.distributed as dist

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "tests"))
from test_dp_gloo import _dp_module, _init, _run  # noqa: E402


def _worker(rank, world, port, q):
    try:
        _init(rank, world, port, 30)
        dp = _dp_module()
        mlp = importlib.import_module("nvfp4_b200.mlp")
        sizes = {0: 1001, 1: 37, 2: 4096}
        opt = dp.ShardedBucketOptimizer(dist.group.WORLD, sizes, "cpu")
        with pytest.raises(RuntimeError):
            opt.wait_grads(0)                              # nothing in flight
        gen = torch.Generator().manual_seed(100 + rank)
        grads = {k: torch.zeros(opt.padded_len(k), dtype=torch.bfloat16) for k in sizes}
        for k, n in sizes.items():
            grads[k][:n] = (torch.randn(n, generator=gen) * 0.1).to(torch.bfloat16)
        whole = {}
        for k in sizes:                                    # the sum a single process would see
            parts = [torch.empty_like(grads[k]) for _ in range(world)]
            dist.all_gather(parts, grads[k])
            whole[k] = sum(p.float() for p in parts).to(torch.bfloat16)
            opt.reduce_scatter(k, grads[k].clone())
        mlp.ops.grad_norm_total = lambda ts: torch.stack([t.double().square().sum() for t in ts]).sum().reshape(1)

        def finish(total, max_norm, grad_scale):
            norm = total.sqrt() * abs(grad_scale)
            return norm.float(), (max_norm / (norm + 1e-6)).clamp(max=1).float()

        mlp.ops.grad_norm_finish = finish
        trainer = types.SimpleNamespace(world=world, opt=opt, reducer=None, pg=dist.group.WORLD, n_blocks=3, blocks=None,
                                        grad_norm=None)
        coef = mlp.NVFP4MLPStackTrainer._clip_coef(trainer, 0.5, 1)
        ref = math.sqrt(sum(float(w.double().square().sum()) for w in whole.values())) / world
        # each rank's sum was rounded to bf16 by the exchange: half a step, 2^-8 of every value
        assert abs(trainer.grad_norm.item() - ref) <= ref * 2.0 ** -8
        assert abs(coef.item() - min(1.0, 0.5 / ref)) <= 2.0 ** -7
        opt.wait_grads(0)                                  # again: nothing to wait for
        seen = {}
        for k in sizes:                                    # the update still runs once per bucket
            opt.update(k, torch.zeros(opt.padded_len(k), dtype=torch.bfloat16),
                       lambda p, g, m, v, k=k: seen.__setitem__(k, g.clone()), gather=False)
            with pytest.raises(RuntimeError):
                opt.update(k, torch.zeros(opt.padded_len(k), dtype=torch.bfloat16), lambda *a: None)
        assert set(seen) == set(sizes)
        dist.barrier()
        dist.destroy_process_group()
        q.put((rank, "ok"))
    except Exception:
        q.put((rank, traceback.format_exc()))


@pytest.mark.parametrize("world", [2, 4])
def test_zero_clipping(world):
    out = _run(_worker, world)
    assert out == {r: "ok" for r in range(world)}, out
