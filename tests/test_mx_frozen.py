"""A frozen MXFP4Linear never drops a gradient in silence: on CPU, with plain
stand-ins for the quantizer and the product."""
import importlib
import os
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
import __graft_entry__ as graft  # noqa: E402

graft.import_package()
f4 = importlib.import_module("nvfp4_b200.float4utils")


@pytest.fixture
def layer(monkeypatch):
    monkeypatch.setattr(f4.ops, "mx_quantize", lambda w: (w.clone(), None))
    monkeypatch.setattr(f4.ops, "mx_linear", lambda x, qw, sw, bias=None: torch.nn.functional.linear(x, qw, bias))
    return f4.MXFP4Linear(64, 32, device="cpu")


def test_frozen_layer_in_grad_mode(layer):
    x = torch.randn(3, 64).to(torch.bfloat16)
    layer.freeze()
    with torch.no_grad():
        ref = layer(x)
    for wanted in ((layer.weight, layer.bias), (layer.weight,), (layer.bias,)):   # a plain input, trainable parameters
        layer.requires_grad_(False)
        for p in wanted:
            p.requires_grad_(True)
        with pytest.raises(RuntimeError, match="no gradients"):
            layer(x)
        with torch.no_grad():
            assert torch.equal(layer(x), ref)
        with torch.inference_mode():
            assert torch.equal(layer(x), ref)
    layer.requires_grad_(False)
    assert torch.equal(layer(x), ref)                  # nothing to give: served in grad mode too
    with pytest.raises(RuntimeError, match="no gradients"):
        layer(x.clone().requires_grad_())


def test_without_a_bias(monkeypatch, layer):
    layer = f4.MXFP4Linear(64, 32, bias=False, device="cpu").freeze()
    x = torch.randn(3, 64).to(torch.bfloat16)
    with pytest.raises(RuntimeError, match="no gradients"):
        layer(x)
    assert layer.requires_grad_(False)(x).shape == (3, 32)
