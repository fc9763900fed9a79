"""The torch extension module follows the installed PyTorch: built again when it
changed, not loaded when it was made for another one.  The compiler is a fake."""
import importlib
import os
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
import __graft_entry__ as graft  # noqa: E402

pkg = graft.import_package()
build, bind = (importlib.import_module(f"nvfp4_b200.{m}") for m in ("_build", "_bind"))


@pytest.fixture
def compiles(monkeypatch, tmp_path):
    monkeypatch.setattr(build, "BINDING_PATH", str(tmp_path / "module.so"))
    monkeypatch.setattr(build, "BINDING_STAMP", str(tmp_path / "module.txt"), raising=False)
    calls = []

    def run(cmd, check):
        calls.append(cmd)
        open(cmd[cmd.index("-o") + 1], "w").close()

    monkeypatch.setattr(build.subprocess, "run", run)
    return calls


def test_built_again_for_another_pytorch(compiles, monkeypatch):
    build.build_binding()
    build.build_binding()
    assert len(compiles) == 1
    monkeypatch.setattr(torch, "__version__", "9.9.9")
    build.build_binding()
    assert len(compiles) == 2
    build.build_binding()
    assert len(compiles) == 2


def test_not_loaded_into_another_pytorch(compiles, monkeypatch):
    build.build_binding()
    monkeypatch.setattr(torch, "__version__", "9.9.9")
    before = bind.ext
    with pytest.raises(pkg.NVFP4Error, match="9.9.9"):
        bind.load()
    assert bind.ext is before
