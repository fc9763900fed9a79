"""The torch extension module ``lib/_nvfp4b200_torch.so`` (csrc/torch_binding.cpp):
checks, allocation and launch of the MXFP4, clipping and sandwich-norm calls
in one C++ call each, on top of the C ABI library next to it.

``ext`` is the module; before the first use it is a stand-in that loads it, so
that the package can be imported in order to build it.  There is no fallback:
a missing module raises NVFP4Error."""
from __future__ import annotations

import importlib.machinery
import importlib.util
import os

from . import _build, _lib


def load():
    """Load the extension module (after the C ABI library, which it links)."""
    global ext
    path = _build.BINDING_PATH
    if not os.path.exists(path):
        raise _lib.NVFP4Error(f"torch binding not found at {path}; build it with "
                              "`python -c 'import __graft_entry__ as g; g.build()'` (no fallback exists)")
    made = _build.binding_built_for()
    if made and made != _build.binding_target():   # its calls into another PyTorch would crash
        raise _lib.NVFP4Error(f"the torch binding was built for {made}, this is {_build.binding_target()}: build it again with "
                              "`python -c 'import __graft_entry__ as g; g.build()'`")
    _lib.load()
    loader = importlib.machinery.ExtensionFileLoader(_build.BINDING_NAME, path)
    module = importlib.util.module_from_spec(importlib.util.spec_from_loader(_build.BINDING_NAME, loader))
    loader.exec_module(module)
    ext = module
    return module


class _Unloaded:
    def __getattr__(self, name):
        return getattr(load(), name)


ext = _Unloaded()
