"""Sources: a kernel's limit of dynamic shared memory belongs to the kernel and
the device, so every launch sets the same one.  A limit that depends on the
call's sizes could be lowered by another host thread between a call's setting
and its launch, which is then refused."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nvfp4.5090_b200", "csrc")


def test_limits_are_constants():
    seen = 0
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu*"))):
        text = open(path).read()
        limits = re.findall(r"allow_smem\([\w:]+, ((?:[^()]|\([^()]*\))+)\)", text)
        limits += re.findall(r"MaxDynamicSharedMemorySize,\s*((?:[^()]|\([^()]*\))+)\)", text)
        for value in limits:
            if os.path.basename(path) == "common.cuh" and value == "most":
                continue   # allow_smem itself
            seen += 1
            name = value.split("::")[-1]
            assert value == "(int)sizeof(TqSmem)" or re.search(rf"constexpr int {name} =", text), f"{os.path.basename(path)}: {value}"
    assert seen >= 7
