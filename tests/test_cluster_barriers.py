"""Sources: the aligned cluster barrier is executed by whole warps, so every
place that issues it lets the warp's lanes meet first."""
import glob
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_lanes_meet_before_an_aligned_cluster_barrier():
    seen = 0
    for path in sorted(glob.glob(os.path.join(ROOT, "nvfp4.5090_b200", "csrc", "*.cu*"))):
        text = open(path).read()
        for m in re.finditer(r"asm volatile\(\s*\"barrier\.cluster\.arrive[.\w]*\.aligned", text):
            seen += 1
            before = text[:m.start()].rstrip()
            assert before.endswith("__syncwarp();"), f"{os.path.basename(path)}: {text[m.start() - 120:m.end()]}"
    assert seen >= 3
