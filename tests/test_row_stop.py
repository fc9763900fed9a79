"""Leaving a row loop after a wait that ran out (csrc/row_stop.h), on CPU: the
threads of a CTA as coroutines under random schedules, some of whose waits run
out.  However they interleave, all leave at the same row's barrier; the loop's
order of steps is that of the norm backward whose rows two CTAs share."""
import ctypes
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "nvfp4.5090_b200", "csrc", "row_stop.h")
SOURCE = f"""
#include "{HEADER}"
extern "C" {{
int never() {{ return nvfp4b200::row_stop::NEVER; }}
int before_barrier(int row) {{ return nvfp4b200::row_stop::before_barrier(row); }}
int after_barrier(int row) {{ return nvfp4b200::row_stop::after_barrier(row); }}
bool leaves(int stop, int row) {{ return nvfp4b200::row_stop::leaves(stop, row); }}
}}
"""


@pytest.fixture(scope="module")
def rule(tmp_path_factory):
    out = tmp_path_factory.mktemp("rows")
    src, so = out / "rows.cpp", out / "rows.so"
    src.write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-fPIC", "-shared", str(src), "-o", str(so)], check=True)
    lib = ctypes.CDLL(str(so))
    lib.leaves.restype = ctypes.c_bool
    return lib


def run(rng, threads, rows, chance, before, after, leaves, never, check_first=True):
    """The rows at which the threads left (None: walked them all).  "hang": some wait
    at a barrier that others will not reach."""
    stop = [never]

    def thread():
        for i in range(rows):
            if rng.random() < chance:                  # the row's copies are late for this thread
                stop[0] = min(stop[0], before(i))
            yield "step"
            yield "barrier"
            if check_first:
                leave = leaves(stop[0], i)
                yield "step"
            late = rng.random() < chance               # the other CTA's sums are late for this thread
            yield "step"
            if late and not (check_first and leave):
                stop[0] = min(stop[0], after(i))
            yield "step"
            if not check_first:
                leave = leaves(stop[0], i)
            if leave:
                return i
            yield "step"

    live, waiting, left = {k: thread() for k in range(threads)}, set(), {}
    while live:
        ready = [k for k in live if k not in waiting]
        if not ready:
            if len(waiting) < threads:                 # a barrier counts every thread of the CTA
                return "hang"
            waiting.clear()
            continue
        k = rng.choice(ready)
        try:
            if next(live[k]) == "barrier":
                waiting.add(k)
        except StopIteration as end:
            left[k] = end.value
            del live[k]
    return left


def test_all_leave_at_one_row(rule):
    rng = random.Random(1)
    stopped = 0
    for _ in range(3000):
        got = run(rng, rng.randint(2, 6), rng.randint(1, 6), 0.05, rule.before_barrier, rule.after_barrier, rule.leaves,
                  rule.never())
        assert got != "hang" and len(set(got.values())) == 1
        stopped += None not in got.values()
    assert stopped > 500


def test_the_schedules_find_a_rule_that_is_not_uniform(rule):
    """The same schedules with the comparison behind the second wait, and that wait's
    row its own: threads part, so the check above means something."""
    rng = random.Random(1)
    got = [run(rng, rng.randint(2, 6), rng.randint(1, 6), 0.05, lambda i: i, lambda i: i, rule.leaves, rule.never(), False)
           for _ in range(3000)]
    assert any(g == "hang" or len(set(g.values())) > 1 for g in got)


class Ring:
    """A ring of single-arrival transaction barriers.  Arming one whose phase is still
    open would be its second arrival in the phase: the hardware leaves that undefined."""

    def __init__(self, stages):
        self.open, self.parity = [False] * stages, [0] * stages

    def arm(self, st):
        assert not self.open[st], "armed twice in one phase"
        self.open[st] = True

    def land(self, st):
        self.open[st] = False
        self.parity[st] ^= 1


@pytest.mark.parametrize("refill_first", [False, True])
def test_refill_behind_the_check(refill_first):
    """A row whose copies are late: the loop leaves before its place is refilled, and
    every place is then waited for in the phase that is still open.  The other order
    arms a barrier twice."""
    def walk():
        for stages in (1, 2, 3):
            for late in range(6):
                ring, stage, parity, rows = Ring(stages), 0, 0, 6
                for st in range(stages):
                    ring.arm(st)
                for i in range(rows):
                    if i != late:
                        ring.land(stage)
                    arrived = ring.parity[stage] != parity
                    if refill_first and i + stages < rows:
                        ring.arm(stage)
                    if not arrived:
                        break
                    if not refill_first and i + stages < rows:
                        ring.arm(stage)
                    stage += 1
                    if stage == stages:
                        stage, parity = 0, parity ^ 1
                for st in range(stages):               # what is still open is waited for in its own phase
                    assert not ring.open[st] or ring.parity[st] == parity ^ (st < stage)

    if refill_first:
        with pytest.raises(AssertionError, match="twice"):
            walk()
    else:
        walk()


def test_kernels_refill_behind_the_check():
    """The order in the sources: each row loop leaves before it refills."""
    text = open(os.path.join(os.path.dirname(HEADER), "norm.cu")).read()
    parts = text.split("row_stop::leaves(")
    assert len(parts) == 3                             # the two loops that wait for copies
    for before, after in zip(parts, parts[1:]):
        loop = before[before.rindex("row_stop::before_barrier("):]
        assert "fetch(" not in loop and after.index("break;") < after.index("fetch(")
