"""Which tile counter a GEMM launch takes (csrc/sched_slots.h), on CPU: no two
launches that can run at the same time ever share one."""
import ctypes
import os
import subprocess
import threading

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "nvfp4.5090_b200", "csrc", "sched_slots.h")
STREAMS, GRAPHS = 4, 6

SOURCE = f"""
#include "{HEADER}"
using S = nvfp4b200::SchedSlots<{STREAMS}, {GRAPHS}>;
extern "C" {{
void* make() {{ return new S; }}
int of_stream(void* s, unsigned long long id) {{ return static_cast<S*>(s)->of_stream(id); }}
int take(void* s) {{ return static_cast<S*>(s)->take(); }}
void give_back(void* s, int slot) {{ static_cast<S*>(s)->give_back(slot); }}
}}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    out = tmp_path_factory.mktemp("slots")
    src, so = out / "slots.cpp", out / "slots.so"
    src.write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-fPIC", "-shared", "-pthread", str(src), "-o", str(so)], check=True)
    lib = ctypes.CDLL(str(so))
    lib.make.restype = ctypes.c_void_p
    lib.of_stream.argtypes = [ctypes.c_void_p, ctypes.c_ulonglong]
    lib.take.argtypes = [ctypes.c_void_p]
    lib.give_back.argtypes = [ctypes.c_void_p, ctypes.c_int]
    return lib


def test_a_stream_keeps_its_counter_however_many_launches(lib):
    s = lib.make()
    ids = [7, 2 ** 40, 9]
    first = [lib.of_stream(s, i) for i in ids]
    assert len(set(first)) == 3 and all(0 <= v < STREAMS for v in first)
    for _ in range(1000):
        assert [lib.of_stream(s, i) for i in ids] == first


def test_captured_launches_share_with_nobody(lib):
    """A captured launch's counter is no stream's and no other captured launch's,
    however many launches come after it, until it is given back."""
    s = lib.make()
    streams = {lib.of_stream(s, i) for i in range(STREAMS)}
    held = [lib.take(s) for _ in range(GRAPHS)]
    for _ in range(1000):
        assert lib.of_stream(s, 0) in streams
    assert len(set(held) | streams) == GRAPHS + STREAMS and min(held) >= STREAMS and max(held) < STREAMS + GRAPHS
    assert lib.take(s) == -1                      # all held: no counter
    assert lib.of_stream(s, 99) == -1             # and none for one more stream
    lib.give_back(s, held[2])
    lib.give_back(s, held[0])
    assert [lib.take(s), lib.take(s), lib.take(s)] == [held[2], held[0], -1]


def test_from_many_threads(lib):
    """Threads that take, hold and give back: nobody is ever handed a held counter."""
    s = lib.make()
    lock, held, bad = threading.Lock(), set(), []

    def work(i):
        for _ in range(2000):
            slot = lib.take(s)
            if slot < 0:
                continue
            with lock:
                if slot in held:
                    bad.append(slot)
                held.add(slot)
            with lock:
                held.discard(slot)
            lib.give_back(s, slot)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_given_back_many_times(lib):
    """Around the end of the list of counters given back, in the order they came."""
    s = lib.make()
    held = [lib.take(s) for _ in range(GRAPHS)]
    for i in range(50):
        out = held[: 1 + i % GRAPHS]
        for slot in out:
            lib.give_back(s, slot)
        again = [lib.take(s) for _ in out]
        assert again == out and lib.take(s) == -1
        held = held[len(out):] + again
    assert sorted(held) == list(range(STREAMS, STREAMS + GRAPHS))


def test_nothing_is_allocated():
    """A C entry point lets no exception through: the header holds no container that can throw."""
    text = open(HEADER).read()
    assert not any(w in text for w in ("unordered_map", "deque", "vector", "new "))
