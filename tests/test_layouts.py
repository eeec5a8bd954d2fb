"""What the launchers ask of strides (launch.h): which layouts lie apart, and which meet a second one beside them."""
import ctypes
import itertools
import os
import random
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mimizuku_b200", "csrc")
CUDA = os.environ.get("CUDA_HOME", "/usr/local/cuda")
SRC = """#include "launch.h"
extern "C" int is_apart(long long room, const int* n, const long long* s) {
    return mmz::apart(room, {{n[0], s[0]}, {n[1], s[1]}, {n[2], s[2]}});
}
extern "C" int do_meet(long long by, long long room, const int* n, const long long* s) {
    return mmz::meet(by, room, {{n[0], s[0]}, {n[1], s[1]}, {n[2], s[2]}});
}
"""


@pytest.fixture(scope="module")
def fns(tmp_path_factory):
    cxx = os.environ.get("CXX", "g++")
    if not shutil.which(cxx):
        pytest.skip("no C++ compiler")
    d = tmp_path_factory.mktemp("layouts")
    (d / "l.cpp").write_text(SRC)
    so = str(d / "l.so")
    subprocess.run([cxx, "-std=c++17", "-shared", "-fPIC", "-I", CSRC, "-I", f"{CUDA}/include", str(d / "l.cpp"), "-o", so],
                   check=True)
    lib = ctypes.CDLL(so)
    n3 = lambda n: (ctypes.c_int * 3)(*n)  # noqa: E731
    s3 = lambda s: (ctypes.c_longlong * 3)(*s)  # noqa: E731
    return (lambda room, n, s: bool(lib.is_apart(ctypes.c_longlong(room), n3(n), s3(s))),
            lambda by, room, n, s: bool(lib.do_meet(ctypes.c_longlong(by), ctypes.c_longlong(room), n3(n), s3(s))))


def places(n, s):
    return [sum(i * x for i, x in zip(at, s)) for at in itertools.product(*map(range, n))]


def test_against_every_pair_of_items(fns):
    apart, meet = fns
    rng = random.Random(5)
    seen = {(a, b): 0 for a in (0, 1) for b in (0, 1)}
    for _ in range(4000):
        room = rng.choice([1, 2, 3, 8])
        n = [rng.choice([1, 2, 3, 4]) for _ in range(3)]
        if rng.random() < 0.5:  # a dense or padded nest in some order
            s, ext = [0, 0, 0], room
            for i in rng.sample(range(3), 3):
                s[i] = (ext + rng.choice([0, 0, 1, 7])) * rng.choice([1, 1, -1, 2])
                ext += abs(s[i]) * (n[i] - 1)
        else:
            s = [rng.randint(-40, 40) for _ in range(3)]
        at = places(n, s)
        clash = any(abs(x - y) < room for x, y in itertools.combinations(at, 2))
        a = apart(room, n, s)
        assert not (a and clash), (room, n, s)
        seen[a, clash] += 1
        if not a:
            continue
        for by in [rng.randint(-120, 120) for _ in range(6)] + [0, room, -room]:
            want = any(abs(x - y - by) < room for x in at for y in at)
            assert meet(by, room, n, s) == want, (by, room, n, s)
    assert seen[1, 0] > 1500 and seen[0, 1] > 500


def test_numbers_near_2_to_63(fns):
    apart, meet = fns
    big = 1 << 62
    assert apart(64, (2, 2, 2), (big, 64, 128)) and meet(big, 64, (2, 2, 2), (big, 64, 128))
    assert meet(-big + 63, 64, (2, 2, 2), (-big, 64, 128)) and not meet(big - 1000, 64, (2, 2, 2), (big, 64, 128))
    low = -(1 << 63)
    assert apart(1, (2, 1, 1), (low, 0, 0)) and meet(low, 1, (2, 1, 1), (low, 0, 0)) and not meet(low + 1, 1, (2, 1, 1), (low, 0, 0))
