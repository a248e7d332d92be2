"""hxinfer_b200/csrc/hx_split.h, which cuts the shared-prefix decode's work into
parts, compiled for the host and checked against Python's integers."""
import ctypes as C
import os
import random
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "hxinfer_b200", "csrc")


@pytest.fixture(scope="module")
def split(tmp_path_factory):
    gxx = shutil.which("g++")
    if not gxx:
        pytest.skip("g++ not present")
    tmp = tmp_path_factory.mktemp("split")
    src, lib = tmp / "split.cpp", tmp / "split.so"
    src.write_text('#include "hx_split.h"\nextern "C" {\n'
                   "int64_t first(int64_t i, int n, int c) { return hx::split_first(i, n, c); }\n"
                   "int owner(int64_t i, int n, int64_t x) { return hx::split_owner(i, n, x); }\n}\n")
    subprocess.run([gxx, "-std=c++17", "-O1", "-shared", "-fPIC", f"-I{CSRC}", str(src), "-o", str(lib)], check=True)
    lib = C.CDLL(str(lib))
    lib.first.restype, lib.first.argtypes = C.c_int64, [C.c_int64, C.c_int, C.c_int]
    lib.owner.restype, lib.owner.argtypes = C.c_int, [C.c_int64, C.c_int, C.c_int64]
    return lib


def test_parts_and_owners(split):
    """Small lists, and lists around and past 2^32 items (whose first items lie
    below it), in as many parts as the GPU has CTAs or suffix warps."""
    rng = random.Random(1)
    for items in [1, 2, 3, 7, 147, 148, 149, 1000, 123457, 2 ** 31 - 1, 2 ** 32 - 1, 2 ** 32, 2 ** 32 + 5, 10 ** 11]:
        for n in (1, 2, 5, 148, 1184):
            if n > items:
                continue
            starts = [items * c // n for c in range(n + 1)]
            for c in range(n + 1):
                assert split.first(items, n, c) == starts[c]
            probe = {0, items - 1, *(x for x in starts[:-1]), *(x - 1 for x in starts[1:])}
            probe |= {rng.randrange(items) for _ in range(50)}
            for x in probe:
                k = split.owner(items, n, x)
                assert starts[k] <= x < starts[k + 1], (items, n, x, k)
