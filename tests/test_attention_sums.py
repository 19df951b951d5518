"""The sum by which the attention kernels count blocks, against adding up, without a GPU."""
import ctypes as C
import os
import random
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "micro-expert-router-ssd-streamed-moe-mer_b200", "csrc")


@pytest.fixture(scope="module")
def points(tmp_path_factory):
    d = tmp_path_factory.mktemp("points")
    src, lib = d / "points.cpp", d / "libpoints.so"
    src.write_text('#include <cuda_runtime.h>\n#include "attend_work.h"\n'
                   'extern "C" uint64_t points(uint32_t n, uint32_t m, uint32_t a, uint32_t b) { return points_under(n, m, a, b); }\n')
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-I", CSRC, "-I", "/usr/local/cuda/include", str(src), "-o", str(lib)])
    f = C.CDLL(str(lib)).points
    f.restype, f.argtypes = C.c_uint64, [C.c_uint32] * 4
    return f


def test_every_small_line(points):
    for m in range(1, 12):
        for a in range(0, 26):
            for b in range(0, 26):
                total = 0
                for n in range(0, 15):
                    assert points(n, m, a, b) == total, (n, m, a, b)
                    total += (a * n + b) // m


def test_lines_of_long_sequences(points):
    rng = random.Random(3)
    for _ in range(300):
        m, a, n = rng.choice([64, 128]), rng.randint(1, 256), rng.randint(1, 5000)
        b = rng.choice([rng.randint(0, 300), rng.randint(0, 1 << 30), (1 << 32) - 1 - a * n])  # up to the last value that 32 bits hold
        assert points(n, m, a, b) == sum((a * i + b) // m for i in range(n)), (n, m, a, b)
