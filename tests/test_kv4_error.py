"""The bound that a key of a cache of 4 bits is quantised by in 32 bits: not below the sum of what its roundings can be."""
import ctypes as C
import math
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "micro-expert-router-ssd-streamed-moe-mer_b200", "csrc")


def key_error(tmp_path):
    src, lib = tmp_path / "bound.cpp", tmp_path / "libbound.so"
    src.write_text('#include "kv4.h"\nextern "C" float key_error() { return KV4_KEY_ERROR; }\n')
    subprocess.check_call(["g++", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-I", CSRC, str(src), "-o", str(lib)])
    f = C.CDLL(str(lib)).key_error
    f.restype = C.c_float
    return f()


def test_the_bound_holds_every_rounding(tmp_path):
    """Of a pair (a, b) = (x norm weight, x' weight') of size r, rotated to values of at most M each: r <= sqrt(2) M, |a| + |b| <= sqrt(2) r, and |a cos| + |b sin| <= r.  A rounding is off by
    at most half a step, u of the value; an ulp of CUDA's functions is a whole step: u for a cosine or a sine below 1, up to 2 u of any other value."""
    u, r, both = 2.0 ** -24, math.sqrt(2.0), 2.0
    for d in range(8, 257, 8):
        lanes = max(8, 1 << (d // 8 - 1).bit_length())  # of a head, eight values each
        angle = math.pi * 2.0 ** -25 * r                # half-turns of at most 1, rounded
        turn = both * u + 2 * r * u                     # sincospif: 1 ulp; times rope_scale, times the weight
        sums = r * u + u                                # the first product, and the fma
        squares = 4 + 1 + math.log2(lanes)              # a lane's two sums of four squares, their sum, exchanges between lanes
        mean = (d & (d - 1) != 0) + 1                   # 1 / d as a 32-bit number, fma with eps
        norm = (squares + mean) / 2 * u + 2 * (2 * u) + u  # through the root half of it; rsqrtf: 2 ulp; the product
        total = angle + turn + sums + norm
        assert (1 + u) ** 64 * total <= key_error(tmp_path), (d, math.log2(total))  # and the roundings' products, and M's own
