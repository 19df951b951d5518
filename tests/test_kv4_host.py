"""A cache of 4 bits, without a GPU: where the bytes of a page lie, and which pages are refused."""
import ctypes as C
import os
import subprocess

import pytest

import mer_b200

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "micro-expert-router-ssd-streamed-moe-mer_b200", "csrc")
SOURCE = r"""
#include "kv4.h"
extern "C" {
void shape(uint32_t d, uint32_t page, uint32_t group, uint64_t *out) {
  const Kv4Shape s = kv4_shape(d, page, group);
  out[0] = s.units, out[1] = s.groups, out[2] = s.codes, out[3] = kv4_block_bytes(s, page);
}
const char *fault(uint32_t d, uint32_t page, uint32_t group, uint32_t heads, uint32_t n, uint64_t page_stride, uint64_t token_stride, uint64_t head_stride) {
  return kv4_pages_fault(kv4_shape(d, page, group), page, heads, n, page_stride, token_stride, head_stride);
}
}
"""


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    d = tmp_path_factory.mktemp("kv4")
    src, lib = d / "rules.cpp", d / "librules.so"
    src.write_text(SOURCE)
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-I", CSRC, str(src), "-o", str(lib)])
    r = C.CDLL(str(lib))
    r.fault.restype = C.c_char_p
    r.fault.argtypes = [C.c_uint32] * 5 + [C.c_uint64] * 3
    return r


def test_blocks_hold_every_code_and_scale(rules):
    out = (C.c_uint64 * 4)()
    for group in (32, 64):
        for d in range(8, 257, 8):
            for page in (1, 2, 5, 16, 24, 1 << 20):
                rules.shape(d, page, group, out)
                units, groups, codes, block = out
                assert units in (2, 3, 4, 6, 8) and 32 * units >= d and groups * group >= 32 * units > (groups - 1) * group
                assert codes == page * units * 16 and block % 16 == 0 and 0 <= block - (codes + page * groups * 4) < 16
                assert mer_b200.kv4_block_bytes(d, page, group) == block
                # every place of a token's codes is one value's: whole words of keys, half words of values
                keys = {((v % 32 // 8) * units + v // 32) * 8 + v % 8 // 2 + v % 2 * 4 for v in range(32 * units)}
                values = {((v % 32 // 4) * units + v // 32) * 4 + v % 4 for v in range(32 * units)}
                assert keys == values == set(range(32 * units))


def test_block_bytes_of_what_is_no_cache():
    for d, page, group in ((0, 16, 32), (12, 16, 32), (264, 16, 32), (64, 0, 32), (64, (1 << 20) + 1, 32), (64, 16, 16), (64, 16, 128)):
        with pytest.raises(ValueError):
            mer_b200.kv4_block_bytes(d, page, group)


def test_pages_that_are_refused(rules):
    block = mer_b200.kv4_block_bytes(128, 16, 32)
    assert block == 16 * 80
    good = dict(d=128, page=16, group=32, heads=4, n=9, page_stride=4 * block, token_stride=0, head_stride=block)
    ask = lambda **kw: rules.fault(*{**good, **kw}.values())  # noqa: E731
    assert ask() is None
    assert ask(page_stride=block, head_stride=9 * block) is None  # heads outermost
    assert ask(heads=1, head_stride=0) is None and ask(n=1, page_stride=0) is None
    assert b"token stride" in ask(token_stride=80)
    for kw in (dict(page_stride=4 * block + 8), dict(head_stride=block + 4)):
        assert b"multiples" in ask(**kw)
    for kw in (dict(page_stride=block - 16), dict(head_stride=block - 16), dict(head_stride=0)):
        assert b"smaller" in ask(**kw)
    for kw in (dict(page_stride=1 << 36), dict(head_stride=1 << 46), dict(page_stride=(1 << 64) - 16), dict(head_stride=(1 << 64) - 16)):
        assert b"64 GB" in ask(**kw)
    assert ask(n=3, page_stride=(1 << 36) - 16) is None
    for kw in (dict(n=0xFFFFFFFF, page_stride=1 << 20), dict(n=4000, page_stride=(1 << 36) - 16), dict(heads=4000, head_stride=(1 << 36) - 16)):
        assert b"2^47" in ask(**kw)
