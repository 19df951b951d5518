"""Registers of the tensor-core attention kernel over a cache of 16 bits, as the compiler reports them: its softmax threads hold a row's scores, and what they spill, all of them wait for.
The forms of a cache of 4 bits share its source."""
import importlib
import os
import re
import subprocess

import mer_b200  # noqa: F401

build = importlib.import_module("mer_b200._build")


def test_16_bit_forms_keep_their_scores_in_registers(tmp_path):
    flags = [f for f in build.NVCC_FLAGS if f != "--use_fast_math=false"]
    said = subprocess.run([build._nvcc(), *flags, "-Xptxas", "-v", "-c", os.path.join(build.CSRC, "kernels_attend_tc.cu"), "-o", str(tmp_path / "tc.o")],
                          check=True, stderr=subprocess.PIPE, text=True).stderr
    # <type, padded head, units of a cache of 4 bits>, mangled
    found = re.findall(r"k_attend_tcI(\w+?)Li(\d+)ELi0EE.*?(\d+) bytes spill stores, (\d+) bytes spill loads", said, re.S)
    spills = {(kind, int(d)): (int(stores), int(loads)) for kind, d, stores, loads in found}
    assert len(spills) == 6, said
    most = {64: (0, 0), 128: (12, 4), 256: (0, 0)}
    assert {k: v for k, v in spills.items() if v[0] > most[k[1]][0] or v[1] > most[k[1]][1]} == {}
