"""The kernels' sources: lanes of a wave that exchange data through LDS are ordered by wave_sync_lds (a fence at wavefront scope
on both sides of the barrier). The bare barrier orders no memory for the compiler, which might move a lane's reads of what other
lanes write across it. Runs on the CPU, over the text."""
import glob
import os
import re

from paths import package

CSRC = os.path.join(os.path.dirname(package().hip_engine.LIBRARY), "csrc")


def test_no_exchange_behind_a_bare_wave_barrier():
    bare = re.compile(r"\b__builtin_amdgcn_wave_barrier\s*\(")
    found = []
    for path in sorted(glob.glob(os.path.join(CSRC, "*"))):
        if not path.endswith((".hip", ".hpp", ".cpp")):
            continue
        lines = open(path).read().splitlines()
        for i, line in enumerate(lines):
            if bare.search(line):
                around = [x for x in lines[max(0, i - 1):i + 2] if '__builtin_amdgcn_fence' in x and '"wavefront"' in x]
                if len(around) < 2:
                    found.append((os.path.basename(path), i + 1))
    assert not found, found
