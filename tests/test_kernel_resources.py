"""Registers that the built forward kernels spill, read from the code objects' own metadata: work that is added for one variant
of a kernel template must not cost the others registers.  (Spills to scratch memory in a tile loop are paid per tile.)"""
import os
import re
import struct
import subprocess

import pytest

import cabi

READOBJ = "/opt/rocm/llvm/bin/llvm-readobj"
MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"


def _code_objects(path):
    """The gfx950 code objects of a library: one bundle per translation unit."""
    data = open(path, "rb").read()
    at = data.find(MAGIC)
    while at >= 0:
        n, = struct.unpack_from("<Q", data, at + len(MAGIC))
        pos = at + len(MAGIC) + 8
        for _ in range(n):
            offset, size, length = struct.unpack_from("<QQQ", data, pos)
            if b"gfx950" in data[pos + 24:pos + 24 + length]:
                yield data[at + offset:at + offset + size]
            pos += 24 + length
        at = data.find(MAGIC, at + len(MAGIC))


def _spills(path, tmp_path):
    found = {}
    for i, obj in enumerate(_code_objects(path)):
        f = tmp_path / ("%d.co" % i)
        f.write_bytes(obj)
        notes = subprocess.run([READOBJ, "--notes", str(f)], capture_output=True, text=True, check=True).stdout
        for m in re.finditer(r"\.symbol:\s+'?(\S+?)\.kd'?\n(?:.*\n)*?\s+\.vgpr_spill_count:\s+(\d+)", notes):
            found[m.group(1)] = int(m.group(2))
    return found


# (DP, load path, dropout, split, packed heads, DV) of fwd_prefill_kernel -> spilled vector registers; the others spill none
SPILLED = {(128, 0, 0, 0, 0, 128): 11, (128, 0, 1, 0, 0, 128): 28, (256, 0, 0, 0, 0, 256): 118, (256, 0, 1, 0, 0, 256): 171,
           (256, 3, 0, 0, 1, 256): 8, (256, 3, 0, 1, 1, 256): 5, (256, 4, 0, 0, 1, 256): 6, (256, 4, 0, 1, 1, 256): 2}


@pytest.mark.skipif(not os.path.exists(READOBJ), reason="no llvm-readobj")
def test_no_forward_kernel_spills_more_than_it_did(tmp_path):
    found = _spills(cabi.LIB_PATH, tmp_path)
    seen = set()
    for name, spills in found.items():
        m = re.search(r"fwd_prefill_kernelILi(\d+)ELb[01]ELi[48]ELi(\d)ELb([01])ELb([01])ELb([01])ELi(\d+)E", name)
        if m:
            key = tuple(int(x) for x in m.groups())
            seen.add(key)
            assert spills <= SPILLED.get(key, 0), "%s spills %d vector registers" % (name, spills)
    assert set(SPILLED) <= seen and len(seen) > 20
