"""The 256 x 256 kernel of the 8-bit linear leaves LDS reads in flight over the barrier
of a stage; those from before the barrier ahead of it have to be over, because the
copies that follow write into the slot they read.  Nothing in the source keeps the
compiler from moving the instructions that wait for them: the built code is looked at."""
import os
import re
import subprocess

import pytest

from nsw import _lib
from test_isa_waits import OBJDUMP, _device_objects


def late_reads(lines):
    """(barriers, LDS reads still in flight at the second barrier after them) of a listing, straight through."""
    flying, era, late = [], 0, 0
    for line in lines:
        op = line.split(None, 1)[0]
        if op.startswith("ds_"):
            flying.append(era if op.startswith("ds_read") else None)
        elif op == "s_waitcnt":
            m = re.search(r"lgkmcnt\((\d+)\)", line)
            if m:
                flying = flying[len(flying) - min(int(m.group(1)), len(flying)):]
        elif op == "s_barrier":
            late += sum(e is not None and e < era for e in flying)
            era += 1
    return era, late


def test_the_scan_sees_a_late_read():
    read, barrier = "ds_read_b128 v[0:3], v4", "s_barrier"
    assert late_reads([read, barrier]) == (1, 0)
    assert late_reads([read, barrier, barrier]) == (2, 1)
    assert late_reads([read, barrier, "s_waitcnt lgkmcnt(0)", barrier]) == (2, 0)
    assert late_reads([read, barrier, read, "s_waitcnt vmcnt(3) lgkmcnt(1)", barrier]) == (2, 0)
    assert late_reads([read, barrier, read, "s_waitcnt lgkmcnt(2)", barrier]) == (2, 1)


@pytest.mark.skipif(not os.path.exists(OBJDUMP), reason="no disassembler for the device code")
def test_reads_end_before_their_slot_is_written(tmp_path):
    seen = 0
    for i, obj in enumerate(_device_objects(_lib.LIB_PATH)):
        f = tmp_path / f"{i}.o"
        f.write_bytes(obj)
        r = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", "--mcpu=gfx950", str(f)], capture_output=True, text=True, check=True)
        for fn in re.split(r"\n(?=[0-9a-f]+ <)", r.stdout):
            if "linear_fp8_deep_kernel" not in fn.split("\n", 1)[0]:
                continue
            lines = [l.split("//")[0].strip() for l in fn.splitlines() if l.startswith("\t")]
            loop = max(i for i, l in enumerate(lines) if l.startswith("v_mfma")) + 1
            # the loop's stages twice over: its last one is followed by its first
            barriers, late = late_reads(lines[:loop] * 2)
            assert barriers >= 8 and late == 0, fn.split("\n", 1)[0]
            seen += 1
    assert seen == 5
