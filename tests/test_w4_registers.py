"""The check that the compiler leaves the hand-scheduled loops' sums alone: what it finds in assembly written out here, and what it says of the library's."""
import os
import re
import shutil
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
sys.path.insert(0, str(ROOT / "tools"))
import check_w4_registers as check  # noqa: E402

LOOP = "\t;;#ASMSTART\n\ts_mov_b32 s72, s4\n\tv_mfma_i32_16x16x64_i8 a[0:3], v[0:3], v[4:7], a[0:3]\n\t;;#ASMEND\n"
FETCH = "\t;;#ASMSTART\n\tv_accvgpr_read_b32 v1, a{0}\n\tv_accvgpr_read_b32 v2, a{1}\n\t;;#ASMEND\n"
NAME = "_Z6kernelv"


def found(*lines):
    return check.overwritten(f"{NAME}:\n" + "".join(line if line.endswith("\n") else "\t" + line + "\n" for line in lines))[NAME]


@pytest.mark.parametrize("line,regs", [
    ("v_accvgpr_write_b32 a16, v3", {16}),
    ("v_accvgpr_mov_b32 a255, a0", {255}),
    ("scratch_load_dwordx4 a[14:17], off, off offset:16", {16, 17}),          # a range that begins among the fetched ones
    ("scratch_load_dword a20, off, off offset:16 ; 4-byte Folded Reload", {20}),
    ("global_load_dwordx2 a[30:31], v[0:1], off", {30, 31}),
    ("buffer_load_dword a40, v0, s[0:3], 0 offen", {40}),
    ("flat_load_dword a41, v[0:1]", {41}),
    ("ds_read_b128 a[252:255], v0", {252, 253, 254, 255}),
    ("v_mfma_f32_16x16x32_f16 a[100:103], v[0:3], v[4:7], 0", {100, 101, 102, 103}),
    ("v_accvgpr_write_b32 a3, v3", set()),                                     # fetched
    ("scratch_store_dwordx4 off, a[16:19], off", set()),                       # reads
    ("buffer_store_dword a40, v0, s[0:3], 0 offen", set()),
    ("ds_write_b32 v0, a17", set()),
    ("v_accvgpr_read_b32 v5, a90", set()),
    ("global_load_dwordx4 v[14:17], v[0:1], off", set()),
])
def test_what_counts_as_a_write(line, regs):
    assert found(LOOP, FETCH.format(0, 1), line) == regs


def test_before_and_behind_the_loop():
    clean = ["v_accvgpr_write_b32 a9, v3", LOOP, *(FETCH.format(16 * i, 16 * i + 1) for i in range(16)), "v_accvgpr_write_b32 a9, v3", "scratch_load_dwordx4 a[0:3], off, off"]
    assert found(*clean) == set()
    assert found(*clean[:9], "v_accvgpr_write_b32 a200, v3", *clean[9:]) == {200}
    assert found(LOOP, "v_accvgpr_write_b32 a1, v3", LOOP) == {1}              # between two loops, the second on top of the first one's sums


def test_status(tmp_path):
    good, bad, none = (tmp_path / f"{n}.s" for n in ("good", "bad", "none"))
    good.write_text(f"{NAME}:\n{LOOP}")
    bad.write_text(f"{NAME}:\n{LOOP}\tv_accvgpr_write_b32 a7, v3\n")
    none.write_text(f"{NAME}:\n\ts_endpgm\n")
    assert check.main([str(good)]) == 0 and check.main([str(bad)]) == 1 and check.main([str(none)]) == 1 and check.main([]) == 1


@pytest.mark.skipif(not shutil.which(os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")), reason="no hipcc")
def test_library():
    """As the build does (nothing to compile behind one)."""
    csrc = ROOT / "quantized-training_amd" / "csrc"
    subprocess.run(["make", "-s", f"-j{min(8, os.cpu_count() or 1)}", "-C", str(csrc), "registers"], check=True, capture_output=True, timeout=900)
    said = (csrc / "build" / "registers.txt").read_text()
    kernels, files, faults = map(int, re.search(r"(\d+) kernels .* in (\d+) files, (\d+) faults", said).groups())
    assert kernels >= 50 and files >= 12 and faults == 0
