"""Checks the compiled code around the hand-scheduled loops (gen_w4_asm.py): they leave their sums in a[0:255], and the statements that fetch them from there
are all that the compiler knows of it.  It must not put a value of its own into an accumulator register that has not been fetched yet -- which it does when an
epilogue needs more registers than are left.  Compiles every source that contains such a loop to assembly and lists what it finds; exit status 1 if anything.

Run after a change to an epilogue of those kernels:  python tools/check_w4_registers.py   (about two minutes)
"""
import re
import subprocess
import sys
import tempfile
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "quantized-training_amd" / "csrc"
FLAGS = ("--offload-arch=gfx950 -O3 -std=c++17 -fPIC -ffp-contract=off -fno-fast-math -w -Xclang -target-feature -Xclang -packed-fp32-ops "
         "--cuda-device-only -S").split()
WRITES = re.compile(r"v_accvgpr_(?:write|mov)_b32 a(\d+)|\b(?:global_load|buffer_load|scratch_load|ds_read)\S* a\[?(\d+)")


def overwritten(text):
    """{kernel: registers that the compiler wrote behind a loop and before they were fetched}"""
    kernel, in_asm, first, seen, left, out = None, False, False, False, set(), {}
    for line in text.splitlines():
        m = re.match(r"(_Z\S+):", line)
        if m:
            kernel, seen = m.group(1), False
        elif "ASMSTART" in line:
            in_asm = first = True
        elif "ASMEND" in line:
            in_asm = False
        elif in_asm and first and re.search(r"s_mov_b32 s(72|92),", line):          # a loop begins
            first, seen, left = False, True, set(range(256))
            out.setdefault(kernel, set())
        elif in_asm and first and "v_accvgpr_read" in line:                         # sixteen sums are fetched
            first, at = False, int(re.search(r", a(\d+)", line).group(1))
            left -= set(range(at, at + 16))
        elif seen and not in_asm:
            for m in WRITES.finditer(line):
                r = int(m.group(1) or m.group(2))
                if r in left:
                    out[kernel].add(r)
    return out


def compile_to_asm(src):
    with tempfile.TemporaryDirectory() as d:
        dst = Path(d) / "out.s"
        subprocess.run(["hipcc", *FLAGS, str(src), "-o", str(dst)], check=True, cwd=CSRC)
        return dst.read_text()


def main():
    sources = [p for p in sorted(CSRC.glob("*.hip")) if re.search(r"gnk_(gemm_w4|grouped)\.h", p.read_text())]
    bad = kernels = 0
    with ThreadPoolExecutor(8) as pool:
        for src, text in zip(sources, pool.map(compile_to_asm, sources)):
            for kernel, regs in overwritten(text).items():
                kernels += 1
                if regs:
                    bad += 1
                    print(f"{src.name}: {kernel} writes a{sorted(regs)} before they are fetched")
    print(f"{kernels} kernels with a hand-scheduled loop in {len(sources)} files, {bad} overwrite sums")
    return 1 if bad or not kernels else 0


if __name__ == "__main__":
    sys.exit(main())
