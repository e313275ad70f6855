"""Checks the compiled code around the hand-scheduled loops (gen_w4_asm.py): they leave their sums in a[0:255], and the statements that fetch them from there
are all that the compiler knows of it.  It must not put a value of its own into an accumulator register that has not been fetched yet -- which it does when an
epilogue needs more registers than are left.  Lists what it finds; exit status 1 if anything, or if no loop was found.

The Makefile of csrc/ compiles every source with such a loop to assembly, with the library's own flags, and links the library only if this passes
(`make -C quantized-training_amd/csrc registers` does that much alone):  python3 tools/check_w4_registers.py FILE.s ...
"""
import re
import sys
from pathlib import Path

# what an instruction writes is its first operand; these have a source there
READS_ONLY = re.compile(r"\w*(?:store|ds_write|atomic)\w*$")
REGISTERS = re.compile(r"a(?:(\d+)|\[(\d+):(\d+)\])$")


def written(line):
    """Accumulator registers that an instruction writes."""
    code = line.split(";")[0].split("//")[0].strip()
    name, _, operands = code.partition(" ")
    m = REGISTERS.match(operands.split(",")[0].strip())
    if not m or READS_ONLY.match(name):
        return set()
    return {int(m[1])} if m[1] else set(range(int(m[2]), int(m[3]) + 1))


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
            out[kernel] |= written(line) & left
    return out


def main(files):
    bad = kernels = 0
    for f in files:
        found = overwritten(Path(f).read_text())
        if not found and Path(f).stem != "gnk_grouped":                            # its entry points; the kernels are in the others
            bad += 1
            print(f"{f}: no hand-scheduled loop")
        for kernel, regs in found.items():
            kernels += 1
            if regs:
                bad += 1
                print(f"{f}: {kernel} writes a{sorted(regs)} before they are fetched")
    print(f"{kernels} kernels with a hand-scheduled loop in {len(files)} files, {bad} faults")
    return 1 if bad or not kernels else 0


if __name__ == "__main__":
    sys.exit(main(sys.argv[1:]))
