"""Build check of the inline-asm loads to LDS.

csrc/attention_batch.hip (load_to_lds) loads straight to LDS with an inline-asm
`buffer_load_dwordx4 ..., offen lds` whose LDS address is in M0 and whose buffer
descriptor the compiler forms with v_readfirstlane.  gfx950 needs 5 wait states
between a vector instruction that writes a scalar register and a
vector-memory instruction that reads it, and one between the write of M0 and
the load; the compiler keeps those distances for its own instructions only, so
the asm block has to bring them.  And M0 is the block's: what the compiler
holds there is lost.

This script reads the device assembly (`hipcc -S --offload-device-only`, inline
asm between `;;#ASMSTART` / `;;#ASMEND` markers) and checks of every inline-asm
load to LDS that its own block writes M0 before it and gives 5 wait states in front
of it (an instruction is one, `s_nop N` N + 1), and of every function that
nothing outside the blocks reads M0 behind one without writing it first.  It
exits non-zero, naming the function, where one does not hold.

Usage: python check_lds_loads.py build/attention_batch.s
"""
import re
import sys

from check_vmcnt import functions

WAIT_STATES = 5
LDS_LOAD = re.compile(r"^buffer_load\w*\s.*\blds\b")
NOP = re.compile(r"^s_nop\s+(0x[0-9a-fA-F]+|\d+)$")
M0_WRITE = re.compile(r"^\w+\s+m0\b")
M0 = re.compile(r"\bm0\b")


def check_function(name, body):
    """Problems found in one function, and the number of loads checked."""
    problems, checked = [], 0
    in_asm = False
    foreign = False  # M0 holds what an asm block wrote
    states = 0       # wait states since the block's start
    wrote = False    # the block has written M0
    for s in body:
        if s.startswith(";;#ASMSTART"):
            in_asm, states, wrote = True, 0, False
            continue
        if s.startswith(";;#ASMEND"):
            in_asm = False
            continue
        s = s.split(";")[0].strip()
        if not s or s.startswith(".") or s.endswith(":"):
            continue
        if not in_asm:
            if M0_WRITE.match(s):
                foreign = bool(foreign and M0.search(s.split(",", 1)[-1]))
            if foreign and M0.search(s):
                problems.append(f"{name}: M0 read behind an asm block that wrote it: {s}")
            continue
        if LDS_LOAD.match(s):
            checked += 1
            if not wrote:
                problems.append(f"{name}: a load to LDS whose block does not write M0")
            if states < WAIT_STATES:
                problems.append(f"{name}: {states} wait states before a load to LDS, {WAIT_STATES} needed")
        if M0_WRITE.match(s):
            wrote = foreign = True
        m = NOP.match(s)
        states += int(m.group(1), 0) + 1 if m else 1
    return problems, checked


def check(text):
    problems, checked = [], 0
    for name, body in functions(text.splitlines()):
        p, c = check_function(name, body)
        problems += p
        checked += c
    return problems, checked


def main(argv):
    if len(argv) != 2:
        print(__doc__.strip().splitlines()[-1])
        return 2
    problems, checked = check(open(argv[1]).read())
    for p in problems[:20]:
        print("check_lds_loads:", p)
    if checked == 0:
        print("check_lds_loads: no loads to LDS found (assembly of csrc/attention_batch.hip expected)")
        return 1
    if problems:
        return 1
    print(f"check_lds_loads: {checked} loads to LDS hold")
    return 0


if __name__ == "__main__":
    sys.exit(main(sys.argv))
