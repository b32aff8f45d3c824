"""Reads of a matrix instruction's result that come too soon (no GPU):  python tests/probes/mfma_wait_scan.py [source.hip ...]   (default: every source of the library)

A vector instruction may read the result of a matrix instruction only some wait states after it; the compiler counts them, but where both arms of a branch lead from the one to
the other it has been seen to count along one arm only.  This compiles each source to assembly and follows every path from every matrix instruction - s_nop n counts n + 1, any
other instruction 1 - until something reads or overwrites its result registers, or enough states have passed.  Prints the suspicious pairs per kernel; the last line of a source
is their number (0 expected)."""
import os
import re
import subprocess
import sys
import tempfile

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.dirname(os.path.abspath(__file__)))))
from diffpure_amd import build  # noqa: E402

# wait states from a matrix instruction to a vector instruction that reads its result, by passes (gfx950)
STATES = [("32x32x16", 12), ("32x32x2_", 18), ("16x16x4_f32", 10), ("16x16x32", 8)]
MOST = 19


def registers(text):
    out = {(m[1], i) for m in re.finditer(r"\b([av])\[(\d+):(\d+)\]", text) for i in range(int(m[2]), int(m[3]) + 1)}
    return out | {(m[1], int(m[2])) for m in re.finditer(r"\b([av])(\d+)\b", text)}


def first_operand(args):
    head = args.split(",")[0]
    return args[:args.index("]") + 1] if "[" in head else head


def too_soon(ins, labels):
    bad = []
    for i, (op, args) in enumerate(ins):
        if not op.startswith("v_mfma"):
            continue
        need = next((n for s, n in STATES if s in op), MOST)
        result, todo, seen = registers(first_operand(args)), [(i + 1, 0)], {}
        while todo:
            j, waited = todo.pop()
            while j < len(ins) and waited < need and seen.get(j, MOST + 1) > waited:
                seen[j] = waited
                o, a = ins[j]
                if o.startswith("v_mfma"):
                    if registers(first_operand(a)) & result:      # accumulates onto it: the hardware's own interlock
                        break
                elif o == "s_endpgm":
                    break
                elif o == "s_branch":
                    j = labels[a.strip()] - 1
                elif o.startswith("s_cbranch"):
                    todo.append((labels[a.strip()], waited + 1))
                elif not o.startswith("s_") and registers(a) & result:
                    bad.append((op, o, waited, need))
                    break
                waited += int(a) + 1 if o == "s_nop" else 1
                j += 1
    return bad


def scan(path):
    with tempfile.TemporaryDirectory() as tmp:
        out = os.path.join(tmp, "a.s")
        subprocess.run([build._hipcc()] + build.HIP_FLAGS + ["--offload-device-only", "-S", "-o", out, path], check=True, cwd=build.CSRC, stderr=subprocess.DEVNULL)
        lines = open(out).read().splitlines()
    total, name, ins, labels = 0, None, [], {}
    for line in lines:
        line = line.split(";")[0].rstrip()
        if m := re.match(r"^(_Z\w+):", line):
            name, ins, labels = m[1], [], {}
        elif m := re.match(r"^(\.LBB\w+):", line):
            labels[m[1]] = len(ins)
        elif line.startswith(".Lfunc_end") and name:
            for mfma, reader, waited, need in too_soon(ins, labels):
                total += 1
                print(f"  {name}: {reader} {waited} of {need} states after {mfma}")
            name = None
        elif name and (m := re.match(r"^\t([a-z]\w+)\s*(.*)$", line)):
            ins.append((m[1], m[2]))
    print(f"{os.path.basename(path)}: {total}", flush=True)
    return total


if __name__ == "__main__":
    sys.exit(sum(scan(p) for p in sys.argv[1:] or [os.path.join(build.CSRC, s) for s in build.SOURCES]) != 0)
