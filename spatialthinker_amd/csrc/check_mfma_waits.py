#!/usr/bin/env python3
"""Checks the built code of kernels whose MFMAs are inline assembly: no other instruction may touch an MFMA's result within the wait states that the
result needs (the compiler inserts these for its own MFMAs only).   check_mfma_waits.py OBJECT...   exits 1 and names what it found.

Every path of that many wait states behind each MFMA is followed, through branches on both sides.  An instruction counts one state, s_nop N counts N + 1, and
another MFMA the passes for which the earlier one holds the matrix pipe.  A later MFMA may read or overwrite the result: the hardware orders
these.  Without an llvm-objdump (ROCm's own, or one on the PATH) nothing is checked and a warning says so."""
import os
import re
import shutil
import subprocess
import sys
import tempfile

LLVM = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin")
STATES, PASSES = 8, 4                        # 16x16x32 bf16: result -> VALU / memory instruction; the next MFMA waits 4 for the matrix pipe


def objdump():
    """The llvm-objdump to use, or None."""
    return shutil.which(os.path.join(LLVM, "llvm-objdump")) or shutil.which("llvm-objdump")


def registers(text):
    """The vector registers that an instruction's operands name, as ("a" | "v", number)."""
    found = set()
    for kind, one, lo, hi in re.findall(r"\b([av])(?:(\d+)\b|\[(\d+):(\d+)\])", text):
        found |= {(kind, int(one))} if one else {(kind, n) for n in range(int(lo), int(hi) + 1)}
    return found


def functions(obj):
    """{name: [(address, instruction, operands, branch target or None)]} of the device code in an object."""
    tool = objdump()
    with tempfile.TemporaryDirectory() as d:
        copy = os.path.join(d, "o.o")
        with open(obj, "rb") as f, open(copy, "wb") as g:
            g.write(f.read())
        subprocess.run([tool, "--offloading", copy], check=True, stdout=subprocess.DEVNULL)
        out, name = {}, None
        for code in sorted(f for f in os.listdir(d) if "amdgcn" in f):
            text = subprocess.run([tool, "-d", os.path.join(d, code)], check=True, stdout=subprocess.PIPE, text=True).stdout
            for line in text.splitlines():
                m = re.match(r"[0-9a-f]+ <(.+)>:$", line)
                if m:
                    name = m.group(1)
                    out[name] = []
                    continue
                m = re.match(r"\s+(\S+)(.*?)\s*// ([0-9A-F]+):(.*)$", line)
                if m and name:
                    target = None
                    if m.group(1).startswith(("s_cbranch", "s_branch")):
                        t = re.search(r"<.*?\+0x([0-9a-f]+)>", m.group(4))
                        target = out[name][0][0] + int(t.group(1), 16) if t and out[name] else None
                    out[name].append((int(m.group(3), 16), m.group(1), m.group(2), target))
        return out


def early(code):
    """The places where an MFMA's result is touched too early."""
    at = {a: i for i, (a, *_) in enumerate(code)}
    bad = set()
    for i, (addr, op, args, _) in enumerate(code):
        if not op.startswith("v_mfma"):
            continue
        result = registers(args.split(",")[0])
        todo, seen = [(i + 1, STATES)], {}
        while todo:
            j, left = todo.pop()
            while j < len(code) and left > 0 and seen.get(j, 0) < left:
                seen[j] = left
                a, o, r, target = code[j]
                if not o.startswith("v_mfma") and registers(r) & result:
                    bad.add("%x: %s%s touches the result of the MFMA at %x" % (a, o, r, addr))
                left -= int(r.split()[0], 0) + 1 if o == "s_nop" else PASSES if o.startswith("v_mfma") else 1
                if target is not None and target in at:
                    todo.append((at[target], left))
                if o in ("s_branch", "s_endpgm"):
                    break
                j += 1
    return sorted(bad)


def main(objects):
    if objdump() is None:
        print("check_mfma_waits.py: warning: no llvm-objdump in %s or on the PATH: wait states not checked" % LLVM, file=sys.stderr)
        return 0
    failed = 0
    for obj in objects:
        for name, code in functions(obj).items():
            bad = early(code)
            failed += bool(bad)
            for b in bad[:4]:
                print("%s: %s: %s" % (os.path.basename(obj), name, b))
    return 1 if failed else 0


if __name__ == "__main__":
    sys.exit(main(sys.argv[1:]))
