"""Scalar registers that a vector instruction writes and a memory instruction reads too soon, in every gfx950 kernel of libdynam3d_hip.so.

    python tools/sgpr_waits.py

A vector memory instruction that reads a scalar register needs 5 wait states behind a VECTOR instruction that wrote it (v_readlane, v_readfirstlane, v_cmp; the
CDNA instruction set's table of software waits).  hipcc inserts them for its own instructions, but does not look into inline assembly: a `global_load_lds` written there
gets whatever stands in front of it -- once its base is a spilled scalar register, a v_readlane.  Too few states read the old value: a wrong address.
Reads the listing of the code built here (llvm-objdump), straight through each function."""
import os
import re
import subprocess
import sys
import tempfile

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from kernel_resources import LIB, _code_objects, demangle_hint

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
STATES = 5
_REG = re.compile(r"\bs\[(\d+):(\d+)\]|\bs(\d+)\b|\bvcc\b")


def _regs(text):
    out = set()
    for a, b, c in _REG.findall(text):
        out |= set(range(int(a), int(b) + 1)) if a else {int(c)} if c else {"vcc"}
    return out


def _written(op, args):
    """Scalar registers that a vector instruction writes."""
    a = args.split(",")
    if op.startswith(("v_readlane", "v_readfirstlane", "v_cmp")):
        return _regs(a[0])
    if "_co_" in op or "div_scale" in op:
        return _regs(a[1]) if len(a) > 1 else set()
    return set()


def scan(listing):
    """[(function, wait states, writer, reader)] of an llvm-objdump listing."""
    found, fn, past = [], None, []
    for line in listing.splitlines():
        m = re.match(r"^[0-9a-f]+ <(.+)>:$", line)
        if m:
            fn, past = m.group(1), []
            continue
        text = line.split("//")[0].strip()
        if not text or not line[:1].isspace():
            continue
        op, _, args = text.partition(" ")
        if op.startswith(("global_", "buffer_", "flat_", "scratch_")):
            need, states = _regs(args), 0
            for n, wrote, what in reversed(past):
                if wrote & need:
                    found.append((fn, states, what, text))
                    break
                states += n
                if states >= STATES:
                    break
        past.append((int(args, 0) + 1 if op == "s_nop" else 1, _written(op, args) if op.startswith("v_") else set(), text))
        past = past[-STATES:]
    return found


def library(lib=LIB):
    """The same over every code object of the library -> (kernels' memory instructions seen, findings)."""
    seen, found = 0, []
    for elf in _code_objects(open(lib, "rb").read()):
        with tempfile.NamedTemporaryFile(suffix=".co") as f:
            f.write(elf)
            f.flush()
            text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", f.name], capture_output=True, text=True, check=True).stdout
        seen += len(re.findall(r"^\s+(?:global|buffer|flat|scratch)_", text, re.M))
        found += scan(text)
    return seen, found


if __name__ == "__main__":
    seen, found = library()
    for fn, states, writer, reader in found:
        print(f"{demangle_hint(fn):40s} {states} states between  {writer}  and  {reader}")
    print(f"{seen} memory instructions, {len(found)} too early")
    sys.exit(1 if found else 0)
