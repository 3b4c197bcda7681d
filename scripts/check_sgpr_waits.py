"""Build gate: five wait states between a VALU write of a scalar register (v_readfirstlane, a compare, ...) and a memory instruction that
takes its address from it.  gfx9's memory instructions do not wait for such a write; the compiler puts the distance in for the loads it
emits, and cannot for one written out in inline assembly, which then may go to an address that is half new and half old.

usage: python scripts/check_sgpr_waits.py [object files...]   (default: every csrc/*.o)   exit code 1 on a finding."""
from __future__ import annotations

import re
import subprocess
import sys
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parent))
from check_packed_fp32 import CSRC, KERNEL, GateError, device_disassembly  # noqa: E402

WAIT_STATES = 5
MEMORY = ("global_", "flat_", "scratch_", "buffer_", "tbuffer_")
NO_RESULT = ("s_waitcnt", "s_nop", "s_barrier", "s_cbranch", "s_branch", "s_cmp", "s_bitcmp", "ds_write", "global_store", "flat_store", "scratch_store", "buffer_store")


def _scalars(operand: str) -> set[int]:
    """The scalar registers of one operand"""
    m = re.match(r"s\[(\d+):(\d+)\]|s(\d+)$", (operand.split() or [""])[0])
    if not m:
        return set()
    return set(range(int(m[1]), int(m[2]) + 1)) if m[1] else {int(m[3])}


def too_close(text: str) -> tuple[dict[str, int], int]:
    """Disassembly (or assembly) -> ({kernel: memory instructions that read a scalar register too early}, memory instructions looked at)"""
    found: dict[str, int] = {}
    kernel, looked, before = "?", 0, []                    # before: (is VALU, scalar registers written, wait states it stands for)
    for line in text.splitlines():
        m = KERNEL.match(line)
        if m:
            kernel, before = m.group(1), []
            continue
        code = re.split(r"//|;", line)[0].strip()
        if not code or code.endswith(":") or code.startswith("."):
            continue
        op, _, rest = code.partition(" ")
        args = [a.strip() for a in rest.split(",")]
        if op.startswith(MEMORY):
            looked += 1
            need, distance = set().union(*(_scalars(a) for a in args)), 0
            for valu, written, states in reversed(before):
                if distance >= WAIT_STATES or not need:
                    break
                if valu and written & need:
                    found[kernel] = found.get(kernel, 0) + 1
                    break
                need -= written                            # (written since by a scalar instruction, which the load does wait for)
                distance += states
        written = set() if op.startswith(NO_RESULT) else _scalars(args[0]) | (_scalars(args[1]) if op.startswith("v_") and "_co_" in op and len(args) > 1 else set())
        before = before[-WAIT_STATES:] + [(op.startswith("v_"), written, int(args[0], 0) + 1 if op == "s_nop" else 1)]
    return found, looked


def check(objs=None) -> dict[str, dict[str, int]]:
    bad, looked = {}, 0
    for o in [Path(o) for o in objs] if objs else sorted(CSRC.glob("*.o")):
        text = device_disassembly(o)
        if text is None:
            continue
        found, n = too_close(text)
        looked += n
        if found:
            bad[o.name] = found
    if not looked:
        raise GateError("no device code could be inspected in any object: the gate did not run")
    return bad


if __name__ == "__main__":
    try:
        bad = check(sys.argv[1:])
    except (GateError, subprocess.CalledProcessError) as e:
        print(f"[sgpr-waits] gate error: {e}", file=sys.stderr)
        sys.exit(2)
    for name, f in bad.items():
        for k, c in f.items():
            print(f"[sgpr-waits] {name}: {c} memory instruction(s) in {k}", file=sys.stderr)
    if bad:
        sys.exit(1)
    print("[sgpr-waits] every address in a scalar register is there before the load")
