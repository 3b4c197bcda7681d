"""CPU-only: what the compiler does not check of instructions written out in inline assembly, checked on the code that was built."""
import importlib
import sys
from pathlib import Path

import pytest

REPO = Path(__file__).resolve().parent.parent
CSRC = REPO / "3deecelltracker_amd" / "csrc"


@pytest.fixture(scope="module")
def waits():
    sys.path.insert(0, str(REPO / "scripts"))
    try:
        import check_sgpr_waits
    finally:
        sys.path.pop(0)
    if not (CSRC / "ct_grouped.o").exists():
        importlib.import_module("__graft_entry__").build()
    return check_sgpr_waits


@pytest.mark.parametrize("text,early", [
    ("v_readfirstlane_b32 s4, v4\nv_readfirstlane_b32 s5, v5\ns_mov_b32 m0, s3\ns_nop 0\nglobal_load_lds_dwordx4 v15, s[4:5]", 1),
    ("v_readfirstlane_b32 s5, v5\ns_mov_b32 m0, s3\ns_nop 2\nglobal_load_lds_dwordx4 v15, s[4:5]", 1),
    ("v_readfirstlane_b32 s5, v5\ns_mov_b32 m0, s3\ns_nop 3\nglobal_load_lds_dwordx4 v15, s[4:5]", 0),
    ("v_readfirstlane_b32 s3, v5\ns_mov_b32 m0, s3\ns_nop 0\nglobal_load_lds_dwordx4 v15, s[4:5]", 0),         # m0 waits by itself
    ("v_readfirstlane_b32 s9, v5\ns_add_u32 s4, s9, 1\ns_addc_u32 s5, s8, 0\nglobal_load_dword v1, v2, s[4:5]", 0),
    ("v_add_co_u32_e64 v1, s[4:5], v2, v3\ns_nop 1\nbuffer_load_dword v1, v2, s[4:7], 0 offen", 1),
    ("v_cmp_lt_i32_e64 s[4:5], v1, v2\nv_add_u32 v3, v1, v2\nv_add_u32 v4, v1, v2\nv_add_u32 v5, v1, v2\nv_add_u32 v6, v1, v2\nglobal_store_dword v1, v2, s[4:5]", 1),
])
def test_the_distance_is_counted(waits, text, early):
    found, looked = waits.too_close(text)
    assert sum(found.values()) == early and looked == 1


def test_no_load_takes_an_address_too_early(waits):
    assert waits.check() == {}


def test_m0_is_used_by_the_direct_loads_alone(waits):
    """Their inline assembly writes m0, which cannot be said in a clobber list (the register is reserved): the compiler must keep nothing in it"""
    text = waits.device_disassembly(CSRC / "ct_grouped.o")
    code = [line.split("//")[0].split() for line in text.splitlines()]
    code = [line for line in code if line]
    at = [i for i, line in enumerate(code) if any(a.strip(",") == "m0" for a in line)]
    assert len(at) > 1000
    for i in at:
        assert code[i][:2] == ["s_mov_b32", "m0,"] and code[i + 1][0] == "s_nop" and code[i + 2][0] == "global_load_lds_dwordx4", code[i:i + 3]
    assert sum(line[0].startswith("global_load_lds") for line in code) == len(at)
