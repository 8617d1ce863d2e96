"""CPU suite: no memory instruction of the built library reads a scalar register sooner than 5 wait states behind the vector instruction that wrote it
(tools/sgpr_waits.py).  hipcc keeps that distance for its own instructions; for `global_load_lds` in inline assembly nobody does but the text of the assembly."""
import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "tools"))

LISTING = """
0000000000001000 <k>:
\tv_readlane_b32 s7, v251, 5                                 // 000000001000: D2890007
\ts_mov_b32 s3, m0                                           // 000000001008: BE83007C
\ts_mov_b32 m0, s2
\ts_nop %d
\tglobal_load_lds_dwordx4 v242, s[6:7]
\tv_cmp_lt_i32_e32 vcc, 0, v1
\tglobal_load_dwordx4 v[0:3], v4, s[10:11]
"""


def test_the_scan_counts_states():
    from sgpr_waits import scan
    assert [(f, n) for f, n, _, _ in scan(LISTING % 0)] == [("k", 3)] and [n for _, n, _, _ in scan(LISTING % 1)] == [4] and not scan(LISTING % 2)
    assert not scan((LISTING % 0).replace("v_readlane_b32 s7", "v_readlane_b32 s8")) and scan((LISTING % 0).replace("v_readlane_b32 s7, v251, 5", "v_readfirstlane_b32 s6, v251"))


def test_no_memory_instruction_reads_a_scalar_register_too_early():
    from sgpr_waits import LIB, OBJDUMP, library
    if not os.path.exists(LIB):
        pytest.skip("libdynam3d_hip.so is not built")
    if not os.path.exists(OBJDUMP):
        pytest.skip("no llvm-objdump")
    seen, found = library()
    assert seen > 20000, seen
    assert not found, found[:8]
