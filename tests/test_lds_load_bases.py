"""The wait states between a vector instruction that writes a scalar register and a load to LDS that takes its base from
there, in the machine code of the built library (the loads stand in inline assembly, where the compiler inserts none)."""
import re
import shutil
import subprocess

import pytest

from dsv41_amd import _lib
from test_lds_loads import OBJDUMP, instructions


def registers(op):
    """The scalar registers that a load to LDS reads as its base."""
    m = re.search(r"\bs\[(\d+):(\d+)\]", op)
    return set(range(int(m.group(1)), int(m.group(2)) + 1)) if m else set()


def written(op):
    """The scalar registers that a vector instruction writes."""
    if not op.startswith("v_"):
        return set()
    dst = op.split(None, 1)[1].split(",")[0].strip() if " " in op else ""
    one, two = re.fullmatch(r"s(\d+)", dst), re.fullmatch(r"s\[(\d+):(\d+)\]", dst)
    return {int(one.group(1))} if one else set(range(int(two.group(1)), int(two.group(2)) + 1)) if two else set()


def wait_states(ins, i, regs):
    """Wait states between the last vector write of regs and instruction i, 9 where there is none near."""
    n = 0
    for prev in reversed(ins[max(0, i - 9):i]):
        if written(prev) & regs:
            return n
        nop = re.match(r"s_nop (\d+)", prev)
        n += int(nop.group(1)) + 1 if nop else 1
    return 9


def test_the_reader_sees_the_hazard():
    ins = ["v_readlane_b32 s63, v1, 3", "v_readlane_b32 s62, v2, 3", "s_mov_b32 m0, s4", "s_nop 0", "global_load_lds_dwordx4 v3, s[62:63]"]
    assert wait_states(ins, 4, registers(ins[4])) == 2
    assert wait_states(ins[:2] + ["s_nop 3"] + ins[2:], 5, registers(ins[4])) == 6
    assert wait_states(["v_cmp_lt_i32_e64 s[62:63], v1, v2", ins[4]], 1, {62, 63}) == 0


def test_bases_of_loads_to_lds_have_settled(tmp_path):
    if not OBJDUMP.exists():
        pytest.skip("no llvm-objdump")
    shutil.copy(_lib.LIB_PATH, tmp_path / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", "lib.so"], check=True, capture_output=True, cwd=tmp_path)
    loads = 0
    for obj in sorted(tmp_path.glob("lib.so.*gfx950")):
        for ins in instructions(obj):
            for i, op in enumerate(ins):
                if re.match(r"global_load\w*_lds", op) and registers(op):
                    loads += 1
                    assert wait_states(ins, i, registers(op)) >= 5, (obj.name, ins[max(0, i - 6):i + 1])
    assert loads > 100
