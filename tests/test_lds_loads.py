"""The wait state between a scalar write of m0 and the load to LDS that takes its address from there, in the machine code
of the built library (the kernels issue these loads from inline assembly, which the compiler does not look into)."""
import os
import re
import shutil
import subprocess
from pathlib import Path

import pytest

from dsv41_amd import _lib
from dsv41_amd.build import CSRC, HIPCC

OBJDUMP = Path(os.path.realpath(HIPCC)).parent.parent / "llvm" / "bin" / "llvm-objdump"


def instructions(obj):
    """Lists of instructions, one a function."""
    out = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", "--no-leading-addr", obj], check=True, capture_output=True, text=True)
    code = []
    for line in out.stdout.split("\n"):
        if re.match(r"^(?:[0-9a-f]+ )?<.+>:$", line.strip()):
            code.append([])
        elif code and line.split("//")[0].strip():
            code[-1].append(line.split("//")[0].strip())
    return code


def wait_states(ins, i):
    """Wait states between the last write of m0 and instruction i."""
    n = 0
    for prev in reversed(ins[:i]):
        if re.match(r"s_\w+ m0\b", prev):
            return n
        nop = re.match(r"s_nop (\d+)", prev)
        n += int(nop.group(1)) + 1 if nop else 1
    raise AssertionError("a load to LDS without a write of m0")


def test_loads_to_lds_stand_a_wait_state_behind_m0(tmp_path):
    if not OBJDUMP.exists():
        pytest.skip("no llvm-objdump")
    shutil.copy(_lib.LIB_PATH, tmp_path / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", "lib.so"], check=True, capture_output=True, cwd=tmp_path)
    loads = 0
    for obj in sorted(tmp_path.glob("lib.so.*gfx950")):
        for ins in instructions(obj):
            for i, op in enumerate(ins):
                if re.match(r"(global|buffer|scratch)_load\w*_lds|buffer_load.* lds\b", op):
                    loads += 1
                    assert wait_states(ins, i) >= 1, (obj.name, ins[max(0, i - 2):i + 1])
    assert loads > 500


def test_loads_to_lds_are_written_once():
    """One helper holds the instruction pair; no other source spells it out."""
    for p in sorted(CSRC.iterdir()):
        if p.name != "common.h":
            assert "load_lds" not in p.read_text() and "s_mov_b32 m0" not in p.read_text(), p.name
