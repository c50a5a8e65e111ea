"""The large-tile kernels issue their matrix instructions from assembly, where the compiler adds no
wait states.  What it must not do around them is checked in the built library: write an operand of
a matrix instruction with a vector instruction less than two wait states ahead, or read an
accumulator before the pipe has settled (18 wait states cover every result of these shapes).  Reads
the code built here; runs without a GPU."""
import os
import re
import shutil
import subprocess

import pytest

from rtatblas_amd import native

OBJDUMP = shutil.which("llvm-objdump") or "/opt/rocm/llvm/bin/llvm-objdump"


def _regs(token):
    m = re.match(r"([va])\[(\d+):(\d+)\]$", token)
    if m:
        return {(m.group(1), i) for i in range(int(m.group(2)), int(m.group(3)) + 1)}
    m = re.match(r"([va])(\d+)$", token)
    return {(m.group(1), int(m.group(2)))} if m else set()


def _operands(line):
    return [o.strip() for o in line.split(None, 1)[1].split(",")]


def _functions(text):
    for part in re.split(r"\n(?=[0-9a-f]{16} <)", text):
        m = re.match(r"[0-9a-f]{16} <(\S+)>:", part)
        if m:
            lines = [l.split("//")[0].strip() for l in part.split("\n")[1:]]
            yield m.group(1), [l for l in lines if l]


def _wait_states(line):
    return int(line.split()[1], 0) + 1 if line.startswith("s_nop") else 1


def test_no_hazard_around_matrix_instructions(tmp_path):
    if not os.path.exists(OBJDUMP):
        pytest.skip("no llvm-objdump")
    lib = shutil.copy(native.LIB_PATH, tmp_path / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", str(lib)], cwd=tmp_path, check=True, capture_output=True)
    objects = [f for f in os.listdir(tmp_path) if "gfx950" in f]
    assert objects
    seen = 0
    for name in objects:
        text = subprocess.run([OBJDUMP, "-d", str(tmp_path / name)], check=True, capture_output=True,
                              text=True).stdout
        for function, lines in _functions(text):
            if "gemm16_dma_kernel" not in function:
                continue
            for i, line in enumerate(lines):
                if line.startswith("v_mfma"):
                    seen += 1
                    use = set().union(*(_regs(o) for o in _operands(line)[1:4]))
                    states = 0
                    for back in reversed(lines[max(0, i - 3):i]):
                        if back.startswith("v_") and not back.startswith(("v_mfma", "v_cmp", "v_readfirstlane")):
                            assert states >= 2 or not _regs(_operands(back)[0]) & use, (function, back, line)
                        states += _wait_states(back)
                elif line.startswith("v_accvgpr_read"):
                    read, states = _regs(_operands(line)[1]), 0
                    for back in reversed(lines[max(0, i - 40):i]):
                        if states >= 18:
                            break
                        assert not (back.startswith("v_mfma") and _regs(_operands(back)[0]) & read), (function, back, line)
                        states += _wait_states(back)
    assert seen >= 24 * 16      # three shapes, four op combinations, two types
