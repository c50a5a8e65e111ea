"""The wait states around the matrix instructions that are issued from assembly, along every path of
the built code: over the back edges of loops and over branches too, where a compiler puts the
copies that a loop carries.  A vector instruction that writes an operand is two wait states ahead of
the matrix instruction, and an accumulator is read no sooner than 18 after the last one that wrote
it.  Reads the code built here; runs without a GPU."""
import os
import re
import shutil
import subprocess

import pytest

from rtatblas_amd import native

OBJDUMP = shutil.which("llvm-objdump") or "/opt/rocm/llvm/bin/llvm-objdump"
# Matrix instructions of each instantiation: blocks of a wave tile, two K-steps, the main loop and
# the last panels.  Tile sides by depth of the ring of panels.
COUNTS = {(256, 2): 64 * 4, (128, 2): 16 * 4, (128, 3): 16 * 4, (64, 2): 4 * 4, (64, 3): 4 * 4}


def _regs(token):
    m = re.match(r"([va])\[(\d+):(\d+)\]$", token)
    if m:
        return {(m.group(1), i) for i in range(int(m.group(2)), int(m.group(3)) + 1)}
    m = re.match(r"([va])(\d+)$", token)
    return {(m.group(1), int(m.group(2)))} if m else set()


def _operands(text):
    parts = text.split(None, 1)
    return [o.strip() for o in parts[1].split(",")] if len(parts) > 1 else []


class Function:
    """Instructions in order and, for each, those that may run right before it."""

    def __init__(self, lines):
        self.code, address = [], []
        for line in lines:
            m = re.match(r"\s*(\S.*?)\s*// ([0-9A-F]{8,16}):", line)
            if m:
                self.code.append(m.group(1))
                address.append(int(m.group(2), 16))
        at = {a: i for i, a in enumerate(address)}
        self.before = [[] for _ in self.code]
        for i, text in enumerate(self.code):
            name = text.split()[0]
            if name.startswith(("s_branch", "s_cbranch")):
                offset = int(text.split()[1]) & 0xffff
                offset -= 0x10000 if offset >= 0x8000 else 0
                self.before[at[address[i] + 4 + 4 * offset]].append(i)
            assert not name.startswith(("s_setpc", "s_swappc", "s_call")), text
            if name not in ("s_branch", "s_endpgm") and i + 1 < len(self.code):
                self.before[i + 1].append(i)

    def states(self, i):
        text = self.code[i]
        return int(text.split()[1], 0) + 1 if text.startswith("s_nop") else 1

    def back_from(self, start, limit):
        """Instructions with fewer than `limit` wait states between them and `start`, on any path."""
        least = {}
        todo = [(p, 0) for p in self.before[start]]
        while todo:
            i, between = todo.pop()
            if between >= limit or least.get(i, limit) <= between:
                continue
            least[i] = between
            todo += [(p, between + self.states(i)) for p in self.before[i]]
        return least


def check(function, name):
    """The number of matrix instructions; raises where a wait state is missing."""
    seen = 0
    for i, text in enumerate(function.code):
        if text.startswith("v_mfma"):
            seen += 1
            use = set().union(*(_regs(o) for o in _operands(text)[1:4]))
            for b in function.back_from(i, 2):
                back = function.code[b]
                if back.startswith("v_") and not back.startswith(("v_mfma", "v_cmp", "v_readfirstlane")):
                    assert not _regs(_operands(back)[0]) & use, (name, back, text)
        elif text.startswith("v_accvgpr_read"):
            read = _regs(_operands(text)[1])
            for b in function.back_from(i, 18):
                back = function.code[b]
                assert not (back.startswith("v_mfma") and _regs(_operands(back)[0]) & read), (name, back, text)
    return seen


def _listing(*lines):
    """A function of four-byte instructions."""
    return Function(["\t%s // %012X: 00000000" % (l, 4 * i) for i, l in enumerate(lines)])


def test_the_walk_follows_branches():
    copy, mfma = "v_mov_b32_e32 v8, v9", "v_mfma_f32_16x16x32_f16 a[0:3], v[8:11], v[4:7], a[0:3]"
    read = "v_accvgpr_read_b32 v1, a2"
    assert check(_listing(copy, "s_nop 1", mfma, "s_nop 15", "s_nop 1", read, "s_endpgm"), "") == 1
    for bad in ([copy, "s_nop 0", mfma, "s_endpgm"], [mfma, "s_nop 15", read, "s_endpgm"],
                # the copy is at the loop's end: only the back edge (four instructions up) leads to the matrix instruction
                ["s_nop 1", mfma, "s_nop 5", copy, "s_cbranch_scc1 65532", "s_endpgm"],
                # the read is jumped to
                [mfma, "s_branch 1", "s_endpgm", read, "s_endpgm"]):
        with pytest.raises(AssertionError):
            check(_listing(*bad), "")
    assert check(_listing("s_nop 1", mfma, "s_nop 5", copy, "s_nop 1", "s_cbranch_scc1 65531", "s_endpgm"), "") == 1


def test_no_hazard_on_any_path(tmp_path):
    if not os.path.exists(OBJDUMP):
        pytest.skip("no llvm-objdump")
    lib = shutil.copy(native.LIB_PATH, tmp_path / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", str(lib)], cwd=tmp_path, check=True, capture_output=True)
    found = {}
    for name in sorted(f for f in os.listdir(tmp_path) if "gfx950" in f):
        text = subprocess.run([OBJDUMP, "-d", str(tmp_path / name)], check=True, capture_output=True, text=True).stdout
        for part in re.split(r"\n(?=[0-9a-f]{16} <)", text):
            m = re.match(r"[0-9a-f]{16} <(\S+)>:", part)
            if m and "gemm16_dma_kernel" in m.group(1):
                found[m.group(1)] = check(Function(part.split("\n")[1:]), m.group(1))
    seen = {}
    for name, count in found.items():
        m = re.search(r"gemm16_dma_kernelI(DF16b|DF16_)NS0_7Shape16ILi(\d+)ELi\2ELi2ELi2ELi\d+ELi(\d)EEELb([01])ELb([01])E", name)
        assert m, name
        seen[m.group(1), int(m.group(2)), int(m.group(3)), m.group(4), m.group(5)] = count
    want = {(t, *shape, a, b): n for t in ("DF16b", "DF16_") for shape, n in COUNTS.items() for a in "01" for b in "01"}
    assert seen == want
