"""The built kernels' matrix instructions: what a vector instruction writes, a matrix
instruction reads two wait states later at the earliest.  The compiler keeps that for its
own instructions, but not for those inside inline assembly, and a kernel that does not
keep it multiplies what its registers held before."""
import os
import re
import subprocess

import pytest

LIB = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gemma4metal_amd", "libturboquant_hip.so")
OBJDUMP = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin", "llvm-objdump")
WAIT_STATES = 2
REG = re.compile(r"\b([av])(?:\[(\d+):(\d+)\]|(\d+)\b)")


def registers(operand):
    out = set()
    for kind, first, last, one in REG.findall(operand):
        out |= {(kind, i) for i in range(int(first or one), int(last or one) + 1)}
    return out


def too_early(lines):
    """Matrix instructions (kernel, line) of a disassembly that read a register too early."""
    found, kernel, last = [], "", []   # last: (written, wait states since it issued)
    for line in lines:
        if line.endswith(">:\n"):
            kernel, last = line.split("<")[-1][:-3], []
            continue
        if not line.startswith("\t"):
            continue
        op, _, rest = line.split("//")[0].strip().partition(" ")
        if "mfma" in op:
            reads = registers(rest.split(",", 1)[1])
            if any(since < WAIT_STATES and written & reads for written, since in last):
                found.append((kernel, line.strip()))
        states = int(rest, 0) + 1 if op == "s_nop" else 1
        last = [(w, s + states) for w, s in last if s + states < WAIT_STATES]
        if op.startswith("v_") and not op.startswith("v_cmp") and "mfma" not in op:
            both = "swap" in op or op.startswith("v_readlane")
            last.append((registers(rest if both else rest.split(",")[0]), 0))
    return found


def test_the_check_itself():
    text = ("0 <k>:\n", "\tv_add_f32_e32 v4, v1, v2\n", "\ts_nop 0\n", "\tv_mfma_f32_16x16x32_f16 a[0:3], v[4:7], v[8:11], a[0:3]\n")
    assert len(too_early(text)) == 1
    assert not too_early(text[:2] + ("\ts_nop 1\n",) + text[3:])
    assert not too_early((text[0], text[1].replace("v4", "v12")) + text[2:])


def test_operands_are_written_before_they_are_read(tmp_path):
    if not os.path.exists(OBJDUMP):
        pytest.skip("no llvm-objdump")
    os.symlink(LIB, tmp_path / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", "lib.so"], cwd=tmp_path, check=True, capture_output=True)
    objects = [f for f in os.listdir(tmp_path) if f.endswith("gfx950")]
    assert len(objects) >= 10
    found, products = [], 0
    for f in objects:
        text = subprocess.run([OBJDUMP, "-d", f], cwd=tmp_path, check=True, capture_output=True, text=True).stdout
        products += text.count("v_mfma_")
        found += too_early(text.splitlines(True))
    assert products > 1000
    assert not found, f"{len(found)}, the first {found[:3]}"
