"""The distances that CDNA code has to keep itself, read from the built library's own
assembly: the compiler keeps them between the instructions it knows, and not from or to
those that inline asm writes.

  * a matrix instruction reads a register two wait states after a vector instruction wrote
    it, at the earliest
  * a memory instruction reads a scalar register five wait states after a vector
    instruction wrote it, at the earliest
An instruction is one wait state, s_nop n is n + 1."""
from __future__ import annotations

import os
import re
import shutil
import subprocess

import pytest

from optimized_rocwmma_samples_amd import build

OBJDUMP = os.path.join(build.ROCM, "lib", "llvm", "bin", "llvm-objdump")
NO_RESULT = ("v_cmp", "v_readlane", "v_readfirstlane", "v_nop")  # no vector register written


def registers(operand, kind):
    """Numbers of the registers of one kind ('v' or 's') in an operand."""
    m = re.fullmatch(r"[-|]*" + kind + r"(?:(\d+)|\[(\d+):(\d+)\])\|?", operand)
    if not m:
        return set()
    return {int(m[1])} if m[1] else set(range(int(m[2]), int(m[3]) + 1))


def before(recent, states):
    """The instructions that lie fewer than `states` wait states back, with how many."""
    at = 0
    for op, args, cost in reversed(recent):
        if at >= states:
            return
        yield op, args, at
        at += cost


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """{kernel: [(instruction, operands, wait states)]} of the built library."""
    if not (os.path.exists(OBJDUMP) and build.LIB_PATH.exists()):
        pytest.skip("needs the built library and ROCm's llvm-objdump")
    tmp = tmp_path_factory.mktemp("code")
    shutil.copy(build.LIB_PATH, tmp / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", "lib.so"], cwd=tmp, check=True, capture_output=True)
    out = {}
    for f in sorted(tmp.glob(f"lib.so.*{build.ARCH}")):
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", str(f)], check=True,
                              capture_output=True, text=True).stdout
        for line in text.splitlines():
            m = re.match(r"[0-9a-f]+ <(.*)>:", line)
            if m:
                code = out.setdefault(m[1], [])
                continue
            parts = line.split("//")[0].split(None, 1)
            if not parts or line[0] not in "\t ":
                continue
            args = re.split(r",\s*|\s+", parts[1].strip()) if len(parts) > 1 else []
            code.append((parts[0], args, int(args[0], 0) + 1 if parts[0] == "s_nop" else 1))
    assert sum(op.startswith("v_mfma") for code in out.values() for op, _, _ in code) > 1000
    return out


def test_matrix_operands(kernels):
    late = []
    for name, code in kernels.items():
        for i, (op, args, _) in enumerate(code):
            if not op.startswith("v_mfma"):
                continue
            reads = set().union(*(registers(a, "v") for a in args[1:4]))
            for o, a, at in before(code[max(0, i - 2):i], 2):
                if o.startswith("v_") and not o.startswith(("v_mfma", *NO_RESULT)) \
                        and registers(a[0], "v") & reads:
                    late.append((name, o, a, at, op, args))
    assert not late, late


def test_scalar_registers_of_memory_instructions(kernels):
    late = []
    for name, code in kernels.items():
        for i, (op, args, _) in enumerate(code):
            if not op.startswith(("buffer_", "global_", "flat_", "scratch_")):
                continue
            reads = set().union(*(registers(a, "s") for a in args))
            for o, a, at in before(code[max(0, i - 5):i], 5):
                if o.startswith("v_") and registers(a[0], "s") & reads:
                    late.append((name, o, a, at, op, args))
    assert not late, late


def test_loads_in_asm_keep_it_themselves(kernels):
    # the loads into LDS of prompt attention: nothing but the asm block's own instructions
    # lies in those five wait states, whatever stands in front of the block
    found = 0
    for name, code in kernels.items():
        if "16attention_kernel" not in name:
            continue
        for i, (op, args, _) in enumerate(code):
            if not (op.startswith("buffer_load") and args[-1] == "lds"):
                continue
            found += 1
            for o, a, at in before(code[max(0, i - 5):i], 5):
                own = o == "s_nop" or a[0] == "m0" or a[-1] == "lds"
                assert own, (name, o, a, at)
    assert found >= 16
