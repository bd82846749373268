"""Waits at the barriers of the kernels whose waves read LDS slots that other waves refill
by direct loads: a barrier hands a slot over, so no wave may pass it with an LDS read of
that slot in flight (no GPU: the built kernels' own code is read)."""
from __future__ import annotations

import os
import re
import subprocess
from pathlib import Path

import pytest

from dflash_mlx import _build
from tests.test_code_objects import _gfx950_objects

OBJDUMP = Path(os.environ.get("ROCM_PATH", "/opt/rocm")) / "llvm" / "bin" / "llvm-objdump"

INSTRUCTION = re.compile(r"^\s+(\S+)(.*?)//\s*([0-9A-F]{12}):")
TARGET = re.compile(r"<[^>]*\+0x([0-9a-f]+)>\s*$|<[^>+]+>\s*$")


def _kernels(tmp, names):
    """(name, [(address, mnemonic, operands, branch target or None)]) of the library's kernels
    whose name holds one of `names`."""
    for n, elf in enumerate(_gfx950_objects(_build.LIB_PATH.read_bytes())):
        if not any(name.encode() in elf for name in names):
            continue
        path = tmp / f"{n}.co"
        path.write_bytes(elf)
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", path], check=True, capture_output=True, text=True).stdout
        name, start, code = None, 0, []
        for line in text.splitlines() + ["0000000000000000 <>:"]:
            if head := re.match(r"^([0-9a-f]{16}) <(.*)>:$", line):
                if code and any(s in name for s in names):
                    yield name, code
                name, start, code = head[2], int(head[1], 16), []
            elif ins := INSTRUCTION.match(line):
                target = None
                if ins[1].startswith(("s_branch", "s_cbranch")):
                    to = TARGET.search(line)
                    target = start + int(to[1] or "0", 16)
                code.append((int(ins[3], 16), ins[1], ins[2], target))


def _reads_in_flight(code):
    """The most LDS reads (and LDS atomics) that may be in flight before each barrier, over all
    paths: [(address, count)]."""
    at = {ins[0]: i for i, ins in enumerate(code)}
    most = [-1] * len(code)
    todo, barriers = [(0, 0)], {}
    while todo:
        i, pending = todo.pop()
        while i < len(code) and pending > most[i]:
            most[i] = pending
            address, op, operands, target = code[i]
            if op.startswith("ds_"):
                pending = min(pending + 1, 16)
            elif op == "s_waitcnt":
                if wait := re.search(r"lgkmcnt\((\d+)\)", operands):
                    pending = min(pending, int(wait[1]))
            elif op == "s_barrier":
                barriers[address] = pending
            if target is not None:
                todo.append((at[target], pending))
            if op in ("s_branch", "s_endpgm") or op.startswith("s_setpc"):
                break
            i += 1
    return sorted(barriers.items())


@pytest.fixture(scope="module")
def library():
    if not _build.LIB_PATH.exists() or not OBJDUMP.exists():
        pytest.skip("library or llvm-objdump not there")


def _check(tmp_path, name, count):
    kernels = 0
    for kernel, code in _kernels(tmp_path, [name]):
        barriers = _reads_in_flight(code)
        assert len(barriers) >= 3, kernel  # of loaders and of compute waves
        assert all(n == 0 for _, n in barriers), (kernel, [(hex(a), n) for a, n in barriers])
        kernels += 1
    assert kernels >= count


def test_the_reading_of_waits():
    """Reads are counted over branches, a wait lowers them, a second path raises them again."""
    code = [(0, "ds_read_b128", "", None), (8, "ds_read_b128", "", None), (16, "s_waitcnt", " lgkmcnt(1)", None),
            (20, "s_barrier", "", None), (24, "s_cbranch_scc1", "", 0), (28, "s_waitcnt", " vmcnt(0) lgkmcnt(0)", None),
            (32, "s_barrier", "", None), (36, "s_endpgm", "", None)]
    assert _reads_in_flight(code) == [(20, 1), (32, 0)]


def test_int8_prompt_products(library, tmp_path):
    _check(tmp_path, "prompt_i8_kernel", 12)


def test_bf16_prompt_products(library, tmp_path):
    _check(tmp_path, "prefill_gemm_wide_kernel", 2)
