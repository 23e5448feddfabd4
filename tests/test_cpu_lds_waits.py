"""CPU: loads that go straight to LDS are issued when what they read is there.

Such a load takes its place in LDS from M0.  Where a scalar instruction writes M0 one wait state has to
lie between; where a vector instruction writes a scalar register that a memory instruction's
address is in, five.  The compiler sees to both for code of its own; it does not look into inline
assembly, where a load that came too early would take an older M0 and write another load's place,
without an error."""

from __future__ import annotations

import re
import shutil
import subprocess

import pytest

from cugo_amd import build
from tests.conftest import REPO
from tests.test_cpu_matrix_waits import OBJDUMP, functions

TO_LDS = re.compile(r"(global|scratch)_load_lds_\w+|buffer_load_\w+")


def to_lds(op: str, args: str) -> bool:
    return bool(TO_LDS.fullmatch(op)) and (not op.startswith("buffer") or args.split()[-1:] == ["lds"])


def scalars(text: str) -> set:
    found = set()
    for a, b in re.findall(r"\bs\[(\d+):(\d+)\]", text):
        found |= set(range(int(a), int(b) + 1))
    return found | {int(a) for a in re.findall(r"\bs(\d+)\b", text)}


def waits(op: str, args: str) -> int:
    return int(args) + 1 if op == "s_nop" else 1


def early_loads(code: list) -> list:
    """(writer, load) of every load to LDS that follows too closely a write of M0, or a vector
    instruction's of its address; code: (operation, operands, ...).  Instructions before a branch's
    target count as in the order of the code, which is one of the paths."""
    found = []
    for i, (op, args, *_) in enumerate(code):
        if not to_lds(op, args):
            continue
        address, waited = scalars(args), 0
        for other, operands, *_ in reversed(code[max(0, i - 8):i]):
            first = operands.split(",")[0].strip()
            late = waited < 1 and first == "m0"
            late = late or (other.startswith("v_") and waited < 5 and scalars(first) & address)
            if late:
                found.append((f"{other} {operands}", f"{op} {args}"))
            waited += waits(other, operands)
            if waited >= 5:
                break
    return found


def test_the_check_finds_an_early_load():
    load = ("global_load_lds_dwordx4", "v3, s[4:5]")
    assert early_loads([("s_mov_b32", "m0, s9"), load])
    assert not early_loads([("s_mov_b32", "m0, s9"), ("s_nop", "0"), load])
    assert not early_loads([("s_mov_b32", "m0, s9"), ("v_mov_b32_e32", "v3, v4"), load])
    assert early_loads([("v_readlane_b32", "s5, v1, 3"), ("s_nop", "3"), load])
    assert not early_loads([("v_readlane_b32", "s5, v1, 3"), ("s_nop", "4"), load])
    assert early_loads([("s_add_u32", "m0, s2, s3"), ("buffer_load_dword", "v1, s[8:11], 0 offen lds")])
    assert not early_loads([("s_mov_b32", "m0, s9"), ("buffer_load_dword", "v0, v1, s[8:11], 0 offen")])


def test_loads_to_lds_wait(tmp_path):
    if not OBJDUMP.exists() or not shutil.which("objcopy"):
        pytest.skip("no ROCm LLVM tools")
    loads = 0
    for obj in build.code_objects(REPO / "cugo_amd" / "libcugo_hip.so", tmp_path):
        text = subprocess.run([str(OBJDUMP), "-d", str(obj)], check=True, capture_output=True,
                              text=True).stdout
        for name, code in functions(text).items():
            loads += sum(to_lds(x[0], x[1]) for x in code)
            early = early_loads(code)
            assert not early, (name, len(early), early[0])
    assert loads > 100
