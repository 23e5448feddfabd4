"""CPU: no register is saved or taken back while only some of its lanes are on.

Where a branch by lanes ends, the lanes that did not take it come back by `s_or_b64 exec, exec, ...`.  In the
largest of the attention's kernels ROCm 7.2's compiler has put a copy to the second register file in front of that:
what all lanes needed afterwards was saved for those of the branch only, and an address made of the others' was
anywhere.  What moves between the register files, or to and from scratch, has no place there."""

from __future__ import annotations

import re
import shutil
import subprocess

import pytest

from cugo_amd import build
from tests.conftest import REPO
from tests.test_cpu_matrix_waits import OBJDUMP, functions

SAVES = re.compile(r"v_accvgpr_\w+|scratch_(load|store)_\w+")


def masked_saves(code: list) -> list:
    """(save, place) between the label at which a branch by lanes ends and the instruction that brings the
    other lanes back; code: (operation, operands, address, target address or None)."""
    labels = {x[3] for x in code if x[0] == "s_cbranch_execz" and x[3] is not None}
    found = []
    for i, (op, args, *_) in enumerate(code):
        if op != "s_or_b64" or not args.replace(" ", "").startswith("exec,exec,"):
            continue
        saves = []
        for other, operands, address, _ in reversed(code[max(0, i - 200):i]):
            if other.startswith(("s_cbranch", "s_branch", "s_barrier")) or "saveexec" in other \
                    or (other.startswith("s_") and operands.startswith("exec")):
                break
            if SAVES.fullmatch(other):
                saves.append((f"{other} {operands}", hex(address)))
            if address in labels:
                found += saves
                break
    return found


def test_the_check_finds_a_masked_save():
    branch = ("s_cbranch_execz", "2", 0, 8)
    body, save = ("v_mov_b32_e32", "v3, -1", 4, None), ("v_accvgpr_write_b32", "a2, v7", 8, None)
    back = ("s_or_b64", "exec, exec, s[16:17]", 16, None)
    assert masked_saves([branch, body, save, back])
    assert not masked_saves([branch, body, ("s_or_b64", "exec, exec, s[16:17]", 8, None), save[:2] + (12, None)])
    # of the branch itself, or of one that no jump leaves out
    short = ("s_and_saveexec_b64", "s[16:17], vcc", 8, None)
    assert not masked_saves([branch, body, short, save[:2] + (12, None), back])
    assert not masked_saves([branch, ("v_accvgpr_write_b32", "a2, v7", 4, None), back[:2] + (8, None)])


def test_registers_are_saved_whole(tmp_path):
    if not OBJDUMP.exists() or not shutil.which("objcopy"):
        pytest.skip("no ROCm LLVM tools")
    branches = 0
    for obj in build.code_objects(REPO / "cugo_amd" / "libcugo_hip.so", tmp_path):
        text = subprocess.run([str(OBJDUMP), "-d", str(obj)], check=True, capture_output=True,
                              text=True).stdout
        for name, code in functions(text).items():
            branches += sum(x[0] == "s_cbranch_execz" for x in code)
            assert not masked_saves(code), name
    assert branches > 1000
