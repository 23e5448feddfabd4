"""CPU: no instruction of the built library reads a matrix instruction's result too early.

The hardware does not wait by itself where vector instructions read what v_mfma writes: eight wait
states have to lie between for 16 x 16 x 32 of 16-bit types, ten for 16 x 16 x 4 float32 (what the
compiler inserts in straight code).  ROCm 7.2's compiler has left two where a
conditional branch came right behind the products: a wrong last score and no error."""

from __future__ import annotations

import re
import shutil
import subprocess

import pytest

from cugo_amd import build
from tests.conftest import REPO

OBJDUMP = build.LLVM_BIN / "llvm-objdump"
WAITS = {"v_mfma_f32_16x16x32_bf16": 8, "v_mfma_f32_16x16x32_f16": 8, "v_mfma_f32_16x16x4_f32": 10}
LINE = re.compile(r"^\t(\S+)\s*(.*?)\s*// ([0-9A-F]+):.*?(?:<\S+\+0x([0-9a-f]+)>)?$")


def registers(text: str) -> set:
    found = set()
    for kind, a, b in re.findall(r"\b([av])\[(\d+):(\d+)\]", text):
        found |= {(kind, i) for i in range(int(a), int(b) + 1)}
    return found | {(kind, int(a)) for kind, a in re.findall(r"\b([av])(\d+)\b", text)}


def early_reads(code: list) -> list:
    """(function's instruction, reader, wait states) of every result read too early, on any path;
    code: (operation, operands, address, target address or None)."""
    at = {x[2]: i for i, x in enumerate(code)}
    found = []
    for i, (op, args, _, _) in enumerate(code):
        if op not in WAITS:
            continue
        result, seen = registers(args.split(",")[0]), set()
        paths = [(i + 1, 0)]
        while paths:
            j, waited = paths.pop()
            while j < len(code) and waited < WAITS[op] and (j, waited) not in seen:
                seen.add((j, waited))
                other, operands, _, target = code[j]
                if other == "s_nop":
                    waited += int(operands) + 1
                elif other == "s_branch":
                    j, waited = at.get(target, len(code)), waited + 1
                    continue
                elif other == "s_endpgm":
                    break
                else:
                    if other.startswith("s_cbranch"):
                        paths.append((at.get(target, len(code)), waited + 1))
                    elif other.startswith("v_mfma"):
                        # products wait for each other by themselves; one may write the result anew
                        if registers(operands.split(",")[0]) >= result:
                            break
                    else:
                        stores = re.match(r"(global|scratch|buffer|flat)_store|ds_write|\w*atomic", other)
                        sources = operands if stores else operands.partition(",")[2]
                        if registers(sources) & result:
                            found.append((f"{op} {args}", f"{other} {operands}", waited))
                            break
                    waited += 1
                j += 1
    return found


def functions(text: str) -> dict:
    found, code, start = {}, None, 0
    for line in text.split("\n"):
        head = re.match(r"^([0-9a-f]{16}) <(\S+)>:", line)
        if head:
            start, code = int(head[1], 16), []
            found[head[2]] = code
        elif code is not None and (m := LINE.match(line)):
            target = None if m[4] is None else start + int(m[4], 16)
            code.append((m[1], m[2], int(m[3], 16), target))
    return found


def test_the_check_finds_an_early_read():
    mfma = ("v_mfma_f32_16x16x32_bf16", "a[0:3], v[0:3], v[4:7], 0", 0, None)
    read = ("v_accvgpr_read_b32", "v9, a3", 12, None)
    assert early_reads([mfma, ("s_cbranch_vccnz", "4", 4, 12), ("s_nop", "15", 8, None), read])
    assert early_reads([mfma, ("s_nop", "6", 8, None), read])
    assert not early_reads([mfma, ("s_nop", "7", 8, None), read])
    assert not early_reads([mfma, ("v_mov_b32_e32", "v9, v10", 4, None)])


def test_results_are_waited_for(tmp_path):
    if not OBJDUMP.exists() or not shutil.which("objcopy"):
        pytest.skip("no ROCm LLVM tools")
    products = 0
    for obj in build.code_objects(REPO / "cugo_amd" / "libcugo_hip.so", tmp_path):
        text = subprocess.run([str(OBJDUMP), "-d", str(obj)], check=True, capture_output=True,
                              text=True).stdout
        for name, code in functions(text).items():
            products += sum(x[0] in WAITS for x in code)
            assert not early_reads(code), name
    assert products > 1000
