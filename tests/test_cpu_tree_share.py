"""CPU: how the attention of drafted tokens shares out its work, built for the host: any offsets, any
remains in the workspace."""

from __future__ import annotations

import os
import shutil
import subprocess
from pathlib import Path

import pytest

from tests.conftest import REPO

HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")


def test_shares_stay_inside(tmp_path):
    """Parts that are joined were written for what they are joined for, also where offsets fall, make
    more work than 32 bits count, and the workspace held other numbers."""
    if not (Path(HIPCC).exists() or shutil.which("hipcc")):
        pytest.skip("hipcc is not installed")
    exe = tmp_path / "share_check"
    subprocess.run([HIPCC, "-O1", "-std=c++17", f"-I{REPO / 'cugo_amd' / 'csrc'}",
                    str(REPO / "tests" / "tree_share_check.cpp"), "-o", str(exe)], check=True,
                   capture_output=True, timeout=300)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "inside" in out.stdout, out.stdout + out.stderr
