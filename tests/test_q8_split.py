"""The work split of the 8-bit decode attention, on the host: pieces, owners, and arrival counters that
return to zero when warps give up (tests/native/q8_split_check.cpp over csrc/q8_split.cuh)."""

from __future__ import annotations

import pathlib
import shutil
import subprocess

import pytest

HERE = pathlib.Path(__file__).resolve().parent
CSRC = HERE.parent / "plastic_infer_b200" / "csrc"


def test_split_and_counters(tmp_path) -> None:
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("g++ is not available")
    exe = tmp_path / "q8_split_check"
    subprocess.run([cxx, "-std=c++17", "-O1", "-Wall", f"-I{CSRC}", "-x", "c++", "-o", str(exe),
                    str(HERE / "native" / "q8_split_check.cpp")], check=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0 and run.stdout.strip() == "ok", run.stdout
