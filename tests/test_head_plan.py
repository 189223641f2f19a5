"""The class head's plans, read without a GPU: head_plan_check.cpp compiles csrc/head_plan.hpp, which the
host side launches by, with a host compiler, and walks every tile of a sweep of calls and of drawn ones."""
from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

HERE = Path(__file__).resolve().parent


def test_every_tile_lies_inside_its_operands(tmp_path):
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no host C++ compiler")
    exe = tmp_path / "head_plan_check"
    subprocess.run([cxx, "-std=c++17", "-O2", "-Wall", "-Werror", f"-I{HERE.parent / 'include'}",
                    f"-I{HERE.parent / 'tiny-metal-nn_amd' / 'csrc'}", str(HERE / "head_plan_check.cpp"), "-o", str(exe)],
                   check=True)
    got = subprocess.run([str(exe), "4000"], capture_output=True, text=True)
    assert got.returncode == 0, got.stdout
    plans, several = (int(got.stdout.splitlines()[-1].split()[i]) for i in (0, 2))
    assert plans > 50000 and several > 5000
