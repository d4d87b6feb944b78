"""The 16-bit cache's integer geometry (p16_geometry.h), compiled with g++ and
checked on the CPU."""

from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

from pth_flash_attn import planner

REPO = Path(__file__).resolve().parent.parent


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_geometry16_header(tmp_path):
    exe = tmp_path / "test_p16_geometry"
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", "-fwrapv",
                    f"-I{REPO / 'pth-flash-attn_amd' / 'csrc'}",
                    str(REPO / "tests" / "cpp" / "test_p16_geometry.cpp"), "-o", str(exe)],
                   check=True)
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stdout + res.stderr
    assert "ALL OK" in res.stdout
    # The planner's sizes are the launcher's.
    sizes = [tuple(map(int, line.split()[1:])) for line in res.stdout.splitlines()
             if line.startswith("workspace")]
    assert {d for d, _, _ in sizes} == {64, 128, 256}
    for d, cus, floats in sizes:
        assert planner.paged16_workspace_floats(D=d, num_sms=cus) == floats


def test_workspace_sizes():
    assert [planner.paged16_workspace_floats(D=d, num_sms=256) for d in (64, 128, 256)] == [
        256 * (768 * 66 + 32), 256 * (512 * 130 + 32), 256 * (256 * 258 + 32)]
