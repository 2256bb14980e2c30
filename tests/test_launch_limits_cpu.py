"""Launch shapes that follow a problem's depth or width (synaptik_amd/csrc/launch_limits.h), built for
the host: within what a grid holds at every accepted extent, and every unit of work reached."""
import shutil
import subprocess
from pathlib import Path

import pytest

HERE = Path(__file__).resolve().parent


def test_launches_stay_within_a_grid(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    exe = tmp_path / "launch_limits_harness"
    subprocess.run([gxx, "-O1", "-std=c++17", "-Wall", "-Werror", "-o", str(exe),
                    str(HERE / "launch_limits_harness.cpp")], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.strip()
    assert out == "ok", out
