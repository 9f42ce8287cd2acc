"""Where the tiles of 4-bit rows read (vectoraccelerate_amd/csrc/va_mx_tile.hpp), checked lane by lane on the CPU by
tests/cpp/mx_tile_host.cpp."""
from __future__ import annotations

import subprocess
from pathlib import Path

SRC = Path(__file__).resolve().parent / "cpp" / "mx_tile_host.cpp"


def test_no_lane_reads_past_its_rows(tmp_path):
    exe = tmp_path / "mx_tile_host"
    proc = subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Wextra", "-Werror", str(SRC), "-o", str(exe)], capture_output=True, text=True)
    assert proc.returncode == 0, proc.stderr
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0 and "ok" in run.stdout, run.stdout + run.stderr
