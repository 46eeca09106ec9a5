"""Which rows are stored through a 16-byte aligned type, without a GPU: nt_rows.hpp built by the host compiler."""

from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_aligned_rows(tmp_path):
    source = Path(__file__).resolve().parent / "host" / "rows_aligned_test.cpp"
    binary = tmp_path / "rows_aligned_test"
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", str(source), "-o", str(binary)], check=True)
    result = subprocess.run([str(binary)], capture_output=True, text=True)
    assert result.returncode == 0, result.stdout + result.stderr
