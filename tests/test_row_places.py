"""The addresses that the lanes of the norms read (csrc/row_places.hpp), held inside the rows (tests/host/row_places_driver.cpp)."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_nothing_is_read_behind_a_row(tmp_path):
    """Rows of two-byte elements that start between two words, of odd and even widths and pitches."""
    if not shutil.which("g++"):
        pytest.skip("no host compiler")
    exe = os.path.join(tmp_path, "places")
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-I", os.path.join(ROOT, "aws_ofi_nccl_amd", "csrc"),
                    os.path.join(ROOT, "tests", "host", "row_places_driver.cpp"), "-o", exe], check=True)
    proc = subprocess.run([exe], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=120)
    assert proc.returncode == 0 and proc.stdout.endswith("ok\n"), proc.stdout[-4000:]
