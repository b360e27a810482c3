"""The row offsets of the token-sequence kernels (cssm_amd/csrc/token_rows.h) against 64-bit arithmetic, on the host:
tests/token_rows_check.hip is built for the host only and run; no GPU."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_offsets_of_long_sequences(tmp_path):
    """sequences whose first and last rows lie more than 2^32 bytes apart, and short ones"""
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("hipcc not available")
    exe = str(tmp_path / "token_rows_check")
    subprocess.run([hipcc, "-O2", "-std=c++17", "--cuda-host-only", "-I", os.path.join(ROOT, "cssm_amd", "csrc"),
                    os.path.join(ROOT, "tests", "token_rows_check.hip"), "-o", exe], check=True, capture_output=True)
    rows = [line.split() for line in subprocess.run([exe], check=True, capture_output=True, text=True).stdout.splitlines()]
    assert len(rows) == 13
    for T, row, narrow, wide in rows:
        assert (int(narrow), int(wide)) == (0, 0), (T, row)
