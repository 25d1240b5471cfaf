"""The rules that the sequence operators' kernels follow
(ml_framework_amd/csrc/sequence_rules.h) against what they are for:
tests/cpp/test_sequence_rules.cpp, on the CPU."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "ml_framework_amd", "csrc")


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not available")
def test_sequence_rules(tmp_path):
    exe = tmp_path / "test_sequence_rules"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", f"-I{CSRC}", os.path.join(ROOT, "tests", "cpp", "test_sequence_rules.cpp"), "-o", str(exe)],
                   check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout
    assert "all checks passed" in out.stdout


def test_row_sums_take_their_half_from_the_rule():
    """A caller of row_sum hands on the block's Halves; no call names a half itself."""
    calls = [line.split("row_sum<NT>(")[1] for line in open(os.path.join(CSRC, "block_norm.hip")) if "row_sum<NT>(" in line]
    assert len(calls) == 4 and all("part, halves)" in c for c in calls), calls
