"""The ways that ml_framework_amd/csrc/f8_routes.h chooses for products of operands in 8 bits at the sizes of
matmul_f8_ways.py: tests/cpp/test_f8_routes.cpp, on the CPU. A change of the rule that takes a way out of the
reach of the GPU tests shows here."""
import os
import shutil
import subprocess

import pytest

from tests.matmul_f8_ways import TILES_128, TILES_256, WAYS

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not available")
def test_ways(tmp_path):
    exe = tmp_path / "test_f8_routes"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", f"-I{os.path.join(ROOT, 'ml_framework_amd', 'csrc')}",
                    os.path.join(ROOT, "tests", "cpp", "test_f8_routes.cpp"), "-o", str(exe)], check=True)

    def run(ways):
        return subprocess.run([str(exe)], input="".join("%d %d %d %d %d\n" % w for w in ways), capture_output=True, text=True)

    out = run(WAYS)
    assert out.returncode == 0 and "all checks passed" in out.stdout, out.stdout
    # planted: a size that takes another way, a way that no size takes, a way with too few tiles
    assert "not 7" in run([*WAYS, (0, 1, 1, 1, TILES_256)]).stdout
    assert "no size takes way 7" in run([w for w in WAYS if w[4] != TILES_256]).stdout
    assert "second tile" in run([*WAYS, (0, 2050, 1300, 1152, TILES_128)]).stdout
