"""CPU: which operands share memory (csrc/overlap.h)."""
import pathlib
import subprocess

import pytest

ROOT = pathlib.Path(__file__).resolve().parents[1]


@pytest.fixture(scope="module")
def driver(tmp_path_factory):
    exe = tmp_path_factory.mktemp("overlap") / "overlap_test"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", f"-I{ROOT / 'affon_amd/csrc'}",
                    str(ROOT / "tests/overlap/overlap_test.cpp"), "-o", str(exe)], check=True)
    return exe


@pytest.mark.parametrize("seed", [1, 2, 3])
def test_rows_that_meet(driver, seed):
    result = subprocess.run([str(driver), str(seed)], capture_output=True, text=True, timeout=60)
    assert result.returncode == 0, result.stdout + result.stderr
