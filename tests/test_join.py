"""CPU: which thread of a join holds what (csrc/join_thread.h)."""
import pathlib
import subprocess

ROOT = pathlib.Path(__file__).resolve().parents[1]


def test_threads_of_a_join(tmp_path):
    exe = tmp_path / "join_test"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", f"-I{ROOT / 'affon_amd/csrc'}", str(ROOT / "tests/join/join_test.cpp"),
                    "-o", str(exe)], check=True)
    result = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert result.returncode == 0, result.stdout + result.stderr
