"""CPU: the pieces that prefixes are cut into, and the room they get (csrc/prefix_cut.h)."""
import pathlib
import subprocess

ROOT = pathlib.Path(__file__).resolve().parents[1]


def test_pieces_of_prefixes(tmp_path):
    exe = tmp_path / "cut_test"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", f"-I{ROOT / 'affon_amd/csrc'}", str(ROOT / "tests/cut/cut_test.cpp"),
                    "-o", str(exe)], check=True)
    result = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert result.returncode == 0, result.stdout + result.stderr
