"""CPU: who gets the counters of a session's launches (csrc/memory.cpp)."""
import pathlib
import subprocess

ROOT = pathlib.Path(__file__).resolve().parents[1]


def test_tickets(tmp_path):
    exe = tmp_path / "tickets_test"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-pthread", f"-I{ROOT / 'tests/memory'}",
                    f"-I{ROOT / 'affon_amd/csrc'}", str(ROOT / "tests/memory/tickets_test.cpp"),
                    str(ROOT / "affon_amd/csrc/memory.cpp"), "-o", str(exe)], check=True)
    result = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert result.returncode == 0, result.stdout + result.stderr
