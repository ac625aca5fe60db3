"""The index arithmetic of draft verification, on the host."""
import subprocess
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]
CXX = "/usr/bin/g++" if Path("/usr/bin/g++").exists() else "g++"


def test_pieces_tile_every_row(tmp_path):
    exe = tmp_path / "pieces"
    r = subprocess.run([CXX, "-std=c++17", "-O2", "-I", str(ROOT / "qwen3.cpp_b200" / "csrc"),
                        str(ROOT / "tests" / "cxx" / "test_verify_pieces.cpp"), "-o", str(exe)],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "verify pieces passed" in r.stdout, r.stdout
