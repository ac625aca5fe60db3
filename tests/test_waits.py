"""The bounded wait of the tensor-core pipelines' warps: one answer for all lanes."""
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]


@pytest.fixture(scope="module")
def waits(tmp_path_factory):
    import build
    exe = tmp_path_factory.mktemp("waits") / "waits"
    r = subprocess.run([build.nvcc(), *build.ARCH, "-O2", "-std=c++17", "-I",
                        str(ROOT / "qwen3.cpp_b200" / "csrc"), str(ROOT / "tests" / "cxx" / "test_waits.cu"),
                        "-o", str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    return exe


def test_wait_program_builds(waits):
    assert waits.exists()


@pytest.mark.gpu
def test_a_warp_waits_together(waits):
    r = subprocess.run([str(waits)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "wait tests passed" in r.stdout, r.stdout + r.stderr
    assert r.stdout.count(": 1") >= 1
