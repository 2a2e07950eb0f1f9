"""The loop of the bounded device-side waits (qwen3x-orin_b200/csrc/bounded_wait.hpp), compiled for the host with a barrier and
a clock made up by the test: time in which the process is switched off the GPU must not fail a wait."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_bounded_wait(tmp_path):
    exe = str(tmp_path / "wait")
    cmd = ["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", os.path.join(ROOT, "tests", "host", "bounded_wait_test.cpp"),
           "-o", exe, "-I", os.path.join(ROOT, "qwen3x-orin_b200", "csrc")]
    subprocess.run(cmd, check=True, capture_output=True, text=True)
    out = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0, out.stdout + out.stderr
    assert "bounded wait tests passed" in out.stdout
