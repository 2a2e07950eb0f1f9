"""The C++ front end of the FP8 operators with a scale per block of 128 (qwen3x-orin_b200/host/q3x_b200_fp8_block.hpp):
compiled and linked like a runner's code; its refusals on the CPU, its calls against the C ABI on a GPU."""
import importlib
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "qwen3x-orin_b200")
CUDA = os.environ.get("CUDA_HOME", "/usr/local/cuda")


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    build = importlib.import_module("qwen3x-orin_b200.build")
    build.build_all()
    exe = str(tmp_path_factory.mktemp("fp8") / "front")
    cmd = ["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", os.path.join(ROOT, "tests", "host", "fp8_block_front_test.cpp"),
           "-o", exe, "-I", os.path.join(PKG, "host"), "-I", os.path.join(ROOT, "include"), "-isystem", os.path.join(CUDA, "include"),
           "-L", PKG, "-lq3x_b200_host", "-lq3x_b200", f"-Wl,-rpath,{PKG}", "-L", os.path.join(CUDA, "lib64"), "-lcudart",
           f"-Wl,-rpath,{os.path.join(CUDA, 'lib64')}", "-Wl,--no-undefined"]
    subprocess.run(cmd, check=True, capture_output=True, text=True)
    return exe


def test_front_end_refusals(program):
    out = subprocess.run([program], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0, out.stdout + out.stderr
    assert "fp8 block front end tests passed" in out.stdout


@pytest.mark.gpu
def test_front_end_equals_the_c_abi(program):
    out = subprocess.run([program, "gpu"], capture_output=True, text=True, timeout=240)
    assert out.returncode == 0, out.stdout + out.stderr
    assert "fp8 block front end tests passed" in out.stdout
