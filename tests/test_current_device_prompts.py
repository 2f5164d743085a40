"""Prompts, trees, page tables and slots leave the caller's current device as it was and launch nothing where theirs can not be made current.

Two devices, by a C++ program that links the library's own sources with a CUDA runtime of its own (tests/native/current_device_prompts.cc)."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    compiler = shutil.which("g++")
    include = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "include")
    if not compiler or not os.path.exists(os.path.join(include, "cuda_runtime.h")):
        pytest.skip("no g++ or no CUDA headers")
    csrc, out = os.path.join(ROOT, "pjrtx_b200", "csrc"), str(tmp_path_factory.mktemp("native") / "current_device_prompts")
    # NVRTC, NCCL and what needs them is not reached, so nothing stands in for it
    subprocess.run([compiler, "-std=c++17", "-O1", "-w", "-I", csrc, "-I", include, os.path.join(ROOT, "tests", "native", "current_device_prompts.cc"),
                    os.path.join(csrc, "operators.cc"), os.path.join(csrc, "device.cc"), "-o", out, "-ldl", "-lpthread",
                    "-Wl,--unresolved-symbols=ignore-all"], check=True)
    return out


@pytest.mark.parametrize("first", ["prompt", "cache"])
def test_operators_leave_the_current_device(program, first):
    done = subprocess.run([program, first], capture_output=True, text=True, timeout=60)
    assert done.returncode == 0 and done.stdout == "", (done.returncode, done.stdout, done.stderr)
