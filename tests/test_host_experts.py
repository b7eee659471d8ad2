"""The C++ binding converts the weights of all experts, a rank-3 tensor, to and from microscaled values in one call."""
import os
import shutil
import subprocess

import pytest

from beantensor_b200 import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def build(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no g++")
    cuda_inc, cuda_lib = "/usr/local/cuda/include", "/usr/local/cuda/lib64"
    if not os.path.isdir(cuda_inc):
        pytest.skip("no CUDA toolkit headers")
    _lib.lib()
    exe = tmp_path / "host_experts"
    libdir = os.path.join(ROOT, "beantensor_b200")
    subprocess.check_call([gxx, "-std=c++23", "-O1", "-Wall", "-Werror", os.path.join(ROOT, "tests", "host_experts_main.cpp"), "-o", str(exe),
                           f"-I{cuda_inc}", f"-L{libdir}", "-lbtm", f"-Wl,-rpath,{libdir}", f"-L{cuda_lib}", "-lcudart", f"-Wl,-rpath,{cuda_lib}"])
    return exe


def test_guards(tmp_path):
    r = subprocess.run([str(build(tmp_path))], capture_output=True, text=True)
    assert r.returncode == 0 and "passed=13" in r.stdout, r.stdout + r.stderr


@pytest.mark.gpu
def test_experts(tmp_path):
    r = subprocess.run([str(build(tmp_path)), "gpu"], capture_output=True, text=True)
    assert r.returncode == 0 and "passed=16" in r.stdout, r.stdout + r.stderr
