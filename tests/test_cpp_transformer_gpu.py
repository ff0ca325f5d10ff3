"""Compiles and runs tests/cpp/test_transformer_mirror.cpp: the embedding, the norm / gate / residual step and the grouped
Adam driven from compiled host code through the C++ mirror."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CUDA = os.environ.get("CUDA_HOME", "/usr/local/cuda")


def _compile(built_library, out):
    lib_dir = os.path.dirname(built_library)
    cmd = ["g++", "-std=c++17", "-O2", os.path.join(ROOT, "tests", "cpp", "test_transformer_mirror.cpp"), "-I", f"{CUDA}/include",
           "-L", lib_dir, "-L", f"{CUDA}/lib64", "-lsharpnet_b200", "-lcudart", f"-Wl,-rpath,{lib_dir}",
           f"-Wl,-rpath,{CUDA}/lib64", "-o", out]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    assert proc.returncode == 0, proc.stdout + proc.stderr
    return out


def test_cpp_transformer_mirror_compiles(built_library, tmp_path):
    _compile(built_library, str(tmp_path / "test_transformer_mirror"))


@pytest.mark.gpu
def test_cpp_transformer_mirror_runs(built_library, tmp_path, wrapper):
    exe = _compile(built_library, str(tmp_path / "test_transformer_mirror"))
    proc = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert proc.returncode == 0, proc.stdout + proc.stderr
    assert proc.stdout.strip().splitlines()[-1].startswith("OK"), proc.stdout
