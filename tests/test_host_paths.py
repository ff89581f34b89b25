"""Builds and runs tests of host code on a device of their own (tests/cpp/fake_device.h; no GPU): the same sources as in the
library, compiled for the host alone."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("name, sources", [
    ("test_index_operands", ["ops_api.cu", "flat_index.cu"]),
    ("test_flat_errors", ["flat_index.cu"]),
    ("test_cluster_limit", []),
])
def test_host_paths(tmp_path, name, sources):
    exe = str(tmp_path / name)
    csrc = [os.path.join(ROOT, "indexsdk_b200", "csrc", s) for s in sources]
    # (CUDA's headers bring string.h for nvcc only)
    subprocess.run(["/usr/bin/g++", "-std=c++17", "-O1", "-x", "c++", "-include", "cstring", "-I", "/usr/local/cuda/include",
                    "-fno-access-control", os.path.join(ROOT, "tests", "cpp", name + ".cpp"), *csrc, "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and "0 failed" in r.stdout, r.stdout + r.stderr
