"""Launches where the runtime refuses programmatic dependent launch, without a GPU: the helpers of vrb_common.cuh are compiled for
the host against a runtime that refuses it, and no kernel is launched in any other way."""
import glob
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "vrhino_b200", "csrc")


def test_refused_attribute(tmp_path):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not (shutil.which("g++") and os.path.exists(nvcc)):
        pytest.skip("needs a host compiler and the CUDA headers")
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(nvcc))), "include")
    program = str(tmp_path / "launch_fallback")
    built = subprocess.run(["g++", "-std=c++17", "-O1", "-I", os.path.join(ROOT, "include"), "-I", CSRC, "-I", include, "-x", "c++",
                            os.path.join(ROOT, "tests", "launch_fallback.cpp"), "-o", program], capture_output=True, text=True)
    assert built.returncode == 0, built.stderr[-3000:]
    done = subprocess.run([program], capture_output=True, text=True, timeout=60)
    assert done.returncode == 0 and "all launches went through" in done.stdout, done.stdout + done.stderr


def test_no_launch_with_attributes_of_its_own():
    """Attributes are put together in one place, the one that knows what to do without them."""
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu"))):
        with open(path) as fh:
            text = re.sub(r"//[^\n]*", "", fh.read())
        assert "cudaLaunchKernelEx" not in text, path
