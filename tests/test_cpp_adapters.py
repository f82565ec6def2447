"""The C++ mirror of the low-rank adapters and of the norm between two blocks (include/mfmoe.hpp), driven by a C++ program: sizes and
refusals on the CPU, results against loops in 64 bits on the GPU."""
import os
import subprocess

import pytest

CPP = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp")


def run(mode):
    binary = os.path.join(CPP, "adapters_test")
    if not os.path.exists(binary):  # normally built by __graft_entry__.build()
        from mference_amd import _capi
        _capi.lib()
        subprocess.run(["make", "-C", CPP, "adapters_test"], check=True, capture_output=True)
    r = subprocess.run([binary, mode], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "adapters_test: ok" in r.stdout
    return r.stdout


def test_cpp_adapters_sizes_and_refusals():
    run("cpu")


@pytest.mark.gpu
def test_cpp_adapters_on_gpu():
    assert run("gpu").count(": ok") == 6
