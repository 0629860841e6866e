"""The training operators refuse buffers on another GPU than the engine's,
whichever argument it is, before any CUDA call: checked on CPU by a small C++
program over engine and buffer objects of its own (refusals_main.cpp)."""

import os
import subprocess

import pytest

import emeans_b200 as eb
from emeans_b200 import build as ebuild

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.mark.timeout(300)
def test_buffers_on_another_gpu_are_refused(tmp_path):
    try:
        nvcc = ebuild.nvcc()
    except RuntimeError:
        pytest.skip("nvcc not available")
    eb.load()
    exe = str(tmp_path / "refusals")
    subprocess.run([nvcc, *ebuild.ARCH, "-O1", "-std=c++17", "-I" + os.path.join(ebuild.ROOT, "include"),
                    "-I" + ebuild.CSRC, os.path.join(HERE, "refusals_main.cpp"), "-o", exe,
                    "-L" + ebuild.HERE, "-lemeans_b200", "-Xlinker", "-rpath," + ebuild.HERE], check=True)
    res = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert res.returncode == 0, res.stdout + res.stderr
