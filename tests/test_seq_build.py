"""What `make` builds, as it would (-n): the C library needs no torch, the calls from Python are built beside it where there is one."""
import os
import subprocess
import sys

import torch

from conftest import ROOT


def _would(python):
    return subprocess.run(["make", "-n", "-B", "-C", os.path.join(ROOT, "tts_amd", "csrc"), "PYTHON=" + python],
                          capture_output=True, text=True, timeout=120)


def test_the_c_library_without_torch():
    for python in ("/bin/false", sys.executable + " -S -E"):        # no interpreter; one without installed packages
        got = _would(python)
        assert got.returncode == 0, got.stderr
        assert "libttsx.so" in got.stdout and "gated_scan.hip" in got.stdout
        assert "seq_calls.cpp" not in got.stdout and "_seqcalls.so is left out" in got.stdout


def test_the_calls_with_torch():
    got = _would(sys.executable)
    assert got.returncode == 0, got.stderr
    lines = got.stdout.replace("\\\n", " ").split("\n")
    line = next(part for part in lines if "seq_calls.cpp" in part)
    assert "-D_GLIBCXX_USE_CXX11_ABI=%d" % torch.compiled_with_cxx11_abi() in line and "left out" not in got.stdout
