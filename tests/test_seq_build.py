"""What `make` builds, as it would (-n): the C library needs no torch, the calls from Python are built beside it where there is one;
and the limits that header, library and Python share."""
import os
import re
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


def test_the_limits_are_the_headers():
    """The largest sizes stand in include/ttsx_seq.h; the checks in Python name the same."""
    from tts_amd import adapters, recurrence
    header = open(os.path.join(ROOT, "include", "ttsx_seq.h")).read()
    limits = {name: 1 << int(bits) for name, bits in re.findall(r"#define TTSX_SEQ_MAX_(\w+) \(1 << (\d+)\)", header)}
    assert limits == {"WIDTH": adapters.MAX_WIDTH, "ROWS": adapters.MAX_ROWS, "VOICES": adapters.MAX_VOICES}
    assert adapters.FURTHEST == recurrence.FURTHEST == recurrence.MAX_CHANNELS == limits["WIDTH"]
    assert recurrence.MAX_STEPS == limits["ROWS"]
    for source in ("gated_scan.hip", "adapters.hip", "seq_calls.cpp"):
        code = re.sub(r"//.*", "", open(os.path.join(ROOT, "tts_amd", "csrc", source)).read())
        assert not re.search(r"1 << (20|24|30)\b", code)            # no second copy beside the header's
