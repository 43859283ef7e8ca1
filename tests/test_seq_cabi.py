"""include/ttsx_seq.h: every declared symbol is exported and bound, and bad arguments come back as errors before any
device call (no GPU needed)."""
import ctypes
import os
import re

import pytest
import torch

from conftest import ROOT


def test_library_exports_every_declared_sequence_operator():
    from tts_amd import _lib
    header = open(os.path.join(ROOT, "include", "ttsx_seq.h")).read()
    code = re.sub(r"/\*.*?\*/", "", header, flags=re.S)
    declared = set(re.findall(r"\b(ttsx_[a-z0-9_]+)\s*\(", code))
    assert declared == set(_lib.SEQ_PROTOTYPES), declared ^ set(_lib.SEQ_PROTOTYPES)
    lib = ctypes.CDLL(_lib.LIB_PATH)
    for name in sorted(declared):
        assert hasattr(lib, name), name


def test_the_block_of_kept_states_is_the_headers():
    from tts_amd import recurrence
    header = open(os.path.join(ROOT, "include", "ttsx_seq.h")).read()
    assert int(re.search(r"#define TTSX_STATE_BLOCK (\d+)", header).group(1)) == recurrence.STATE_BLOCK


ONE = ctypes.c_void_p(256)   # non-null, never dereferenced on these paths


def _scan(lib, x=ONE, g=ONE, B=2, T=8, D=16, dtype=0, h=ONE, h_last=ONE, ws=None, n=0):
    return lib.ttsx_gated_scan(x, 8, 8, g, 8, 8, None, None, B, T, D, dtype, 0, h, h_last, None, ws, n, None)


def _scan_backward(lib, dh=ONE, states=ONE, B=2, T=8, D=16, dtype=0, dx=ONE, ws=None, n=0):
    return lib.ttsx_gated_scan_backward(dh, 8, 8, ONE, 8, 8, ONE, 8, 8, states, None, None, B, T, D, dtype, 0, dx, ONE,
                                        ONE, ws, n, None)


def _step(lib, x=ONE, h=ONE, B=2, D=16, dtype=0, y=ONE):
    return lib.ttsx_gated_step(x, 8, ONE, 8, h, B, D, dtype, y, ONE, None)


@pytest.mark.parametrize("call,bad", [
    (_scan, dict(x=None)), (_scan, dict(g=None)), (_scan, dict(h=None)), (_scan, dict(h_last=None)),
    (_scan, dict(B=0)), (_scan, dict(T=0)), (_scan, dict(D=0)), (_scan, dict(T=-1)), (_scan, dict(dtype=3)),
    (_scan, dict(B=1, T=100000)),                    # a cut time axis without its workspace
    (_scan, dict(B=1, T=100000, ws=ONE, n=16)),      # or with too little of it
    (_scan_backward, dict(dh=None)), (_scan_backward, dict(states=None)), (_scan_backward, dict(dx=None)),
    (_scan_backward, dict(B=0)), (_scan_backward, dict(T=0)), (_scan_backward, dict(D=0)),
    (_scan_backward, dict(dtype=-1)), (_scan_backward, dict(B=1, T=100000)),
    (_step, dict(x=None)), (_step, dict(h=None)), (_step, dict(y=None)), (_step, dict(B=0)), (_step, dict(D=0)),
    (_step, dict(dtype=7)),
])
def test_bad_arguments_of_the_recurrence(call, bad):
    from tts_amd import _lib
    lib = _lib.load()
    assert call(lib, **bad) == _lib.ERR_ARG
    assert lib.ttsx_last_error_string().decode().startswith("ttsx_gated_")


def test_workspace_of_the_recurrence():
    from tts_amd import _lib
    lib = _lib.load()
    assert lib.ttsx_gated_scan_workspace(0, 8, 8, 0, 0) == _lib.ERR_ARG
    assert lib.ttsx_gated_scan_workspace(1, 8, 8, 5, 0) == _lib.ERR_ARG
    for backward in (0, 1):
        for dtype in (0, 1, 2):
            assert lib.ttsx_gated_scan_workspace(1, 1, 8, dtype, backward) == 0
            assert lib.ttsx_gated_scan_workspace(64, 800, 4096, dtype, backward) == 0
            assert lib.ttsx_gated_scan_workspace(1, 100000, 64, dtype, backward) > 0


def test_python_refusals_of_the_recurrence():
    """Shapes, types and places are checked before anything is launched; CPU tensors are refused, not computed."""
    from tts_amd import _lib
    from tts_amd.recurrence import gated_scan, gated_scan_backward, gated_step
    x = torch.zeros(2, 5, 8)
    with pytest.raises(_lib.TtsxError, match="no CPU path"):
        gated_scan(x, x)
    with pytest.raises(_lib.TtsxError, match="no CPU path"):
        gated_scan_backward(x, x, x, torch.zeros(2, 1, 8))
    with pytest.raises(_lib.TtsxError, match="no CPU path"):
        gated_step(x[:, 0], x[:, 0], x[:, 0])
    for args, kw, why in [
            ((x, x[:, :4]), {}, "must both be"), ((x[0], x[0]), {}, "must both be"),
            ((x, x.half()), {}, "float32, bfloat16 or float16"), ((x.double(), x.double()), {}, "float32, bfloat16"),
            ((x, None), {}, "must be a tensor"), ((x, x), dict(h0=torch.zeros(2, 9)), "h0 must be float32"),
            ((x, x), dict(h0=torch.zeros(2, 8).half()), "h0 must be float32"),
            ((x.requires_grad_(), x), {}, "records no autograd graph")]:
        with pytest.raises(ValueError, match=why):
            gated_scan(*args, **kw)
    x = torch.zeros(2, 5, 8)
    for args, why in [((x[:, :4], x, x, torch.zeros(2, 1, 8)), "dh must be"), ((x, x, x, torch.zeros(2, 2, 8)), "states must"),
                      ((x, x, x, torch.zeros(2, 1, 8).half()), "states must"), ((x, x, x, None), "must be a tensor")]:
        with pytest.raises(ValueError, match=why):
            gated_scan_backward(*args)
    for args, why in [((x, x, x), "must both be"), ((x[:, 0], x[:, 0], x[:, 0].half()), "h must be float32"),
                      ((x[:, 0], x[:, 0], x[:1, 0]), "h must be float32")]:
        with pytest.raises(ValueError, match=why):
            gated_step(*args)


def test_lengths_are_checked_on_the_host():
    from tts_amd._seq import lengths_on
    assert lengths_on("f", None, 2, 5, torch.device("cpu")) is None
    assert lengths_on("f", [0, 5], 2, 5, torch.device("cpu")).dtype == torch.int32
    for bad in ([6, 1], [-1, 1], [1], [0.5, 1.0]):
        with pytest.raises(ValueError):
            lengths_on("f", bad, 2, 5, torch.device("cpu"))
