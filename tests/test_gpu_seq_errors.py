"""What becomes of errors of the GPU's runtime in the sequence operators: a call is made once, whoever left the error."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu


def _runtime():
    """The HIP runtime that this process has loaded."""
    from tts_amd import _lib
    _lib.load()
    path = next(line.split()[-1] for line in open("/proc/self/maps") if "libamdhip64" in line)
    return ctypes.CDLL(path)


def _inputs():
    gen = torch.Generator(device="cuda").manual_seed(1)
    x, g, h = (torch.randn(3, 8, device="cuda", generator=gen) for _ in range(3))
    m = torch.randn(2, 4, 8, device="cuda", generator=gen)
    return x, g, h, m, torch.tensor([1, 0, -1], dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("native", [True, False])
def test_an_error_that_another_call_left(native, monkeypatch):
    """The update in place happens once, nothing is reported, and the error is still there for the one it belongs to."""
    from tts_amd import _seq
    from tts_amd.adapters import adapter_add
    from tts_amd.recurrence import gated_scan, gated_step
    _seq._bind()
    if not native:
        monkeypatch.setattr(_seq.ways, "ordinary", _seq._Unbound)
    hip = _runtime()
    x, g, h, m, voices = _inputs()
    want, out, seq = gated_step(x, g, h)[1], adapter_add(g, x, m, m, voices), gated_scan(x[:, None], g[:, None], h0=h)[1]
    for call, state, new in ((lambda: gated_step(x, g, h, out=h), h, want),
                             (lambda: adapter_add(g, x, m, m, voices, out=g), g, out)):
        torch.cuda.synchronize()
        assert hip.hipSetDevice(99) != 0                # refused on the host, and remembered
        call()
        assert hip.hipGetLastError() != 0 and hip.hipGetLastError() == 0
        torch.cuda.synchronize()
        assert torch.equal(state, new)
    assert torch.equal(seq, want)


def test_a_launch_that_fails_is_reported_once():
    """Entry points that report an error of the runtime: each is called once, and its error comes out."""
    from tts_amd import _lib, _seq, _seqcalls
    from tts_amd.adapters import adapter_add, adapter_backward
    from tts_amd.recurrence import gated_scan, gated_scan_backward, gated_step
    _seq._bind()
    lib, calls = _lib.load(), []
    x, g, h, m, voices = _inputs()
    x3, states = x[:, None].contiguous(), torch.zeros(3, 1, 8, device="cuda")

    def failing(name):
        res, args = _lib.SEQ_PROTOTYPES[name]

        def entry(*_):
            calls.append(name)
            return _lib.ERR_HIP
        return ctypes.CFUNCTYPE(res, *args)(entry)
    names = ("ttsx_gated_step", "ttsx_gated_scan", "ttsx_gated_scan_backward", "ttsx_gated_scan_workspace", "ttsx_adapter_add",
             "ttsx_adapter_backward", "ttsx_adapter_backward_workspace")
    stubs = [getattr(lib, n) if n.endswith("workspace") else failing(n) for n in names]
    _seqcalls.bind(*(ctypes.cast(s, ctypes.c_void_p).value for s in stubs))
    try:
        for f in (lambda: gated_step(x, g, h, out=h), lambda: gated_scan(x3, x3), lambda: gated_scan_backward(x3, x3, x3, states),
                  lambda: adapter_add(g, x, m, m, voices, out=g), lambda: adapter_backward(g, x, m, m, voices)):
            before = len(calls)
            with pytest.raises(_lib.TtsxError, match="ttsx_"):
                f()
            assert len(calls) == before + 1
    finally:
        _seq._bind()
    assert sorted(calls) == sorted(n for n in names if not n.endswith("workspace"))
