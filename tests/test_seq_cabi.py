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
    from tts_amd._seq import lengths_on, voices_on
    like = torch.zeros(1)
    assert lengths_on("f", None, 2, 5, like) is None
    assert lengths_on("f", [0, 5], 2, 5, like).dtype == torch.int32
    for bad in ([6, 1], [-1, 1], [1], [0.5, 1.0]):
        with pytest.raises(ValueError):
            lengths_on("f", bad, 2, 5, like)
    assert voices_on("f", [-1, 4], 2, 5, like).tolist() == [-1, 4]
    for bad in ([5, 0], [-2, 0]):
        with pytest.raises(IndexError):
            voices_on("f", bad, 2, 5, like)


def _add(lib, y=ONE, x=ONE, down=ONE, up=ONE, voices=ONE, B=2, T=8, K=16, N=24, R=4, V=3, dtype=0, out=ONE, out_rows=24):
    return lib.ttsx_adapter_add(y, 192, 24, x, 128, 16, down, up, voices, None, None, B, T, K, N, R, V, dtype, out, 192,
                                out_rows, None)


def _add_backward(lib, dy=ONE, voices=ONE, B=2, T=8, K=16, N=24, R=4, V=3, dtype=0, dx=ONE, dup=ONE, ws=ONE, n=1 << 30):
    return lib.ttsx_adapter_backward(dy, 192, 24, ONE, 128, 16, ONE, ONE, voices, None, None, B, T, K, N, R, V, dtype, dx,
                                     ONE, dup, ws, n, None)


@pytest.mark.parametrize("call,bad", [
    (_add, dict(y=None)), (_add, dict(x=None)), (_add, dict(down=None)), (_add, dict(up=None)), (_add, dict(voices=None)),
    (_add, dict(out=None)), (_add, dict(B=0)), (_add, dict(T=0)), (_add, dict(K=0)), (_add, dict(N=0)), (_add, dict(R=0)),
    (_add, dict(R=65)), (_add, dict(V=0)), (_add, dict(dtype=3)), (_add, dict(out_rows=25)),
    (_add_backward, dict(dy=None)), (_add_backward, dict(voices=None)), (_add_backward, dict(dx=None)),
    (_add_backward, dict(dup=None)), (_add_backward, dict(ws=None)), (_add_backward, dict(n=64)),
    (_add_backward, dict(ws=ctypes.c_void_p(260))), (_add_backward, dict(B=0)), (_add_backward, dict(R=65)),
    (_add_backward, dict(dtype=-1)),
])
def test_bad_arguments_of_the_adapters(call, bad):
    from tts_amd import _lib
    lib = _lib.load()
    assert call(lib, **bad) == _lib.ERR_ARG
    assert lib.ttsx_last_error_string().decode().startswith("ttsx_adapter_")


def test_workspace_and_rank_limit_of_the_adapters():
    from tts_amd import _lib, adapters
    lib = _lib.load()
    header = open(os.path.join(ROOT, "include", "ttsx_seq.h")).read()
    assert int(re.search(r"#define TTSX_ADAPTER_MAX_RANK (\d+)", header).group(1)) == adapters.MAX_RANK
    assert lib.ttsx_adapter_backward_workspace(1, 1, 1, 1, 65, 0) == _lib.ERR_ARG
    assert lib.ttsx_adapter_backward_workspace(1, 1, 1, 1, 1, 3) == _lib.ERR_ARG
    small = lib.ttsx_adapter_backward_workspace(1, 1, 1, 1, 1, 0)
    assert 0 < small < lib.ttsx_adapter_backward_workspace(64, 800, 512, 2048, 32, 1)


def test_python_refusals_of_the_adapters():
    from tts_amd import _lib
    from tts_amd.adapters import adapter_add, adapter_backward
    y, x, down, up = torch.zeros(2, 5, 6), torch.zeros(2, 5, 8), torch.zeros(3, 4, 8), torch.zeros(3, 4, 6)
    v = torch.zeros(2, dtype=torch.int32)
    for call in (adapter_add, adapter_backward):
        with pytest.raises(_lib.TtsxError, match="no CPU path"):
            call(y, x, down, up, v)
        for args, kw, why in [
                ((y, x[:, :4], down, up, v), {}, "must agree"), ((y[0, 0], x[0, 0], down, up, v), {}, "must agree"),
                ((y, x, down[..., :7], up, v), {}, "down and up must be"), ((y, x, down[:2], up, v), {}, "down and up must be"),
                ((y, x, down[:, :0], up[:, :0], v), {}, "rank must lie"),
                ((y, x, torch.zeros(3, 65, 8), torch.zeros(3, 65, 6), v), {}, "rank must lie"),
                ((y.half(), x, down, up, v), {}, "must all be"), ((y, x, down.bfloat16(), up, v), {}, "must all be"),
                ((y.double(), x.double(), down.double(), up.double(), v), {}, "must all be"),
                ((y, x, torch.zeros(3, 8, 4).transpose(1, 2), up, v), {}, "must be contiguous"),
                ((y, x, down, up, v), dict(scale=torch.zeros(2)), "scale must be"),
                ((y, x, down, up, v), dict(scale=torch.zeros(3).half()), "scale must be"),
                ((y, x, down, None, v), {}, "must be a tensor"),
                ((y, x, down, up.clone().requires_grad_(), v), {}, "records no autograd graph")]:
            with pytest.raises(ValueError, match=why):
                call(*args, **kw)


def test_columns_of_one_buffer():
    from tts_amd._seq import columns_apart, overlaps, writable_rows
    buf = torch.zeros(3, 10, 40)
    assert overlaps(buf[..., :16], buf[..., 16:]) and columns_apart(buf[..., :16], buf[..., 16:])
    assert columns_apart(buf[..., 30:], buf[..., :30])
    assert not columns_apart(buf[..., :17], buf[..., 16:])
    assert not columns_apart(buf[:, :5, :20], buf[:, 5:, :20])          # not the same rows: decided by ranges alone
    writable_rows("f", "out", buf.transpose(0, 1))
    for bad in (buf[:1].expand(3, -1, -1), buf.transpose(1, 2), torch.zeros(60).as_strided((2, 3, 8), (24, 4, 1))):
        with pytest.raises(ValueError):
            writable_rows("f", "out", bad)


def test_sizes_beyond_the_entry_points_are_refused():
    """Counts are 32-bit integers at the entry points: a larger one is refused, not cut."""
    from tts_amd.adapters import adapter_add, adapter_backward
    from tts_amd.recurrence import gated_scan, gated_step
    one = torch.zeros(1, 1, 1)
    for shape, why in (((2 ** 32 + 1, 1, 1), "requests and steps"), ((1, 2 ** 32 + 1, 1), "requests and steps"),
                       ((1, 1, 2 ** 20 + 1), "channels")):
        with pytest.raises(ValueError, match=why):
            gated_scan(one.expand(shape), one.expand(shape))
    with pytest.raises(ValueError, match="requests and steps"):
        gated_step(one[0].expand(2 ** 32 + 1, 1), one[0].expand(2 ** 32 + 1, 1), one[0])
    v = torch.zeros(1, dtype=torch.int32)
    for call in (adapter_add, adapter_backward):
        for shape in ((2 ** 32 + 1, 1, 1), (1, 2 ** 32 + 1, 1)):
            with pytest.raises(ValueError, match="requests and positions"):
                call(one.expand(shape), one.expand(shape), one, one, v)
        with pytest.raises(ValueError, match="voices"):
            call(one, one, one.expand(2 ** 32 + 1, 1, 1), one.expand(2 ** 32 + 1, 1, 1), v)
        with pytest.raises(ValueError, match="columns"):
            call(one, one.expand(1, 1, 2 ** 20 + 1), one.expand(1, 1, 2 ** 20 + 1), one, v)


@pytest.mark.parametrize("call,bad", [
    (_scan, dict(B=2 ** 31 - 1, D=64)),              # more threads than a launch counts
    (_step, dict(B=2 ** 31 - 1, D=64)),
    (_add, dict(B=2 ** 31 - 1)), (_add_backward, dict(B=2 ** 27, n=1 << 62)),
])
def test_launches_beyond_32_bits_are_refused(call, bad):
    from tts_amd import _lib
    lib = _lib.load()
    assert call(lib, **bad) == _lib.ERR_ARG
    assert "too many" in lib.ttsx_last_error_string().decode()


def test_an_empty_batch_takes_empty_lists():
    from tts_amd._seq import lengths_on, voices_on
    like = torch.zeros(1)
    assert lengths_on("f", [], 0, 5, like).shape == voices_on("f", [], 0, 5, like).shape == (0,)
    with pytest.raises(ValueError):
        lengths_on("f", 3, 1, 5, like)


def test_the_native_way_takes_ordinary_calls_only():
    """Anything else comes back as None, to be checked in Python; nothing of these reaches a GPU."""
    from tts_amd import _seq, _seqcalls
    _seq._bind()
    assert _seq.ways.ordinary is _seqcalls
    t, s = torch.zeros(2, 5, 8), torch.zeros(2, 8)
    v = torch.zeros(2, dtype=torch.int32)
    for args in ((t[:, 0], t[:, 0], s, None), (1, 2, 3, None), (None,) * 4):
        assert _seqcalls.step(*args) is None
    assert _seqcalls.scan(t, t, None, None, False, True) is None and _seqcalls.scan(t, t, s, [1, 2], False, True) is None
    assert _seqcalls.scan_backward(t, t, t, t, None, None, False) is None
    assert _seqcalls.adapter_add(t, t, t, t, v, None, None, None) is None
    assert _seqcalls.adapter_backward(t, t, t, t, [0, 1], None, None) is None
    for call, n in ((_seqcalls.step, 4), (_seqcalls.scan, 6), (_seqcalls.scan_backward, 7), (_seqcalls.adapter_add, 8),
                    (_seqcalls.adapter_backward, 7), (_seqcalls.bind, 7)):
        with pytest.raises(TypeError):
            call(*[None] * (n + 1))
    with pytest.raises(TypeError):
        _seqcalls.bind(*["x"] * 7)
