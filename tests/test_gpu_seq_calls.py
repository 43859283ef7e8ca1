"""The two ways into a sequence operator on the GPU: calls made natively and calls checked in Python give the same results,
and what the native way does not take is converted or refused as before."""
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


class _Counted:
    """The native way, noting whether it took the call."""

    def __init__(self, native):
        self.native, self.taken = native, []

    def __getattr__(self, name):
        def call(*args):
            done = getattr(self.native, name)(*args)
            self.taken.append(done is not None)
            return done
        return call


@pytest.fixture
def both(monkeypatch):
    """Runs a call both ways; returns the results and whether the native way took it."""
    from tts_amd import _seq, _seqcalls
    _seq._bind()

    def run(f):
        counted = _Counted(_seqcalls)
        monkeypatch.setattr(_seq.ways, "ordinary", counted)
        first = f()
        monkeypatch.setattr(_seq.ways, "ordinary", _seq._Unbound)
        second = f()
        monkeypatch.setattr(_seq.ways, "ordinary", _seqcalls)
        first, second = ((t,) if isinstance(t, torch.Tensor) else t for t in (first, second))
        assert len(first) == len(second)
        for a, b in zip(first, second):
            assert a.dtype == b.dtype and a.shape == b.shape and a.stride() == b.stride() and torch.equal(a, b)
        assert len(counted.taken) == 1
        return counted.taken[0]
    return run


def _rand(*shape, dtype=torch.float32, seed=1):
    return torch.randn(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_the_recurrence_both_ways(both, dtype):
    from tts_amd.recurrence import gated_scan, gated_scan_backward, gated_step
    B, T, D = 3, 900, 24
    z = _rand(B, T, 2 * D, dtype=dtype)
    x, g, h0 = z[..., :D], z[..., D:], _rand(B, D)
    lengths = torch.tensor([900, 0, 77], dtype=torch.int32, device="cuda")
    assert both(lambda: gated_scan(x, g))
    assert both(lambda: gated_scan(x, g, h0=h0, lengths=lengths, reverse=True, save_states=True))
    _, _, states = gated_scan(x, g, h0=h0, lengths=lengths, save_states=True)
    dh, last = _rand(B, T, D, dtype=dtype, seed=2), _rand(B, D, seed=3)
    assert both(lambda: gated_scan_backward(dh, x, g, states, lengths=lengths))
    assert both(lambda: gated_scan_backward(dh, x, g, states, dh_last=last, lengths=lengths, reverse=True))
    assert both(lambda: gated_step(x[:, 0], g[:, 0], h0))
    assert both(lambda: (lambda h: (*gated_step(x[:, 0], g[:, 0], h, out=h), h))(h0.clone()))
    assert both(lambda: gated_scan(torch.nn.Parameter(x, requires_grad=False), g))
    # not ordinary, and still the same
    assert not both(lambda: gated_scan(x, g, lengths=[900, 0, 77]))
    assert not both(lambda: gated_scan(x, g, lengths=lengths.long()))
    assert not both(lambda: gated_scan(x.transpose(1, 2).contiguous().transpose(1, 2), g))
    assert not both(lambda: gated_scan(x, g, h0=h0.t().contiguous().t()))
    assert not both(lambda: gated_scan(x[:, :0], g[:, :0], h0=h0))
    assert not both(lambda: gated_step(x[:, 0], g[:, 0], h0, out=torch.empty_like(h0)))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_the_adapters_both_ways(both, dtype):
    from tts_amd.adapters import adapter_add, adapter_backward
    B, T, K, N, R, V = 3, 40, 33, 70, 5, 2
    y, x = _rand(B, T, N, dtype=dtype), _rand(B, T, K, dtype=dtype, seed=2)
    down, up, scale = _rand(V, R, K, dtype=dtype, seed=3), _rand(V, R, N, dtype=dtype, seed=4), _rand(V, seed=5)
    voices, lengths = (torch.tensor(t, dtype=torch.int32, device="cuda") for t in ([1, -1, 0], [40, 3, 17]))
    for call in (adapter_add, adapter_backward):
        assert both(lambda: call(y, x, down, up, voices))
        assert both(lambda: call(y, x, down, up, voices, scale=scale, lengths=lengths))
        assert both(lambda: call(y[:, 0], x[:, 0], down, up, voices, scale=scale))
        assert both(lambda: call(y.transpose(0, 1).contiguous().transpose(0, 1), x, down, up, voices))
        assert not both(lambda: call(y, x, down, up, [1, -1, 0]))
        assert not both(lambda: call(y, x, down, up, voices, lengths=[40, 3, 17]))
        assert not both(lambda: call(y, x.transpose(1, 2).contiguous().transpose(1, 2), down, up, voices))
        assert not both(lambda: call(y[:0], x[:0], down, up, voices[:0]))
    assert both(lambda: (lambda o: adapter_add(o, x, down, up, voices, lengths=lengths, out=o))(y.clone()))
    assert both(lambda: (lambda o: adapter_add(o, x[:, 0], down, up, voices, out=o))(y[:, 0].clone()))
    assert not both(lambda: adapter_add(y, x, down, up, voices, out=torch.empty_like(y)))
    buf = torch.cat([x, y], -1)
    assert not both(lambda: (lambda o: adapter_add(o[..., K:], o[..., :K], down, up, voices, out=o[..., K:]))(buf.clone()))


def test_refusals_do_not_depend_on_the_way():
    from tts_amd import _lib, _seq
    from tts_amd.adapters import adapter_add
    from tts_amd.recurrence import gated_scan, gated_step
    _seq._bind()
    x, h = _rand(2, 5, 8), _rand(2, 8)
    for f, error in (
            (lambda: gated_scan(x, x[:, :4]), ValueError), (lambda: gated_scan(x, x.half()), ValueError),
            (lambda: gated_scan(x, x.cpu()), _lib.TtsxError), (lambda: gated_scan(x, None), ValueError),
            (lambda: gated_scan(x.clone().requires_grad_(), x), ValueError),
            (lambda: gated_scan(x, x, h0=h.half()), ValueError),
            (lambda: gated_scan(x, x, lengths=torch.zeros(3, dtype=torch.int32, device="cuda")), ValueError),
            (lambda: gated_step(x[:, 0], x[:, 0], h.double()), ValueError),
            (lambda: gated_step(h, h, h, out=h), ValueError),
            (lambda: adapter_add(x, x, x, x, torch.zeros(3, dtype=torch.int32, device="cuda")), ValueError),
            (lambda: adapter_add(x, x, x[:, :0], x[:, :0], torch.zeros(2, dtype=torch.int32, device="cuda")), ValueError),
            (lambda: adapter_add(x, x, x.clone(), x.clone(), torch.zeros(2, dtype=torch.int32, device="cuda"), out=x), ValueError)):
        with pytest.raises(error):
            f()
    with torch.no_grad():                                       # allowed there, as the documentation says
        gated_scan(x.clone().requires_grad_(), x)
