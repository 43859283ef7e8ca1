"""Inputs that an operator takes or refuses: a single row with a far stride, tangents of forward-mode differentiation, negated views,
results placed over indices."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _rand(*shape, seed=1, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(dtype)


@pytest.fixture(params=["native", "python"])
def way(request, monkeypatch):
    from tts_amd import _seq
    _seq._bind()
    if request.param == "python":
        monkeypatch.setattr(_seq.ways, "ordinary", _seq._Unbound)
    return request.param


def _far(t):
    """The same [B,1,n] with a row stride beyond 2^20: there is no second row for it to lead to."""
    buf = torch.zeros(t.shape[0], t.shape[2], device="cuda", dtype=t.dtype)
    out = buf.as_strided(t.shape, (t.shape[2], 3 << 20, 1))
    out.copy_(t)
    return out


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("B", [1, 3])
def test_a_single_row_lies_anywhere(B, dtype, way):
    from tts_amd.adapters import adapter_add, adapter_backward
    from tts_amd.recurrence import gated_scan, gated_scan_backward
    x, g, dh = (_rand(B, 1, 24, seed=k, dtype=dtype) for k in range(3))
    want = gated_scan(x, g, save_states=True)
    grads = gated_scan_backward(dh, x, g, want[2])
    assert all(torch.equal(a, b) for a, b in zip(want, gated_scan(_far(x), _far(g), save_states=True)))
    assert all(torch.equal(a, b) for a, b in zip(grads, gated_scan_backward(_far(dh), _far(x), _far(g), want[2])))
    m, voices = _rand(2, 5, 24, seed=4, dtype=dtype), torch.zeros(B, dtype=torch.int32, device="cuda")
    out, grads = adapter_add(g, x, m, m, voices), adapter_backward(g, x, m, m, voices)
    assert torch.equal(adapter_add(_far(g), _far(x), m, m, voices), out)
    assert all(torch.equal(a, b) for a, b in zip(grads, adapter_backward(_far(g), _far(x), m, m, voices)))
    here = _far(g)
    assert adapter_add(here, _far(x), m, m, voices, out=here) is here and torch.equal(here, out)
    there = _far(x)
    assert adapter_add(g, x, m, m, voices, out=there) is there and torch.equal(there, out)


def test_a_tangent_is_refused(way):
    """The calls give no tangent: an input that carries one is refused as one that requires grad is, with no_grad() too, which
    leaves forward mode as it is; inside a dual level without tangents nothing changes."""
    from tts_amd.adapters import adapter_add, adapter_backward
    from tts_amd.recurrence import gated_scan, gated_scan_backward, gated_step
    x, m, voices = _rand(2, 5, 8), _rand(2, 4, 8), torch.zeros(2, dtype=torch.int32, device="cuda")
    h, states = _rand(2, 8), _rand(2, 1, 8)
    scale = torch.ones(2, device="cuda")
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, torch.ones_like(x))
        dh, dm = forward_ad.make_dual(h, torch.ones_like(h)), forward_ad.make_dual(m, torch.ones_like(m))
        ds = forward_ad.make_dual(scale, torch.ones_like(scale))
        calls = [lambda: gated_scan(d, x), lambda: gated_scan(x, d), lambda: gated_scan(x, x, h0=dh),
                 lambda: gated_scan_backward(d, x, x, states), lambda: gated_scan_backward(x, x, x, states, dh_last=dh),
                 lambda: gated_step(x[:, 0], x[:, 0], dh), lambda: gated_step(d[:, 0], x[:, 0], h),
                 lambda: adapter_add(d, x, m, m, voices), lambda: adapter_add(x, x, m, dm, voices),
                 lambda: adapter_add(x, x, m, m, voices, scale=ds), lambda: adapter_backward(x, d, m, m, voices)]
        for call in calls:
            with pytest.raises(ValueError, match="tangent"):
                call()
            with torch.no_grad(), pytest.raises(ValueError, match="tangent"):
                call()
        want = gated_scan(x, x)
        primal = forward_ad.unpack_dual(d).primal
        assert all(torch.equal(a, b) for a, b in zip(want, gated_scan(primal, x)))
    assert all(torch.equal(a, b) for a, b in zip(want, gated_scan(x, x)))


def test_a_negated_view_is_refused(way):
    """The imaginary part of a conjugate is a view with its sign in a flag, which a kernel would not see."""
    from tts_amd.adapters import adapter_add, adapter_backward
    from tts_amd.recurrence import gated_scan, gated_scan_backward, gated_step
    z = torch.randn(2, 5, 8, dtype=torch.complex64, device="cuda")
    neg = z.conj().imag
    assert neg.is_neg()
    x, m, voices, states = _rand(2, 5, 8), _rand(2, 4, 8), torch.zeros(2, dtype=torch.int32, device="cuda"), _rand(2, 1, 8)
    for call in (lambda: gated_scan(neg, x), lambda: gated_scan(x, x, h0=neg[:, 0]), lambda: gated_step(x[:, 0], neg[:, 0], x[:, 1]),
                 lambda: gated_scan_backward(neg, x, x, states), lambda: gated_scan_backward(x, x, x, neg[:, :1]),
                 lambda: adapter_add(x, neg, m, m, voices), lambda: adapter_backward(neg, x, m, m, voices),
                 lambda: adapter_add(x, x, m, m, voices, scale=neg[:, 0, 0])):
        with pytest.raises(ValueError, match="resolve_neg"):
            call()
    assert all(torch.equal(a, b) for a, b in zip(gated_scan(neg.resolve_neg(), x), gated_scan(-z.imag, x)))


def test_a_result_over_the_indices_is_refused(way):
    """voices and lengths are read while out is written."""
    from tts_amd.adapters import adapter_add
    x, m = _rand(2, 1, 8), _rand(2, 4, 8)
    buf = torch.zeros(64, dtype=torch.int32, device="cuda")
    out = buf[:16].view(torch.float32).view(2, 1, 8)
    index = buf[14:16]
    with pytest.raises(ValueError, match="out overlaps voices"):
        adapter_add(x, x, m, m, index, out=out)
    with pytest.raises(ValueError, match="out overlaps voices"):
        adapter_add(out, x, m, m, index, out=out)
    with pytest.raises(ValueError, match="out overlaps lengths"):
        adapter_add(x, x, m, m, buf[32:34], lengths=index, out=out)
    assert adapter_add(out, x, m, m, buf[32:34], lengths=buf[34:36], out=out) is out
    with pytest.raises(ValueError, match="out overlaps voices"):
        adapter_add(x, x, m, m, buf[8:12].view(torch.int64), out=out)
