"""Views that an operator takes: a single row with a far stride."""
import pytest
import torch

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
