"""The gradients of the operators as they are used together: a shared projection, each request's voice beside it, the recurrence
over its two halves.  Every operator is held to its own bound on what the one before it left, and no limit lets a result of zero pass."""
import pytest
import torch

from seq_ref import F32, adapter, adapter_backward, half_step, scan, scan_backward, scan_error

pytestmark = pytest.mark.gpu


def _held(got, want, limit):
    assert float(((got.cpu().double() - want).abs() - limit).max()) <= 0
    live = want != 0
    assert float(limit[live].median()) < 0.05 * float(want[live].abs().median())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("reverse", [False, True])
def test_gradients_of_an_adapted_layer(dtype, reverse):
    from tts_amd.adapters import adapter_add
    from tts_amd.adapters import adapter_backward as add_backward
    from tts_amd.recurrence import gated_scan, gated_scan_backward
    gen = torch.Generator().manual_seed(3)
    B, T, K, D, R, V = 4, 90, 24, 20, 4, 3
    x = torch.randn(B, T, K, generator=gen).to(dtype)
    base = torch.randn(B, T, 2 * D, generator=gen).to(dtype)
    down, up = (torch.randn(V, R, K, generator=gen) / K ** 0.5).to(dtype), (torch.randn(V, R, 2 * D, generator=gen) / R ** 0.5).to(dtype)
    voices, lengths = torch.tensor([2, -1, 0, 2], dtype=torch.int32), torch.tensor([90, 41, 64, 1], dtype=torch.int32)
    dh = torch.randn(B, T, D, generator=gen).to(dtype)
    gx, gd, gu, gv, gl = (t.cuda() for t in (x, down, up, voices, lengths))
    small = 2.0 ** -25 if dtype == torch.float16 else 0.0

    both = adapter_add(base.cuda(), gx, gd, gu, gv, lengths=gl)
    want, tol = adapter(base, x, down, up, voices, None, lengths)
    _held(both, want, tol * (1 + half_step(dtype)) + half_step(dtype) * want.abs() + small)

    v, g = both[..., :D], both[..., D:]
    h, last, states = gated_scan(v, g, lengths=gl, reverse=reverse, save_states=True)
    cv, cg = v.cpu(), g.cpu()
    want_h, _, _ = scan(cv, cg, None, lengths, reverse)
    eh = scan_error(cv, cg, None, T, lengths)
    _held(h, want_h, eh + half_step(dtype) * want_h.abs() + small)

    dx, dg, dh0 = gated_scan_backward(dh.cuda(), v, g, states, lengths=gl, reverse=reverse)
    wx, wg, w0, G, before = scan_backward(dh, cv, cg, None, None, lengths, reverse)
    # G runs through the maps of the state with dh in the place of w x: the same bound on its own largest value
    live = (torch.arange(T)[None, :] < lengths[:, None])[:, :, None]
    logits = torch.where(live, cg.double(), 0.0)
    eG = 16 * F32 * float(G.abs().max()) * min(T, 1 + float(torch.exp(logits.max())))
    f, w = torch.sigmoid(logits), torch.sigmoid(-logits)
    diff = (before - cv.double()).abs()
    own = 16 * F32 * (1 + logits.abs()) * G.abs()
    _held(dx, wx, torch.where(live, half_step(dtype) * wx.abs() + small + w * (eG + own), 0.0))
    _held(dg, wg, torch.where(live, half_step(dtype) * wg.abs() + small + f * w * (eh * G.abs() + diff * eG + own * diff), 0.0))
    _held(dh0, w0, torch.full_like(w0, eG))

    d = torch.cat([dx, dg], -1)
    got = add_backward(d, gx, gd, gu, gv, lengths=gl)
    for a, (want, tol) in zip(got, adapter_backward(d.cpu(), x, down, up, voices, lengths=lengths)):
        _held(a, want, torch.where((want != 0) | (tol > 0), tol * (1 + half_step(dtype)) + half_step(dtype) * want.abs() + small, 0.0))
