"""Refusals of the sequence operators that need no GPU: the checks in Python come before the place of the tensors."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad


def test_a_tangent_is_refused():
    from tts_amd import _lib
    from tts_amd.adapters import adapter_add
    from tts_amd.recurrence import gated_scan, gated_step
    x, m, v = torch.zeros(2, 5, 8), torch.zeros(2, 4, 8), torch.zeros(2, dtype=torch.int32)
    with forward_ad.dual_level():
        d, dh = forward_ad.make_dual(x, torch.ones_like(x)), forward_ad.make_dual(x[:, 0].clone(), torch.ones(2, 8))
        for call in (lambda: gated_scan(d, x), lambda: gated_scan(x, x, h0=dh), lambda: gated_step(x[:, 0], x[:, 0], dh),
                     lambda: adapter_add(x, d, m, m, v)):
            with torch.no_grad(), pytest.raises(ValueError, match="tangent"):
                call()
        with pytest.raises(_lib.TtsxError, match="no CPU path"):
            gated_scan(forward_ad.unpack_dual(d).primal, x)
    with pytest.raises(_lib.TtsxError, match="no CPU path"):
        gated_scan(d, x)


def test_a_negated_view_is_refused():
    from tts_amd.recurrence import gated_scan
    x, neg = torch.zeros(2, 5, 8), torch.zeros(2, 5, 8, dtype=torch.complex64).conj().imag
    for args in ((neg, x), (x, neg)):
        with pytest.raises(ValueError, match="resolve_neg"):
            gated_scan(*args)
