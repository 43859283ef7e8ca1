"""The gate of the recurrence on the GPU, relative to its own size: w = sigmoid(-g) over all logits.

Bounds in units F32 = 2^-24 of the value (half a unit in the last place).  The hardware's exponential and reciprocal are
off by one unit in the last place, 2 F32 each.  fp32: e = e^g is the exponential, one fused product (1), and a remainder
that is exact to second order: 3.  16-bit logits: 2 + 1, and what the correction leaves out, the second order of bf16's, (85 x
4.89e-6)^2 / 2 = 1.5 F32 at the farthest logits here, or the third of fp16's, (85 x 4.72e-5)^3 / 6 = 0.2: 5.  w = 1 / (1 + e): e's error, the sum's 1, the reciprocal's 2: 6 and 8."""
import pytest
import torch

from seq_ref import F32

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
W_UNITS = {torch.float32: 6, torch.bfloat16: 8, torch.float16: 8}


def _logits(dtype, low=-85.0, high=85.0):
    """Evenly over the range where w is a normal number, and more of them around zero."""
    g = torch.cat([torch.linspace(low, high, 40001), torch.linspace(-20, 20, 40001)]).to(dtype)
    return g.clamp(low, high)


def _off(got, want, units):
    """How far the worst element is beyond that many units of its own size (a number at or below 0 passes)."""
    want = want.double()
    return float(((got.double().cpu() - want).abs() / want.abs() / F32).max()) - units


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_the_written_share(dtype):
    """h0 = 0 and x = 1: the state is w itself."""
    from tts_amd.recurrence import gated_scan, gated_step
    g = _logits(dtype)[None]
    w = 1 / (1 + torch.exp(g.double()))
    one, zero = torch.ones_like(g).cuda(), torch.zeros(g.shape, device="cuda")
    _, h = gated_step(one, g.cuda(), zero)
    assert _off(h, w, W_UNITS[dtype]) <= 0
    assert torch.equal(gated_scan(one[:, None], g.cuda()[:, None])[1], h)
