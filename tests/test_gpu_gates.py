"""The gate of the recurrence on the GPU, relative to its own size: w = sigmoid(-g) and f = sigmoid(g) over all
logits.

Bounds in units F32 = 2^-24 of the value (half a unit in the last place).  The hardware's exponential and reciprocal are
off by one unit in the last place, 2 F32 each.  fp32: e = e^g is the exponential, one fused product (1), and a remainder
that is exact to second order: 3.  16-bit logits: 2 + 1, and what the correction leaves out, the second order of bf16's, (85 x
4.89e-6)^2 / 2 = 1.5 F32 at the farthest logits here, or the third of fp16's, (85 x 4.72e-5)^3 / 6 = 0.2: 5.  w = 1 / (1 + e): e's error, the sum's 1, the reciprocal's 2: 6 and 8.
f = e w below a half (e < 1, where 1 + e has half of e's error at most): e's own, half of it again, 3 of w and 1 of the
product: 9 and 12; f = 1 - w above, where w is the smaller: w's and 1."""
import pytest
import torch

from seq_ref import F32

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
W_UNITS = {torch.float32: 6, torch.bfloat16: 8, torch.float16: 8}
F_UNITS = {torch.float32: 9, torch.bfloat16: 12, torch.float16: 12}


def _logits(dtype, low=-85.0, high=85.0):
    """Evenly over the range where f and w are normal numbers, and more of them around zero."""
    g = torch.cat([torch.linspace(low, high, 40001), torch.linspace(-20, 20, 40001)]).to(dtype)
    return g.clamp(low, high)


def _off(got, want, units):
    """How far the worst element is beyond that many units of its own size (a number at or below 0 passes)."""
    want = want.double()
    return float(((got.double().cpu() - want).abs() / want.abs() / F32).max()) - units


def _gates(g):
    return 1 / (1 + torch.exp(-g.double())), 1 / (1 + torch.exp(g.double()))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_the_written_share(dtype):
    """h0 = 0 and x = 1: the state is w itself."""
    from tts_amd.recurrence import gated_scan, gated_step
    g = _logits(dtype)[None]
    _, w = _gates(g)
    one, zero = torch.ones_like(g).cuda(), torch.zeros(g.shape, device="cuda")
    _, h = gated_step(one, g.cuda(), zero)
    assert _off(h, w, W_UNITS[dtype]) <= 0
    assert torch.equal(gated_scan(one[:, None], g.cuda()[:, None])[1], h)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_the_kept_share(dtype):
    """h0 = 1 and x = 0: the state is f itself, and so is the gradient of h0; that of x is w."""
    from tts_amd.recurrence import gated_scan, gated_scan_backward, gated_step
    g = _logits(dtype)[None]
    f, w = _gates(g)
    zero, one = torch.zeros_like(g).cuda(), torch.ones(g.shape, device="cuda")
    _, h = gated_step(zero, g.cuda(), one)
    assert _off(h, f, F_UNITS[dtype]) <= 0
    for n in (g.shape[1], g.shape[1] - 1):      # lanes of several channels and of one
        z, gn = zero[:, None, :n], g.cuda()[:, None, :n]
        _, last, states = gated_scan(z, gn, h0=one[:, :n], save_states=True)
        assert torch.equal(last, h[:, :n])
        dx, dg, dh0 = gated_scan_backward(z, z, gn, states, dh_last=one[:, :n])
        assert _off(dh0, f[:, :n], F_UNITS[dtype]) <= 0
        if dtype == torch.float32:              # the 16-bit types round dx and dg
            assert _off(dx[:, 0], w[:, :n], W_UNITS[dtype]) <= 0
            assert _off(dg[:, 0], (f * w)[:, :n], F_UNITS[dtype] + W_UNITS[dtype] + 1) <= 0


def _memory(T, D, dtype, seed):
    """Long memories with a few steps that forget almost everything."""
    gen = torch.Generator().manual_seed(seed)
    g = 9 + 3 * torch.rand(1, T, D, generator=gen)
    for t, low in ((T // 5, -14.0), (T // 2, -9.0), (T - 3, -17.0)):
        g[:, t] = low - torch.rand(D, generator=gen)
    return g.to(dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("T,D", [(7, 40), (300, 33), (1000, 64), (6000, 12)], ids=str)
def test_a_state_that_nothing_enters(T, D, dtype):
    """x = 0: the last state is the product of all f, and with dh = 0 the gradient of h0 is that of dh_last.  A product of T
    factors carries each one's error and a rounding of its own."""
    from tts_amd.recurrence import gated_scan, gated_scan_backward
    g = _memory(T, D, dtype, T)
    f, _ = _gates(g)
    zero, one = torch.zeros_like(g).cuda(), torch.ones(1, D, device="cuda")
    for reverse in (False, True):
        _, last, states = gated_scan(zero, g.cuda(), h0=one, reverse=reverse, save_states=True)
        assert _off(last, f.prod(1), T * (F_UNITS[dtype] + 1)) <= 0
        _, _, dh0 = gated_scan_backward(zero, zero, g.cuda(), states, dh_last=one, reverse=reverse)
        assert _off(dh0, f.prod(1), T * (F_UNITS[dtype] + 1)) <= 0
