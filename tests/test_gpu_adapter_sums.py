"""The hidden values u = x A^T between the adapters' two products are fp32: where the second sum cancels what they have in
common, their last digits are the result.

Every case has pairs of terms of the second sum with opposite signs whose hidden values differ in one input of one step of the
16-bit type: about 2^-11 of u is left, rounded to the type at 2^-20 of u, beside 2^-17 of u that a sum of two bf16 numbers
would lose.  (In fp32 one step of one input is less than what the first sum itself may be off by: nothing would be shown.)"""
import pytest
import torch

import seq_ref
from seq_ref import half_step

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16]
# what u may lose on its way from one product to the next, of the row's largest
LOSS = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -23}


def _rounding(dtype, want):
    return half_step(dtype) * want.abs() + (2.0 ** -25 if dtype == torch.float16 else 0.0)


def _near(t, dtype):
    """t, and t with one element of each last axis moved by one step of the type."""
    t = t.to(dtype)
    other = t.clone()
    other[..., 3] *= 1 + torch.finfo(dtype).eps
    return t, other


def _pairs(a, b, axis):
    """a and b in turn along an axis of their own length twice."""
    return torch.stack([a, b], axis + 1).flatten(axis, axis + 1)


def _check(got, want):
    for g, (w, tol) in zip(got, want):
        limit = tol * (1 + half_step(g.dtype)) + _rounding(g.dtype, w)
        assert float(((g.cpu().double() - w).abs() - limit).max()) <= 0
        assert bool((limit < w.abs()).any())                       # the limit tells the result from nothing


# few tiles and many, every class of ranks
SIZES = [(2, 40, 8, 160, 4), (3, 33, 16, 130, 30), (2, 50, 8, 96, 64), (160, 128, 8, 136, 6), (160, 128, 8, 40, 24),
         (140, 140, 8, 40, 48)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_ranks_that_cancel(size, dtype, monkeypatch):
    from tts_amd.adapters import adapter_add, adapter_backward
    monkeypatch.setattr(seq_ref, "SPLIT", LOSS)
    B, T, K, N, R = size
    gen = torch.Generator().manual_seed(B + R)
    voices = (torch.arange(B) % 2).int()
    x = (1 + torch.rand(B, T, K, generator=gen)).to(dtype)
    down = _pairs(*_near(1 + torch.rand(2, R // 2, K, generator=gen), dtype), 1)
    up = torch.randn(2, R // 2, N, generator=gen).to(dtype)
    up = _pairs(up, -up, 1)
    y = torch.zeros(B, T, N, dtype=dtype)
    want = seq_ref.adapter(y, x, down, up, voices)
    args = [t.cuda() for t in (y, x, down, up, voices)]
    _check([adapter_add(*args)], [want])
    # the same for dx, with dy in the place of x
    args = [t.cuda() for t in (x, y, up, down, voices)]
    want = seq_ref.adapter_backward(x, y, up, down, voices)[0]
    _check([adapter_backward(*args)[0]], [want])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("size", [(2, 2, 8, 160, 4), (3, 2, 16, 130, 30), (2, 2, 8, 96, 64)], ids=str)
def test_rows_that_cancel(size, dtype, monkeypatch):
    """The weights' gradients of two rows: dy of opposite signs under hidden values that are near, and x under near du."""
    from tts_amd.adapters import adapter_backward
    monkeypatch.setattr(seq_ref, "SPLIT", LOSS)
    B, T, K, N, R = size
    gen = torch.Generator().manual_seed(B + R)
    voices = torch.arange(B).int()
    x = _pairs(*_near(1 + torch.rand(B, 1, K, generator=gen), dtype), 1)
    dy = torch.randn(B, 1, N, generator=gen).to(dtype)
    dy = _pairs(dy, -dy, 1)
    down = (1 + torch.rand(B, R, K, generator=gen)).to(dtype)
    up = torch.zeros(B, R, N, dtype=dtype)
    _, _, dup = adapter_backward(*(t.cuda() for t in (dy, x, down, up, voices)))
    _check([dup], [seq_ref.adapter_backward(dy, x, down, up, voices)[2]])
    _, ddown, _ = adapter_backward(*(t.cuda() for t in (x, dy, up, down, voices)))
    _check([ddown], [seq_ref.adapter_backward(x, dy, up, down, voices)[1]])
