"""Infinite weights and activations of the adapters: infinity, its sign and NaN are those of the formula, and what no infinity enters
is as it was to the bit."""
import pytest
import torch

import seq_ref

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
INF = float("inf")
# few tiles, a tile to a CU, many; every class of ranks
SIZES = [(1, 40, 32, 150, 5), (2, 33, 40, 70, 16), (3, 20, 24, 136, 30), (2, 50, 40, 96, 61), (150, 130, 24, 72, 16),
         (140, 150, 24, 40, 33)]


def _inputs(B, T, K, N, R, dtype):
    gen = torch.Generator().manual_seed(B + T + R)
    y, x = (torch.randn(B, T, n, generator=gen).to(dtype) for n in (N, K))
    down, up = (torch.randn(2, R, n, generator=gen).to(dtype) for n in (K, N))
    return y, x, down, up, (torch.arange(B) % 2).int(), 0.5 + torch.rand(2, generator=gen)


def _same(got, clean, want):
    """Infinities and NaN of the formula; every other element as without them."""
    got, clean = got.cpu(), clean.cpu()
    wild = ~torch.isfinite(want)
    assert bool(wild.any()) and not bool(wild.all())
    assert torch.equal(~torch.isfinite(got), wild)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got[wild].double().nan_to_num(0.0), want[wild].nan_to_num(0.0))
    assert torch.equal(got[~wild], clean[~wild])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_infinite_weights(size, dtype):
    from tts_amd.adapters import adapter_add, adapter_backward
    y, x, down, up, voices, scale = _inputs(*size, dtype)
    x[0, 5] = 0.0                                                     # u of this row is zero: 0 x infinity
    kw = dict(scale=scale.cuda())
    gy, gx, gd, gu, gv = (t.cuda() for t in (y, x, down, up, voices))
    out, dx = adapter_add(gy, gx, gd, gu, gv, **kw), adapter_backward(gx, gy, gu, gd, gv, **kw)[0]
    up[0, 2, 7], up[0, 0, -1], up[0, 3, -1], up[-1, 1, 20] = INF, -INF, INF, float("nan")
    want, _ = seq_ref.adapter(y, x, down, up, voices, scale)
    _same(adapter_add(gy, gx, gd, up.cuda(), gv, **kw), out, want)
    # the same product as the gradient of the activations, with the two matrices swapped
    want = seq_ref.adapter_backward(x, y, up, down, voices, scale)[0][0]
    _same(adapter_backward(gx, gy, up.cuda(), gd, gv, **kw)[0], dx, want)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_infinite_activations(size, dtype):
    from tts_amd.adapters import adapter_add, adapter_backward
    y, x, down, up, voices, scale = _inputs(*size, dtype)
    kw = dict(scale=scale.cuda())
    gy, gx, gd, gu, gv = (t.cuda() for t in (y, x, down, up, voices))
    out, clean = adapter_add(gy, gx, gd, gu, gv, **kw), adapter_backward(gy, gx, gd, gu, gv, **kw)
    x[0, 3, 9] = INF
    want, _ = seq_ref.adapter(y, x, down, up, voices, scale)
    _same(adapter_add(gy, x.cuda(), gd, gu, gv, **kw), out, want)
    got, want = adapter_backward(gy, x.cuda(), gd, gu, gv, **kw), seq_ref.adapter_backward(y, x, down, up, voices, scale)
    assert torch.equal(got[0], clean[0])                              # dx does not depend on x
    _same(got[1], clean[1], want[1][0])
    if size[0] > 1:
        _same(got[2], clean[2], want[2][0])                           # a whole voice
    dy = y.clone()
    dy[0, 2, 4] = -INF
    got, want = adapter_backward(dy.cuda(), gx, gd, gu, gv, **kw), seq_ref.adapter_backward(dy, x.nan_to_num(posinf=0.0), down, up,
                                                                                            voices, scale)
    _same(got[0], clean[0], want[0][0])
    _same(got[2], clean[2], want[2][0])
