"""Low-rank adapters of many voices on the GPU against their formulas in float64: types, odd sizes, every rank class,
ragged and empty requests, requests without a voice, strides, places, gradients, streams and graphs."""
import pytest
import torch

from seq_ref import F32, adapter, adapter_backward, half_step, scan, scan_backward

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
#        B   T    K     N    R   V
SIZES = [(1, 1, 1, 1, 1, 1), (2, 1, 64, 96, 4, 3), (64, 1, 129, 260, 16, 5), (3, 31, 40, 136, 8, 2),
         (2, 32, 256, 1025, 16, 2), (5, 33, 17, 65, 17, 9), (4, 65, 512, 80, 32, 3), (1, 100, 80, 512, 33, 1),
         (3, 130, 1025, 256, 64, 2), (9, 70, 48, 72, 5, 4), (2, 257, 96, 300, 61, 2)]


def _inputs(B, T, K, N, R, V, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    wide = torch.randn(B, T, N, generator=gen).to(dtype)
    x = torch.randn(B, T, K, generator=gen).to(dtype)
    down = (torch.randn(V, R, K, generator=gen) / K ** 0.5).to(dtype)
    up = (torch.randn(V, R, N, generator=gen) / R ** 0.5).to(dtype)
    voices = torch.randint(-1, V, (B,), generator=gen, dtype=torch.int32)
    scale = torch.randn(V, generator=gen)
    lengths = None
    if B > 1 and T > 1:
        lengths = torch.randint(0, T + 1, (B,), generator=gen, dtype=torch.int32)
        lengths[0] = T
        if B > 2:
            lengths[1], lengths[2] = 0, 1
    if B > 2:
        voices[0], voices[2] = V - 1, 0
    else:
        voices[0] = V - 1
    return wide, x, down, up, voices, scale, lengths


def _cuda(*tensors):
    return [None if t is None else t.cuda() for t in tensors]


def _excess(got, want, tol):
    return float(((got.cpu().double() - want).abs() - tol).max())


def _rounding(dtype, want):
    return half_step(dtype) * want.abs() + (2.0 ** -25 if dtype == torch.float16 else 0.0)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_add_matches_the_formula(size, dtype):
    from tts_amd.adapters import adapter_add
    y, x, down, up, voices, scale, lengths = _inputs(*size, dtype, sum(size))
    want, tol = adapter(y, x, down, up, voices, scale, lengths)
    gy, gx, gd, gu, gv, gs, gl = _cuda(y, x, down, up, voices, scale, lengths)
    out = adapter_add(gy, gx, gd, gu, gv, scale=gs, lengths=gl)
    assert out.dtype == dtype and torch.equal(gy.cpu(), y)
    assert _excess(out, want, tol * (1 + half_step(dtype)) + _rounding(dtype, want)) <= 0
    same = adapter_add(gy, gx, gd, gu, gv, scale=gs, lengths=gl, out=gy)      # in place
    assert same is gy and torch.equal(gy, out)
    for b in range(size[0]):   # rows without an adapter are y's, to the bit
        n = 0 if int(voices[b]) < 0 else size[1] if lengths is None else int(lengths[b])
        assert torch.equal(out[b, n:].cpu(), y[b, n:])
    want, tol = adapter(y, x, down, up, voices)
    out = adapter_add(y.cuda(), gx, gd, gu, voices.tolist())                  # no scale, no lengths, voices on the host
    assert _excess(out, want, tol * (1 + half_step(dtype)) + _rounding(dtype, want)) <= 0


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("size", [(260, 130, 24, 40, 5, 7), (200, 190, 72, 136, 20, 3), (150, 250, 40, 65, 40, 11)], ids=str)
def test_many_requests(size, dtype):
    """Batches that fill the chip take their rows in larger tiles."""
    from tts_amd.adapters import adapter_add
    y, x, down, up, voices, scale, lengths = _inputs(*size, dtype, 7)
    want, tol = adapter(y, x, down, up, voices, scale, lengths)
    gy, gx, gd, gu, gv, gs, gl = _cuda(y, x, down, up, voices, scale, lengths)
    out = adapter_add(gy, gx, gd, gu, gv, scale=gs, lengths=gl)
    assert _excess(out, want, tol * (1 + half_step(dtype)) + _rounding(dtype, want)) <= 0
    assert torch.equal(adapter_add(gy, gx, gd, gu, gv, scale=gs, lengths=gl, out=gy), out)
    _check_backward(size, dtype, 8)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_single_positions(dtype):
    """[B,N] and [B,K] are the [B,1,.] call."""
    from tts_amd.adapters import adapter_add
    from tts_amd.adapters import adapter_backward as backward
    y, x, down, up, voices, scale, _ = _cuda(*_inputs(6, 1, 72, 130, 8, 3, dtype, 5))
    want = adapter_add(y, x, down, up, voices, scale=scale)
    assert torch.equal(adapter_add(y[:, 0], x[:, 0], down, up, voices, scale=scale), want[:, 0])
    state = y[:, 0].clone()
    assert adapter_add(state, x[:, 0], down, up, voices, scale=scale, out=state) is state and torch.equal(state, want[:, 0])
    a = backward(y, x, down, up, voices, scale=scale)
    b = backward(y[:, 0], x[:, 0], down, up, voices, scale=scale)
    assert torch.equal(a[0][:, 0], b[0]) and torch.equal(a[1], b[1]) and torch.equal(a[2], b[2])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_strides_and_slices(dtype):
    """y and x as slices of one buffer at odd offsets, time-major, and x repeated over the batch."""
    from tts_amd.adapters import adapter_add
    from tts_amd.adapters import adapter_backward as backward
    y, x, down, up, voices, scale, lengths = _cuda(*_inputs(3, 70, 40, 75, 9, 2, dtype, 6))
    want = adapter_add(y, x, down, up, voices, scale=scale, lengths=lengths)
    grads = backward(y, x, down, up, voices, scale=scale, lengths=lengths)
    buf = torch.zeros(3, 70, 40 + 75 + 6, device="cuda", dtype=dtype)
    buf[..., 1:41], buf[..., 44:119] = x, y
    before = buf.clone()
    assert torch.equal(adapter_add(buf[..., 44:119], buf[..., 1:41], down, up, voices, scale=scale, lengths=lengths), want)
    for a, b in zip(grads, backward(buf[..., 44:119], buf[..., 1:41], down, up, voices, scale=scale, lengths=lengths)):
        assert torch.equal(a, b)
    adapter_add(buf[..., 44:119], buf[..., 1:41], down, up, voices, scale=scale, lengths=lengths, out=buf[..., 44:119])
    assert torch.equal(buf[..., 44:119], want)
    buf[..., 44:119] = before[..., 44:119]
    assert torch.equal(buf, before)                                       # the columns beside it are as they were
    ty, tx = y.transpose(0, 1).contiguous().transpose(0, 1), x.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(adapter_add(ty, tx, down, up, voices, scale=scale, lengths=lengths, out=ty), want)
    cx = x.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(adapter_add(y, cx, down, up, voices, scale=scale, lengths=lengths), want)
    one = x[:1].expand(3, -1, -1)
    assert torch.equal(adapter_add(y, one, down, up, voices, scale=scale),
                       adapter_add(y, one.contiguous(), down, up, voices, scale=scale))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_rows_behind_the_end_are_not_read_or_written(dtype):
    from tts_amd.adapters import adapter_add
    from tts_amd.adapters import adapter_backward as backward
    y, x, down, up, _, scale, _ = _inputs(4, 50, 33, 70, 8, 2, dtype, 7)
    lengths, voices = torch.tensor([50, 0, 33, 7], dtype=torch.int32), torch.tensor([0, 1, 1, -1], dtype=torch.int32)
    results = []
    for fill in (0.0, float("nan"), float("inf")):
        dy = y.clone()
        for b, n in enumerate(lengths.tolist()):
            n = 0 if voices[b] < 0 else n
            x[b, n:], dy[b, n:] = fill, fill
        gy, gx, gd, gu, gv, gs, gl = _cuda(y, x, down, up, voices, scale, lengths)
        out = adapter_add(gy, gx, gd, gu, gv, scale=gs, lengths=gl)
        results.append([out, *backward(dy.cuda(), gx, gd, gu, gv, scale=gs, lengths=gl)])
        assert torch.equal(out[1].cpu(), y[1]) and torch.equal(out[3].cpu(), y[3])
        marked = gy.clone()
        marked[0, 20:] = 5.0
        adapter_add(marked, gx, gd, gu, gv, scale=gs, lengths=[20, 0, 0, 0], out=marked)
        assert bool((marked[0, 20:] == 5.0).all()) and torch.equal(marked[0, :20], out[0, :20])
    for other in results[1:]:
        for a, b in zip(results[0], other):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_infinities_stay_in_their_row(dtype):
    from tts_amd.adapters import adapter_add
    y, x, down, up, _, _, _ = _cuda(*_inputs(1, 40, 32, 64, 8, 1, dtype, 8))
    voices = torch.zeros(1, dtype=torch.int32, device="cuda")
    want = adapter_add(y, x, down, up, voices)
    x[0, 3, 5], x[0, 9, 1] = float("inf"), float("nan")
    got = adapter_add(y, x, down, up, voices)
    keep = torch.ones(40, dtype=torch.bool, device="cuda")
    keep[3] = keep[9] = False
    assert torch.equal(got[0, keep], want[0, keep])
    assert not torch.isfinite(got[0, 3]).any() and torch.isnan(got[0, 9]).all()


def test_large_and_small_hidden_values_of_fp16():
    """u beyond fp16's own range, and far below its smallest numbers, still gives the right sum."""
    from tts_amd.adapters import adapter_add
    for a, b in ((60000.0, 1e-4), (6e-5, 60.0)):
        y = torch.zeros(1, 4, 16)
        x = torch.full((1, 4, 64), a)
        down, up = torch.ones(1, 2, 64), torch.full((1, 2, 16), b)
        y, x, down, up = (t.half() for t in (y, x, down, up))
        want, tol = adapter(y, x, down, up, [0])
        out = adapter_add(*_cuda(y, x, down, up), [0])
        assert _excess(out, want, tol + _rounding(torch.float16, want)) <= 0 and bool((want > 0).all())


def test_voices_outside_the_table_have_no_adapter():
    from tts_amd.adapters import adapter_add
    from tts_amd.adapters import adapter_backward as backward
    y, x, down, up, _, _, _ = _cuda(*_inputs(4, 40, 32, 64, 8, 2, torch.float32, 9))
    wild = torch.tensor([0, -7, 2, 2 ** 31 - 1], device="cuda")
    tame = torch.tensor([0, -1, -1, -1], device="cuda")
    for t in (torch.int32, torch.int64):
        assert torch.equal(adapter_add(y, x, down, up, wild.to(t)), adapter_add(y, x, down, up, tame.to(t)))
        for a, b in zip(backward(y, x, down, up, wild.to(t)), backward(y, x, down, up, tame.to(t))):
            assert torch.equal(a, b)
    assert not backward(y, x, down, up, wild)[1][1].any()                   # a voice that no request has


def _check_backward(size, dtype, seed):
    from tts_amd.adapters import adapter_backward as kernel
    dy, x, down, up, voices, scale, lengths = _inputs(*size, dtype, seed)
    want = adapter_backward(dy, x, down, up, voices, scale, lengths)
    args = _cuda(dy, x, down, up, voices)
    kw = dict(zip(("scale", "lengths"), _cuda(scale, lengths)))
    got = kernel(*args, **kw)
    for g, (w, tol) in zip(got, want):
        assert g.dtype == dtype
        limit = tol * (1 + half_step(dtype)) + torch.where((w != 0) | (tol > 0), _rounding(dtype, w), 0.0)
        assert _excess(g, w, limit) <= 0
    for a, b in zip(got, kernel(*args, **kw)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_backward_matches_the_formulas(size, dtype):
    _check_backward(size, dtype, 100 + sum(size))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_backward_with_many_requests_of_a_voice(dtype):
    _check_backward((40, 45, 24, 40, 12, 2), dtype, 3)
    _check_backward((1, 1500, 24, 40, 12, 1), dtype, 4)   # one long request: its rows are cut


def test_gradients_against_differences():
    """Central differences of the definition in float64, linear in each argument: with steps of 1e-4 they are off by less
    than 1e-6 here; the rest is the kernel's bound."""
    from tts_amd.adapters import adapter_backward as kernel
    dy, x, down, up, voices, scale, lengths = _inputs(4, 20, 12, 18, 3, 2, torch.float32, 11)
    got = kernel(*_cuda(dy, x, down, up, voices), scale=scale.cuda(), lengths=lengths.cuda())
    bounds = adapter_backward(dy, x, down, up, voices, scale, lengths)
    zero = torch.zeros_like(dy).double()
    gen = torch.Generator().manual_seed(1)

    def loss(x, down, up):
        return float((adapter(zero, x, down, up, voices, scale, lengths)[0] * dy.double()).sum())

    for at in range(3):
        base = [t.double() for t in (x, down, up)]
        v = torch.randn(base[at].shape, generator=gen).double()
        plus, minus = list(base), list(base)
        plus[at], minus[at] = base[at] + 1e-4 * v, base[at] - 1e-4 * v
        slope = (loss(*plus) - loss(*minus)) / 2e-4
        w, tol = bounds[at]
        limit = 1e-6 + float(((tol + F32 * w.abs()) * v.abs()).sum())
        assert abs(float((got[at].cpu().double() * v).sum()) - slope) <= limit


def test_empty_inputs():
    from tts_amd.adapters import adapter_add
    from tts_amd.adapters import adapter_backward as backward
    down, up = torch.randn(2, 4, 8, device="cuda"), torch.randn(2, 4, 6, device="cuda")
    for B, T in ((0, 5), (3, 0)):
        y, x = torch.empty(B, T, 6, device="cuda"), torch.empty(B, T, 8, device="cuda")
        voices = torch.zeros(B, dtype=torch.int32, device="cuda")
        assert adapter_add(y, x, down, up, voices).shape == (B, T, 6)
        dx, ddown, dup = backward(y, x, down, up, voices)
        assert dx.shape == x.shape and not ddown.any() and not dup.any()


def test_refusals_on_the_device():
    from tts_amd.adapters import adapter_add
    y, x, down, up, voices, scale, _ = _cuda(*_inputs(3, 10, 16, 24, 4, 2, torch.float32, 12))
    with pytest.raises(IndexError, match="voices"):
        adapter_add(y, x, down, up, [0, 2, 1])
    with pytest.raises(ValueError, match="lengths"):
        adapter_add(y, x, down, up, voices, lengths=[0, 11, 1])
    with pytest.raises(ValueError, match="voices must be"):
        adapter_add(y, x, down, up, voices[:2])
    buf = torch.zeros(3, 10, 40, device="cuda")
    with pytest.raises(ValueError, match="out overlaps x"):
        adapter_add(y, buf[..., :16], down, up, voices, out=buf[..., 8:32])
    with pytest.raises(ValueError, match="out overlaps y"):
        adapter_add(buf[..., :24], x, down, up, voices, out=buf[..., 1:25])
    with pytest.raises(ValueError, match="share memory"):
        adapter_add(y, x, down, up, voices, out=y[:1].expand(3, -1, -1))
    with pytest.raises(ValueError, match="contiguous"):
        adapter_add(y, x, down, up, voices, out=torch.zeros(3, 24, 10, device="cuda").transpose(1, 2))
    with pytest.raises(ValueError, match="overlaps an adapter"):
        adapter_add(y[:1, :2], x[:1, :2], down, up, voices[:1], out=up.view(-1)[:48].view(1, 2, 24))


def test_another_stream_and_a_replayed_graph():
    from tts_amd.adapters import adapter_add
    from tts_amd.adapters import adapter_backward as backward
    y, x, down, up, voices, scale, lengths = _cuda(*_inputs(5, 90, 64, 136, 16, 3, torch.bfloat16, 13))

    def work():
        return [adapter_add(y, x, down, up, voices, scale=scale, lengths=lengths),
                *backward(y, x, down, up, voices, scale=scale, lengths=lengths)]
    want = [t.clone() for t in work()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = work()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for k in range(4):
        x.copy_(torch.randn(x.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(k)))
        eager = [t.clone() for t in work()]
        for t in out:
            t.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, out))


def test_an_adapted_projection_in_front_of_the_recurrence():
    """The operators as they are used: a shared projection leaves values and gate logits, each request's voice adapts
    them in place, the recurrence runs over the two halves; a stream that takes the same positions one at a time ends in
    the same state, and the gradients flow back through both."""
    from tts_amd.adapters import adapter_add
    from tts_amd.adapters import adapter_backward as backward
    from tts_amd.recurrence import gated_scan, gated_scan_backward, gated_step
    gen = torch.Generator().manual_seed(2)
    B, T, K, D, R, V = 4, 90, 24, 20, 4, 3
    x = torch.randn(B, T, K, generator=gen)
    W = torch.randn(2 * D, K, generator=gen) / K ** 0.5
    down, up = torch.randn(V, R, K, generator=gen) / K ** 0.5, torch.randn(V, R, 2 * D, generator=gen) / R ** 0.5
    voices, lengths = torch.tensor([2, -1, 0, 2]), torch.tensor([90, 41, 64, 1])
    gx, gW, gd, gu, gv = _cuda(x, W, down, up, voices.int())
    both = gx @ gW.t()
    adapter_add(both, gx, gd, gu, gv, lengths=lengths.tolist(), out=both)
    h, last, states = gated_scan(both[..., :D], both[..., D:], lengths=lengths.tolist(), save_states=True)
    # step by step, one position of every request at a time
    state = torch.zeros(B, D, device="cuda")
    for t in range(T):
        now = gx[:, t] @ gW.t()
        now = adapter_add(now, gx[:, t], gd, gu, gv)
        _, new = gated_step(now[:, :D], now[:, D:], state)
        state = torch.where((lengths > t).cuda()[:, None], new, state)
    # float64 throughout
    ref_both = x.double() @ W.double().t()
    for b in range(B):
        if voices[b] >= 0:
            n = int(lengths[b])
            ref_both[b, :n] += (x[b, :n].double() @ down[voices[b]].double().t()) @ up[voices[b]].double()
    ref_h, ref_last, _ = scan(ref_both[..., :D], ref_both[..., D:], None, lengths)
    # values and logits are sums of 28 products of size below 20, off by at most 64 F32 of that; a state collects
    # that once per step at worst
    tol = 64 * F32 * 20 * T
    assert _excess(h, ref_h, tol) <= 0 and _excess(last, ref_last, tol) <= 0 and _excess(state, ref_last, tol) <= 0
    dh = torch.randn(B, T, D, generator=gen)
    dx_, dg_, _ = gated_scan_backward(dh.cuda(), both[..., :D], both[..., D:], states, lengths=lengths.tolist())
    dx, ddown, dup = backward(torch.cat([dx_, dg_], -1), gx, gd, gu, gv, lengths=lengths.tolist())
    rx, rg, _, _, _ = scan_backward(dh, ref_both[..., :D], ref_both[..., D:], None, None, lengths)
    d = torch.cat([rx, rg], -1)
    for g, (w, bound) in zip((dx, ddown, dup), adapter_backward(d, x, down, up, voices, lengths=lengths)):
        # d itself is off by `tol` of its largest value; `bound` holds the sums of magnitudes in units of about K F32
        assert _excess(g, w, tol * float(d.abs().max()) * (1 + bound / (4 * F32))) <= 0


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("size", [(40, 130, 80, 260, 12, 3), (30, 200, 264, 90, 30, 4), (50, 100, 96, 140, 64, 2)], ids=str)
def test_middling_batches(size, dtype):
    """Between few tiles, which are cut into halves, and many, which get four waves each."""
    from tts_amd.adapters import adapter_add
    y, x, down, up, voices, scale, lengths = _inputs(*size, dtype, 9)
    want, tol = adapter(y, x, down, up, voices, scale, lengths)
    out = adapter_add(*_cuda(y, x, down, up, voices), scale=scale.cuda(), lengths=lengths.cuda())
    assert _excess(out, want, tol * (1 + half_step(dtype)) + _rounding(dtype, want)) <= 0
    _check_backward(size, dtype, 10)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rank", [4, 20, 40])
@pytest.mark.parametrize("B,T", [(3, 41), (20, 900)])
def test_columns_behind_the_last_block(B, T, rank, dtype):
    """Rows that end one to nine columns behind a block of 64 (fp32) or 128, few tiles and many."""
    from tts_amd.adapters import adapter_add
    for N in (65, 66, 68, 73, 129, 130, 132, 133):
        y, x, down, up, voices, scale, lengths = _inputs(B, T, 24, N, rank, 2, dtype, N)
        want, tol = adapter(y, x, down, up, voices, scale, lengths)
        gy, gx, gd, gu, gv, gs, gl = _cuda(y, x, down, up, voices, scale, lengths)
        out = adapter_add(gy, gx, gd, gu, gv, scale=gs, lengths=gl)
        assert _excess(out, want, tol * (1 + half_step(dtype)) + _rounding(dtype, want)) <= 0
        for b in range(B):
            n = 0 if int(voices[b]) < 0 else int(lengths[b])
            assert torch.equal(out[b, n:].cpu(), y[b, n:])
        assert torch.equal(adapter_add(gy, gx, gd, gu, gv, scale=gs, lengths=gl, out=gy), out)
    _check_backward((B, T, 129, 65, rank, 2), dtype, 5)
    _check_backward((B, T, 66, 132, rank, 2), dtype, 6)
