"""The gated linear recurrence on the GPU against its formulas in float64: types, odd sizes, ragged and empty requests,
both directions, strides, carried state, gradients, the step form, streams and graphs."""
import pytest
import torch

from seq_ref import F32, half_step, scan, scan_backward, scan_error

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _inputs(B, T, D, dtype, seed, ragged=False, strided=True):
    gen = torch.Generator().manual_seed(seed)
    both = torch.randn(B, T, 2 * D + 3, generator=gen)
    both[..., D:] = both[..., D:] * 1.5 + torch.linspace(-2, 5, D + 3)
    both = both.to(dtype)
    if strided:   # two slices of one projection, the second at an odd offset
        x, g = both[..., 1:D + 1], both[..., D + 2:2 * D + 2]
    else:
        x, g = both[..., :D].contiguous(), both[..., D:2 * D].contiguous()
    h0 = torch.randn(B, D, generator=gen)
    lengths = None
    if ragged:
        lengths = torch.randint(0, T + 1, (B,), generator=gen, dtype=torch.int32)
        lengths[0] = T
        if B > 2:
            lengths[1], lengths[2] = 0, 1
    return x, g, h0, lengths


def _gpu(t):
    if t is None:
        return None
    out = torch.empty(0)
    if t.is_contiguous():
        return t.cuda()
    base = torch.as_strided(t, (t.untyped_storage().nbytes() // t.element_size(),), (1,), 0).cuda()   # the same strides on the device
    out = torch.as_strided(base, t.shape, t.stride(), t.storage_offset())
    return out


def _excess(got, want, tol):
    """How far the worst element is beyond its tolerance (a number at or below 0 passes)."""
    return float(((got.cpu().double() - want).abs() - tol).max())


SIZES = [(1, 1, 1), (1, 1, 512), (3, 2, 7), (2, 63, 33), (1, 64, 64), (4, 65, 129), (3, 129, 8), (5, 255, 40), (2, 257, 72),
         (1, 1000, 20), (3, 700, 136)]


def _check_scan(x, g, h0, lengths, reverse, dtype):
    from tts_amd.recurrence import gated_scan
    want_h, want_last, want_states = scan(x, g, h0, lengths, reverse)
    h, last, states = gated_scan(_gpu(x), _gpu(g), h0=_gpu(h0), lengths=_gpu(lengths), reverse=reverse, save_states=True)
    assert h.dtype == dtype and last.dtype == states.dtype == torch.float32
    tol = scan_error(x, g, h0, x.shape[1], lengths)
    small = 2.0 ** -25 if dtype == torch.float16 else 0.0   # half a step of its smallest values
    assert _excess(h, want_h, tol + small + half_step(dtype) * want_h.abs()) <= 0
    assert _excess(last, want_last, tol) <= 0
    assert _excess(states, want_states, tol) <= 0
    if lengths is not None:
        for b, n in enumerate(lengths.tolist()):
            assert not h[b, n:].any()
    h2, last2 = gated_scan(_gpu(x), _gpu(g), h0=_gpu(h0), lengths=_gpu(lengths), reverse=reverse)
    assert torch.equal(h, h2) and torch.equal(last, last2)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("reverse", [False, True])
def test_scan_matches_the_steps(size, dtype, reverse):
    x, g, h0, lengths = _inputs(*size, dtype, 1 + sum(size), ragged=size[0] > 1)
    _check_scan(x, g, h0 if size[0] != 3 else None, lengths, reverse, dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_scan_over_a_cut_time_axis(dtype):
    """One request, few channels: the time axis is spread over the chip."""
    x, g, h0, _ = _inputs(1, 9000, 9, dtype, 5)
    _check_scan(x, g, h0, None, False, dtype)
    x, g, h0, lengths = _inputs(3, 5000, 17, dtype, 6, ragged=True)
    _check_scan(x, g, h0, lengths, True, dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("reverse", [False, True])
def test_cut_time_axis_of_whole_channel_groups(dtype, reverse):
    """The same where lanes take several channels: both passes, short requests that end chunks early."""
    x, g, h0, lengths = _inputs(4, 4100, 16, dtype, 7, ragged=True)
    _check_scan(x, g, h0, lengths, reverse, dtype)
    _check_backward(x, g, h0, lengths, reverse, dtype, 9)


def test_scan_of_strided_and_repeated_inputs():
    """Time-major activations, a channel axis that is not contiguous, and a batch that repeats one request."""
    from tts_amd.recurrence import gated_scan
    x, g, h0, _ = _inputs(4, 50, 24, torch.float32, 3, strided=False)
    want, last = gated_scan(x.cuda(), g.cuda())
    tx, tg = x.transpose(0, 1).contiguous().cuda().transpose(0, 1), g.transpose(0, 1).contiguous().cuda().transpose(0, 1)
    assert torch.equal(gated_scan(tx, tg)[0], want)
    cx = x.transpose(1, 2).contiguous().cuda().transpose(1, 2)
    assert torch.equal(gated_scan(cx, g.cuda())[0], want)
    one = gated_scan(x[:1].cuda().expand(4, -1, -1), g.cuda())[0]
    assert torch.equal(one[0], want[0])
    assert torch.equal(one, gated_scan(x[:1].repeat(4, 1, 1).cuda(), g.cuda())[0])


def test_gates_at_their_ends():
    """A logit of -inf restarts the state at x, +inf keeps it; far logits stay finite."""
    from tts_amd.recurrence import gated_scan, gated_scan_backward
    for dtype in TYPES:
        x = torch.tensor([1.0, 2.0, 3.0, 4.0, 5.0, 6.0]).view(1, 6, 1).to(dtype).cuda()
        inf = float("inf")
        far = 60000.0
        g = torch.tensor([-inf, inf, -far, far, inf, -inf]).view(1, 6, 1).to(dtype).cuda()
        h, last, states = gated_scan(x, g, h0=torch.full((1, 1), 9.0, device="cuda"), save_states=True)
        assert h.flatten().tolist() == [1, 1, 3, 3, 3, 6] and float(last) == 6
        dx, dg, dh0 = gated_scan_backward(torch.ones_like(x), x, g, states)
        assert dx.flatten().tolist() == [2, 0, 3, 0, 0, 1] and not dg.any() and float(dh0) == 0


def test_what_lies_behind_the_end_is_not_read():
    from tts_amd.recurrence import gated_scan, gated_scan_backward
    x, g, h0, _ = _inputs(4, 150, 40, torch.bfloat16, 8, strided=False)
    lengths = torch.tensor([150, 0, 64, 77], dtype=torch.int32)
    dh = torch.randn(4, 150, 40, generator=torch.Generator().manual_seed(1)).bfloat16()
    clean = []
    for fill in (0.0, float("nan"), float("inf")):
        for b, n in enumerate(lengths.tolist()):
            x[b, n:], g[b, n:], dh[b, n:] = fill, fill, fill
        h, last, states = gated_scan(x.cuda(), g.cuda(), h0=h0.cuda(), lengths=lengths.cuda(), save_states=True)
        grads = gated_scan_backward(dh.cuda(), x.cuda(), g.cuda(), states, lengths=lengths.cuda())
        clean.append([h, last, states, *grads])
    for other in clean[1:]:
        for a, b in zip(clean[0], other):
            assert torch.equal(a, b)
    assert torch.equal(clean[0][1][1].cpu(), h0[1])


def test_lengths_out_of_range_are_clamped_on_the_device():
    from tts_amd.recurrence import gated_scan
    x, g, h0, _ = _inputs(3, 20, 8, torch.float32, 9, strided=False)
    wild = torch.tensor([-5, 1000, 7], dtype=torch.int32, device="cuda")
    h, last = gated_scan(x.cuda(), g.cuda(), lengths=wild)
    want, want_last = gated_scan(x.cuda(), g.cuda(), lengths=[0, 20, 7])
    assert torch.equal(h, want) and torch.equal(last, want_last)
    assert torch.equal(gated_scan(x.cuda(), g.cuda(), lengths=wild.long() * 2 ** 33 // 2 ** 33)[0], want)


def _check_backward(x, g, h0, lengths, reverse, dtype, seed):
    from tts_amd.recurrence import gated_scan, gated_scan_backward
    gen = torch.Generator().manual_seed(seed)
    dh = torch.randn(x.shape, generator=gen).to(dtype)
    dh_last = torch.randn(x.shape[0], x.shape[2], generator=gen)
    dx, dg, dh0, G, before = scan_backward(dh, x, g, h0, dh_last, lengths, reverse)
    _, _, states = gated_scan(_gpu(x), _gpu(g), h0=_gpu(h0), lengths=_gpu(lengths), reverse=reverse, save_states=True)
    got = gated_scan_backward(dh.cuda(), _gpu(x), _gpu(g), states, dh_last=dh_last.cuda(), lengths=_gpu(lengths),
                              reverse=reverse)
    T = x.shape[1]
    eh = scan_error(x, g, h0, T, lengths)
    # G runs through the same maps with dh in the place of w x: the same bound on its own largest value
    m = max(float(G.abs().max()), float(dh_last.abs().max()))
    eG = 16 * F32 * m * min(T, 1 + float(torch.exp(g.double().max())))
    f, w = torch.sigmoid(g.double()), torch.sigmoid(-g.double())
    diff = (before - x.double()).abs()
    small = 2.0 ** -25 if dtype == torch.float16 else 0.0   # half a step of its smallest values
    tol_x = half_step(dtype) * dx.abs() + w * (eG + 16 * F32 * (1 + g.double().abs()) * G.abs()) + small
    tol_g = half_step(dtype) * dg.abs() + small + f * w * (eh * G.abs() + diff * eG + 16 * F32 * (1 + g.double().abs()) * diff * G.abs())
    if lengths is not None:
        live = torch.arange(T)[None, :] < lengths[:, None]
        tol_x, tol_g = (torch.where(live[:, :, None], t, 0.0) for t in (tol_x, tol_g))
    assert _excess(got[0], dx, tol_x) <= 0
    assert _excess(got[1], dg, tol_g) <= 0
    assert _excess(got[2], dh0, eG) <= 0


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("reverse", [False, True])
def test_backward_matches_the_formulas(size, dtype, reverse):
    x, g, h0, lengths = _inputs(*size, dtype, 2 + sum(size), ragged=size[0] > 1)
    _check_backward(x, g, h0, lengths, reverse, dtype, sum(size))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_backward_over_a_cut_time_axis(dtype):
    x, g, h0, _ = _inputs(1, 7000, 9, dtype, 15)
    _check_backward(x, g, h0, None, True, dtype, 3)
    x, g, h0, lengths = _inputs(3, 4000, 17, dtype, 16, ragged=True)
    _check_backward(x, g, h0, lengths, False, dtype, 4)


def test_gradients_against_differences():
    """Central differences of the definition in float64; their own error is below 1e-9 here, so the kernel's bound (16
    units over a memory of at most 70 steps, of sums of 130 terms below 20) holds alone."""
    from tts_amd.recurrence import gated_scan, gated_scan_backward
    x, g, h0, lengths = _inputs(3, 70, 5, torch.float32, 21, ragged=True, strided=False)
    gen = torch.Generator().manual_seed(4)
    dh, dh_last = torch.randn(3, 70, 5, generator=gen), torch.randn(3, 5, generator=gen)
    _, _, states = gated_scan(x.cuda(), g.cuda(), h0=h0.cuda(), lengths=lengths.cuda(), save_states=True)
    dx, dg, dh0 = gated_scan_backward(dh.cuda(), x.cuda(), g.cuda(), states, dh_last=dh_last.cuda(), lengths=lengths.cuda())

    def loss(x, g, h0):
        h, last, _ = scan(x, g, h0, lengths)
        return float((h * dh.double()).sum() + (last * dh_last.double()).sum())
    eps = 1e-5
    for k in range(3):
        vx, vg, vh = (torch.randn(t.shape, generator=gen).double() for t in (x, g, h0))
        for v, grad, at in ((vx, dx, 0), (vg, dg, 1), (vh, dh0, 2)):
            plus, minus = [t.double() for t in (x, g, h0)], [t.double() for t in (x, g, h0)]
            plus[at], minus[at] = plus[at] + eps * v, minus[at] - eps * v
            slope = (loss(*plus) - loss(*minus)) / (2 * eps)
            terms = grad.cpu().double() * v
            bound = 1e-7 + 16 * F32 * 70 * float(v.abs().sum()) * 20
            assert abs(float(terms.sum()) - slope) <= bound


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("size", [(1, 1), (1, 512), (3, 7), (17, 129), (256, 64)], ids=str)
def test_step_equals_a_scan_of_one(size, dtype):
    from tts_amd.recurrence import gated_scan, gated_step
    x, g, h0, _ = _inputs(size[0], 1, size[1], dtype, 30 + size[1])
    y, h = gated_step(_gpu(x)[:, 0], _gpu(g)[:, 0], h0.cuda())
    want_y, want_h = gated_scan(_gpu(x), _gpu(g), h0=h0.cuda())
    assert torch.equal(y, want_y[:, 0]) and torch.equal(h, want_h)
    state = h0.cuda()
    y2, same = gated_step(_gpu(x)[:, 0], _gpu(g)[:, 0], state, out=state)
    assert same is state and torch.equal(state, h) and torch.equal(y2, y)


def test_steps_chunks_and_the_whole_sequence_agree():
    """A stream taken step by step, in chunks with the state carried, and at once."""
    from tts_amd.recurrence import gated_scan, gated_step
    x, g, h0, _ = _inputs(2, 200, 24, torch.float32, 40, strided=False)
    x, g, h0 = x.cuda(), g.cuda(), h0.cuda()
    whole, last = gated_scan(x, g, h0=h0)
    tol = 2 * scan_error(x.cpu(), g.cpu(), h0.cpu(), 200)
    h, parts = h0, []
    for a, b in ((0, 1), (1, 70), (70, 71), (71, 200)):
        y, h = gated_scan(x[:, a:b], g[:, a:b], h0=h)
        parts.append(y)
    assert (torch.cat(parts, 1) - whole).abs().max() <= tol and (h - last).abs().max() <= tol
    h = h0.clone()
    for t in range(200):
        y, _ = gated_step(x[:, t], g[:, t], h, out=h)
        assert (y - whole[:, t]).abs().max() <= tol
    assert (h - last).abs().max() <= tol


def test_empty_inputs():
    from tts_amd.recurrence import gated_scan, gated_scan_backward, gated_step
    x, h0 = torch.empty(2, 0, 8, device="cuda"), torch.randn(2, 8, device="cuda")
    h, last, states = gated_scan(x, x, h0=h0, save_states=True)
    assert h.shape == (2, 0, 8) and torch.equal(last, h0) and states.shape == (2, 0, 8)
    assert torch.equal(gated_scan_backward(x, x, x, states, dh_last=h0)[2], h0)
    none = torch.empty(0, 8, device="cuda")
    assert gated_step(none, none, none)[0].shape == (0, 8)


def test_refusals_on_the_device():
    from tts_amd.recurrence import gated_scan, gated_step
    x = torch.zeros(2, 5, 8, device="cuda")
    with pytest.raises(ValueError, match="lengths"):
        gated_scan(x, x, lengths=[6, 1])
    with pytest.raises(ValueError, match="lengths"):
        gated_scan(x, x, lengths=torch.tensor([1.0, 2.0], device="cuda"))
    with pytest.raises(Exception, match="no CPU path"):
        gated_scan(x, x.cpu())
    h = torch.zeros(3, 8, device="cuda")
    with pytest.raises(ValueError, match="overlaps h"):
        gated_step(x[:, 0], x[:, 0], h[:2], out=h[1:])
    with pytest.raises(ValueError, match="overlaps x"):
        gated_step(x[:, 0], torch.zeros(2, 8, device="cuda"), h[:2], out=x.view(-1)[:16].view(2, 8))
    with pytest.raises(ValueError, match="out must be"):
        gated_step(x[:, 0], x[:, 0], h[:2], out=torch.zeros(2, 8, device="cuda", dtype=torch.bfloat16))


def test_another_stream_and_a_replayed_graph():
    """Results do not depend on the stream, and a captured call gives the eager result on every replay, also while
    eager calls run between the replays."""
    from tts_amd.recurrence import gated_scan, gated_scan_backward, gated_step
    x, g, h0, lengths = _inputs(2, 3000, 24, torch.bfloat16, 50, ragged=True, strided=False)
    x, g, h0, lengths, dh = x.cuda(), g.cuda(), h0.cuda(), lengths.cuda(), torch.randn(2, 3000, 24, device="cuda").bfloat16()

    def work():
        h, last, states = gated_scan(x, g, h0=h0, lengths=lengths, save_states=True)
        y, hn = gated_step(x[:, 0], g[:, 0], last)
        return [h, last, states, y, hn, *gated_scan_backward(dh, x, g, states, lengths=lengths)]
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
