"""The sequence operators at the ends of their ranges on the GPU: offsets beyond 32 bits, rows at the furthest distance and
beyond it, several calls at once, and what a refused call leaves behind."""
import pytest
import torch

pytestmark = pytest.mark.gpu

FAR = 1 << 20        # elements between two rows, at most


def _far(T, stride, columns, seed, first=5):
    """[1,T,columns] bfloat16 whose rows lie `stride` elements apart, and the same contiguous."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    near = torch.randn(1, T, columns, device="cuda", generator=gen).bfloat16()
    buf = torch.empty(T * stride, dtype=torch.bfloat16, device="cuda")
    far = buf.as_strided((1, T, columns), (T * stride, stride, 1), first)
    far.copy_(near)
    return far, near


@pytest.mark.parametrize("stride", [FAR, FAR + 8], ids=["furthest", "copied"])
@pytest.mark.parametrize("reverse", [False, True])
def test_rows_far_apart_in_the_recurrence(stride, reverse):
    """2100 rows, the last one more than 2^31 elements behind the first."""
    from tts_amd.recurrence import gated_scan, gated_scan_backward
    both, near = _far(2100, stride, 48, 1)
    dh, near_dh = _far(2100, stride, 24, 2)
    want = gated_scan(near[..., :24], near[..., 24:], reverse=reverse, save_states=True)
    got = gated_scan(both[..., :24], both[..., 24:], reverse=reverse, save_states=True)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    a = gated_scan_backward(near_dh, near[..., :24], near[..., 24:], want[2], reverse=reverse)
    b = gated_scan_backward(dh, both[..., :24], both[..., 24:], want[2], reverse=reverse)
    assert all(torch.equal(s, t) for s, t in zip(a, b))


def test_results_beyond_32_bits_of_the_recurrence():
    """2100 steps of 2^20 channels.  A logit of -inf makes the state x, its gradient that of the state."""
    from tts_amd.recurrence import gated_scan, gated_scan_backward, gated_step
    T, D = 2100, FAR
    gen = torch.Generator(device="cuda").manual_seed(3)
    row = torch.randn(1, 1, D, device="cuda", generator=gen).bfloat16()
    x, g = row.expand(1, T, D), torch.full_like(row, -float("inf")).expand(1, T, D)
    h, last, states = gated_scan(x, g, save_states=True)
    assert bool((h == row).all()) and torch.equal(last, row[:, 0].float()) and bool((states[:, 1:] == row.float()).all())
    del h
    dx, dg, dh0 = gated_scan_backward(x, x, g, states)
    assert bool((dx == row).all()) and not dg.any() and not dh0.any()
    del dx, dg, states
    state = torch.zeros(T, D, device="cuda")
    y, _ = gated_step(x[0], g[0], state, out=state)
    assert bool((y == row[0]).all()) and bool((state == row[0].float()).all())


@pytest.mark.parametrize("stride", [FAR, FAR + 8], ids=["furthest", "copied"])
def test_rows_far_apart_in_the_adapters(stride):
    from tts_amd.adapters import adapter_add, adapter_backward
    gen = torch.Generator(device="cuda").manual_seed(4)
    K, N, R, V = 40, 72, 6, 2
    down = (torch.randn(V, R, K, device="cuda", generator=gen) / K ** 0.5).bfloat16()
    up = torch.randn(V, R, N, device="cuda", generator=gen).bfloat16()
    both, near = _far(2100, stride, K + N, 5)
    want = adapter_add(near[..., K:], near[..., :K], down, up, [1])
    assert torch.equal(adapter_add(both[..., K:], both[..., :K], down, up, [1]), want)
    for a, b in zip(adapter_backward(near[..., K:], near[..., :K], down, up, [1]),
                    adapter_backward(both[..., K:], both[..., :K], down, up, [1])):
        assert torch.equal(a, b)
    if stride == FAR:
        out = adapter_add(both[..., K:], both[..., :K], down, up, [1], out=both[..., K:])
        assert torch.equal(out, want) and torch.equal(both[..., :K], near[..., :K])
    else:                                                        # an output is not copied: its rows are as near as that
        with pytest.raises(Exception, match="row stride"):
            adapter_add(near[..., K:], near[..., :K], down, up, [1], out=both[..., K:])


def test_adapters_of_voices_nobody_has_are_not_read():
    from tts_amd.adapters import adapter_add, adapter_backward
    gen = torch.Generator(device="cuda").manual_seed(6)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        y, x = (torch.randn(3, 40, n, device="cuda", generator=gen).to(dtype) for n in (72, 33))
        down, up = (torch.randn(3, 5, n, device="cuda", generator=gen).to(dtype) for n in (33, 72))
        scale = torch.rand(3, device="cuda", generator=gen)
        results = []
        for fill in (0.0, float("nan")):
            down[1], up[1], scale[1] = fill, fill, fill
            results.append([adapter_add(y, x, down, up, [2, 0, -1], scale=scale),
                            *adapter_backward(y, x, down, up, [2, 0, -1], scale=scale)])
        assert all(torch.equal(a, b) for a, b in zip(*results))
        assert not results[1][2][1].any() and not results[1][3][1].any()


def test_calls_at_once_on_several_streams():
    from tts_amd.adapters import adapter_add, adapter_backward
    from tts_amd.recurrence import gated_scan, gated_scan_backward
    gen = torch.Generator(device="cuda").manual_seed(7)
    sets = [(torch.randn(2, 3000, 64, device="cuda", generator=gen), torch.randn(2, 5, 64, device="cuda", generator=gen) / 8)
            for _ in range(3)]
    voices = torch.tensor([1, 0], dtype=torch.int32, device="cuda")

    def work(x, m):
        h, last, states = gated_scan(x, x, save_states=True)
        return [h, last, adapter_add(h, x, m, m, voices), *gated_scan_backward(x, x, x, states),
                *adapter_backward(h, x, m, m, voices)]
    want = [work(*s) for s in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], []
    for _ in range(2):
        got = []
        for s, stream in zip(sets, streams):
            with torch.cuda.stream(stream):
                got.append(work(*s))
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(s, t) for s, t in zip(a, b))


def test_a_refused_voice_leaves_the_carried_state():
    from tts_amd import synthetic
    from tts_amd.tacotron2 import Tacotron2
    m = Tacotron2(num_chars=129, num_speakers=0, r=7, attn_norm="sigmoid", prenet_type="bn", prenet_dropout=False,
                  separate_stopnet=True)
    m.load_state_dict(synthetic.t2_state_dict(seed=0))
    m = m.cuda().eval()
    m.load_voices(torch.randn(2, 4, 512) / 512 ** 0.5, torch.randn(2, 4, 512))
    ids = torch.as_tensor(synthetic.t2_text_ids(3, 1, 20)).cuda().long()
    state = (torch.zeros(2, 1, 256, device="cuda"), torch.zeros(2, 1, 256, device="cuda"))
    for bad in ([2], [0, 1], [0.5]):
        with pytest.raises((IndexError, ValueError)):
            m.encode(ids, rnn_state=state, voice_ids=bad)
    assert not state[0].any() and not state[1].any()
    plain = m.encode(ids, rnn_state=state)
    again = (torch.zeros(2, 1, 256, device="cuda"), torch.zeros(2, 1, 256, device="cuda"))
    got = m.encode(ids, rnn_state=again, voice_ids=[1])
    assert torch.equal(state[0], again[0]) and torch.equal(state[1], again[1])       # beside the layer, not inside it
    assert not torch.equal(got, plain)
    m.decoder.set_r(1)
    one = m.inference_truncated(ids)[0]
    m.reset_truncated()
    m.decoder.max_decoder_steps = 12
    m.reset_truncated()
    two = m.inference_truncated(ids, voice_ids=[1])[0]
    n = min(one.shape[1], two.shape[1])
    assert torch.isfinite(two).all() and not torch.equal(one[:, :n], two[:, :n])


def test_very_many_short_requests():
    """70 000 requests of three steps: the same as the same requests in two calls."""
    from tts_amd.adapters import adapter_add, adapter_backward
    from tts_amd.recurrence import gated_scan, gated_scan_backward, gated_step
    gen = torch.Generator(device="cuda").manual_seed(8)
    B, T, D, V = 70000, 3, 4, 2
    x, g, dh = (torch.randn(B, T, D, device="cuda", generator=gen) for _ in range(3))
    lengths = torch.randint(0, T + 1, (B,), device="cuda", generator=gen, dtype=torch.int32)
    halves = [slice(0, B // 2), slice(B // 2, B)]
    h, last, states = gated_scan(x, g, lengths=lengths, save_states=True)
    grads = gated_scan_backward(dh, x, g, states, lengths=lengths)
    for s in halves:
        a, b, c = gated_scan(x[s], g[s], lengths=lengths[s].clone(), save_states=True)
        assert torch.equal(a, h[s]) and torch.equal(b, last[s])
        for p, q in zip(gated_scan_backward(dh[s], x[s], g[s], c, lengths=lengths[s].clone()), grads):
            assert torch.equal(p, q[s])
    y, _ = gated_step(x[:, 0], g[:, 0], last)
    assert torch.equal(y[-5:], gated_step(x[-5:, 0], g[-5:, 0], last[-5:])[0])
    m = torch.randn(V, 3, D, device="cuda", generator=gen)
    voices = torch.randint(-1, V, (B,), device="cuda", generator=gen, dtype=torch.int32)
    out = adapter_add(x, g, m, m, voices, lengths=lengths)
    dx, ddown, dup = adapter_backward(x, g, m, m, voices, lengths=lengths)
    parts = [adapter_backward(x[s], g[s], m, m, voices[s].clone(), lengths=lengths[s].clone()) for s in halves]
    for s, p in zip(halves, parts):
        assert torch.equal(adapter_add(x[s], g[s], m, m, voices[s].clone(), lengths=lengths[s].clone()), out[s])
        assert torch.equal(p[0], dx[s])
    # whole numbers, whose sums stay below 2^24: the weights' gradients are exact
    x, g = (torch.randint(-2, 3, (B, T, D), device="cuda", generator=gen).float() for _ in range(2))
    m = torch.randint(-1, 2, (V, 3, D), device="cuda", generator=gen).float()
    _, ddown, dup = adapter_backward(x, g, m, m, voices, lengths=lengths)
    live = (torch.arange(T, device="cuda")[None] < lengths[:, None]).double()[..., None]
    for v in range(V):
        d, i = x[voices == v].double(), g[voices == v].double()
        d, i = (d * live[voices == v]).reshape(-1, D), (i * live[voices == v]).reshape(-1, D)
        assert torch.equal(ddown[v].double(), (d @ m[v].double().t()).t().contiguous() @ i)
        assert torch.equal(dup[v].double(), (i @ m[v].double().t()).t().contiguous() @ d)


def test_no_columns():
    """A projection without inputs adds nothing; one without outputs has nothing to add to."""
    from tts_amd.adapters import adapter_add, adapter_backward
    y, v = torch.randn(2, 5, 6, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    none, up = torch.empty(2, 5, 0, device="cuda"), torch.randn(1, 3, 6, device="cuda")
    out = adapter_add(y, none, torch.empty(1, 3, 0, device="cuda"), up, v)
    assert torch.equal(out, y) and out.data_ptr() != y.data_ptr()
    assert adapter_add(y, none, torch.empty(1, 3, 0, device="cuda"), up, v, out=y) is y
    dx, ddown, dup = adapter_backward(y, none, torch.empty(1, 3, 0, device="cuda"), up, v)
    assert dx.shape == none.shape and ddown.shape == (1, 3, 0) and not dup.any()
    assert adapter_add(none, y, up, torch.empty(1, 3, 0, device="cuda"), v).shape == (2, 5, 0)
    assert not adapter_backward(none, y, up, torch.empty(1, 3, 0, device="cuda"), v)[0].any()
