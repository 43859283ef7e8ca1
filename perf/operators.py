"""Cases of the sequence operators: the gated linear recurrence (`tts_amd.recurrence`) and the voices' low-rank
adapters (`tts_amd.adapters`), each in its plain form (elementary torch operations in 32 bits) and as a call of the
framework's kernels.

    gated_scan            h_t = f_t h_{t-1} + (1 - f_t) x_t,  f_t = sigmoid(g_t), over [B,T,D]
    gated_scan_backward   its gradients, from the states that the forward pass left every 64 steps
    gated_step            one step for every request of a batch
    adapter_add           y + scale_v (x down_v^T) up_v, each request with a voice of its own
    adapter_backward      its gradients for x, down and up

Lengths and voices: a ragged batch has a fixed set of lengths per case (one empty request and one of a single step
from 16 requests on) that the seed deals out; every eighth request of a batch speaks with the shared weights alone
(voice -1).
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BLOCK = 64   # steps between two states that the forward pass keeps for the backward pass


# ---------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one sentence of a hundred symbols through a recurrent layer of the encoder's width, as it arrives
        dict(name="scan_sentence", op="scan", B=1, T=100, D=512, dtype="fp32", ragged=False, reverse=False, keep=False),
        # a padded batch of 64 utterances of up to 800 frames, right to left
        dict(name="scan_frames", op="scan", B=64, T=800, D=512, dtype="fp32", ragged=True, reverse=True, keep=False),
        # one long text as frames, half an hour of 16-bit activations: few channels, a long axis; the states are kept
        dict(name="scan_long", op="scan", B=1, T=32000, D=1024, dtype="bf16", ragged=False, reverse=False, keep=True),
        # a small training batch of odd sizes
        dict(name="scan_backward_odd", op="scan_backward", B=5, T=301, D=257, dtype="fp32", ragged=True, reverse=True),
        # the training batch: 64 utterances of up to 800 frames
        dict(name="scan_backward_frames", op="scan_backward", B=64, T=800, D=1024, dtype="bf16", ragged=True,
             reverse=False),
        # the next frame of one stream
        dict(name="step_one", op="step", B=1, D=512, dtype="fp32"),
        # the next frame of 256 streams served together
        dict(name="step_many", op="step", B=256, D=2048, dtype="bf16"),
        # the next frame of 64 streams: one row each, the decoder's gate projection
        dict(name="adapter_single", op="adapter", B=64, T=1, K=1024, N=4096, R=16, V=16, dtype="bf16", ragged=False),
        # a batch of 64 texts beside the input projection of the bidirectional encoder layer
        dict(name="adapter_text", op="adapter", B=64, T=128, K=512, N=2048, R=32, V=8, dtype="bf16", ragged=True),
        # 64 utterances of up to 800 frames beside the projection to the linear spectrogram
        dict(name="adapter_frames", op="adapter", B=64, T=800, K=256, N=1025, R=16, V=8, dtype="fp32", ragged=True),
        # fitting the adapters of a few voices to a batch of texts
        dict(name="adapter_backward_text", op="adapter_backward", B=32, T=128, K=512, N=2048, R=16, V=4, dtype="fp32",
             ragged=True),
        # fitting them to whole utterances
        dict(name="adapter_backward_frames", op="adapter_backward", B=64, T=800, K=512, N=2048, R=32, V=8,
             dtype="bf16", ragged=True),
    ]


def _log_size(rng, lo, hi, step=8):
    """A whole number spread over the logarithm of [lo, hi]; half of them multiples of `step`."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5 and n >= step:
        n -= n % step
    return max(lo, min(hi, n))


def _draw_once(rng):
    op = rng.choice(["scan", "scan_backward", "step", "adapter", "adapter_backward"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if op == "step":
        return dict(op=op, B=_log_size(rng, 1, 256), D=_log_size(rng, 16, 2048), dtype=dtype)
    if op in ("scan", "scan_backward"):
        case = dict(op=op, B=_log_size(rng, 1, 64), T=_log_size(rng, 1, 32000, 64), D=_log_size(rng, 16, 1024),
                    dtype=dtype, ragged=rng.random() < 0.6, reverse=rng.random() < 0.5)
        if op == "scan":
            case["keep"] = rng.random() < 0.5
        return case
    T = 1 if op == "adapter" and rng.random() < 0.3 else _log_size(rng, 2, 800)
    return dict(op=op, B=_log_size(rng, 1, 64), T=T, K=_log_size(rng, 16, 2048, 64), N=_log_size(rng, 16, 4096, 64),
                R=rng.choice([4, 8, 16, 32, 64, rng.randint(1, 64)]), V=_log_size(rng, 1, 32), dtype=dtype,
                ragged=T > 1 and rng.random() < 0.6)


def draw(rng):
    most_bytes = max(work(c)["bytes"] for c in listed())
    most_flops = max(work(c)["flops"] for c in listed())
    while True:
        case = _draw_once(rng)
        need = work(case)
        if need["bytes"] <= most_bytes and need["flops"] <= most_flops and need["bytes"] > 0:
            return case


def _lengths(case):
    """The set of lengths of a case (the seed deals them out)."""
    B, T = case["B"], case["T"]
    if not case["ragged"]:
        return [T] * B
    lens = [max(1, min(T, int(round(T * (0.4 + 0.6 * (i + 1) / B))))) for i in range(B)]
    if B >= 16:
        lens[0], lens[1] = 0, 1
    return lens


def _voices(case):
    """Voice of every request, before the seed deals them out: every eighth has none."""
    return [-1 if i % 8 == 7 else i % case["V"] for i in range(case["B"])]


def work(case):
    op = case["op"]
    size = 4 if case["dtype"] == "fp32" else 2
    B, D = case["B"], case.get("D")
    if op == "step":
        return {"bytes": B * D * (3 * size + 8), "flops": 8 * B * D}
    rows, all_rows = sum(_lengths(case)), B * case["T"]
    if op == "scan":
        kept = -(-case["T"] // BLOCK) if case["keep"] else 0
        return {"bytes": D * ((2 * rows + all_rows) * size + (2 + kept) * B * 4), "flops": 8 * rows * D}
    if op == "scan_backward":
        blocks = sum(-(-n // BLOCK) for n in _lengths(case))
        return {"bytes": D * ((3 * rows + 2 * all_rows) * size + (blocks + 2 * B) * 4), "flops": 16 * rows * D}
    K, N, R, V = case["K"], case["N"], case["R"], case["V"]
    voices, lens = _voices(case), _lengths(case)
    live = sum(n for n, v in zip(lens, voices) if v >= 0)
    used = len({v for n, v in zip(lens, voices) if v >= 0 and n > 0})
    if op == "adapter":
        return {"bytes": (live * K + 2 * all_rows * N + used * R * (K + N)) * size, "flops": 2 * live * R * (K + N)}
    return {"bytes": (live * (K + N) + all_rows * K + (used + V) * R * (K + N)) * size,
            "flops": 2 * live * R * (3 * K + 2 * N)}


# --------------------------------------------------------------------------------------------------------- inputs
def _deal(case, gen):
    order = torch.randperm(case["B"], generator=gen, device="cuda").tolist()
    lens = _lengths(case)
    lengths = torch.tensor([lens[i] for i in order], dtype=torch.int32, device="cuda") if case["ragged"] else None
    if "V" not in case:
        return lengths, None
    voices = _voices(case)
    return lengths, torch.tensor([voices[i] for i in order], dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    op, B = case["op"], case["B"]

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=gen, device="cuda").mul_(scale).to(dtype)

    state = dict(case=case, op=op)
    if op in ("scan", "scan_backward", "step"):
        D = case["D"]
        # gate logits around a bias per channel: memories from one step to several hundred
        bias = torch.linspace(-2.0, 6.0, D, device="cuda")[torch.randperm(D, generator=gen, device="cuda")]
        h0 = torch.randn(B, D, generator=gen, device="cuda")
        if op == "step":
            g = (torch.randn(B, D, generator=gen, device="cuda") + bias).to(dtype)
            return dict(state, x=normal(B, D), g=g, h=h0)
        T = case["T"]
        # what a projection leaves: values and gate logits side by side
        both = torch.empty(B, T, 2 * D, device="cuda", dtype=dtype)
        both[..., :D] = torch.randn(B, T, D, generator=gen, device="cuda")
        both[..., D:] = torch.randn(B, T, D, generator=gen, device="cuda") + bias
        state["x"], state["g"] = both[..., :D], both[..., D:]
        state["lengths"], _ = _deal(case, gen)
        if op == "scan":
            return dict(state, h0=h0)
        _, _, states = _plain_scan(state["x"], state["g"], h0, state["lengths"], case["reverse"], True)
        return dict(state, h0=h0, states=states, dh=normal(B, T, D), dh_last=torch.randn(B, D, generator=gen, device="cuda"))
    T, K, N, R, V = (case[k] for k in ("T", "K", "N", "R", "V"))
    state["lengths"], state["voices"] = _deal(case, gen)
    state["x"] = normal(B, T, K)
    state["down"] = normal(V, R, K, scale=K ** -0.5)
    state["up"] = normal(V, R, N, scale=R ** -0.5)
    state["scale"] = 0.25 + torch.rand(V, generator=gen, device="cuda")
    state["y" if op == "adapter" else "dy"] = normal(B, T, N)
    return state


# ----------------------------------------------------------------------------------------------------- plain forms
def _in_order(t, lengths, reverse):
    """Rows of [B,T,D] in the order they are processed in (its own inverse): row p of request b is row
    lengths[b] - 1 - p where the recurrence runs right to left."""
    if not reverse:
        return t
    if lengths is None:
        return t.flip(1)
    p = torch.arange(t.shape[1], device=t.device)[None, :]
    last = lengths.long()[:, None]
    at = torch.where(p < last, last - 1 - p, p)
    return torch.gather(t, 1, at[:, :, None].expand_as(t))


def _alive(t, lengths):
    if lengths is None:
        return None
    return (torch.arange(t.shape[1], device=t.device)[None, :] < lengths[:, None])[:, :, None]


def _doubling(a, b):
    """All prefixes of the maps h -> a h + b along axis 1, by doubling."""
    step = 1
    while step < a.shape[1]:
        b = torch.cat([b[:, :step], b[:, step:] + a[:, step:] * b[:, :-step]], 1)
        a = torch.cat([a[:, :step], a[:, step:] * a[:, :-step]], 1)
        step *= 2
    return a, b


def _gates(x, g, lengths, reverse):
    """Keep and write shares of the gates and the values in 32 bits, in processing order; a row past the end keeps
    the state as it is."""
    x, g = _in_order(x.float(), lengths, reverse), _in_order(g.float(), lengths, reverse)
    f, w = torch.sigmoid(g), torch.sigmoid(-g)
    live = _alive(x, lengths)
    if live is not None:
        f, w, x = torch.where(live, f, 1.0), torch.where(live, w, 0.0), torch.where(live, x, 0.0)
    return f, w, x, live


def _plain_scan(x, g, h0, lengths, reverse, keep):
    f, w, v, live = _gates(x, g, lengths, reverse)
    a, b = _doubling(f, w * v)
    h = a * h0[:, None] + b
    last = h[:, -1].clone()
    out = h if live is None else torch.where(live, h, 0.0)
    out = _in_order(out, lengths, reverse).to(x.dtype)
    if not keep:
        return out, last, None
    states = torch.cat([h0[:, None], h[:, BLOCK - 1:-1:BLOCK]], 1)
    return out, last, states


def _plain_scan_backward(state):
    case, lengths, states = state["case"], state["lengths"], state["states"]
    f, w, v, live = _gates(state["x"], state["g"], lengths, case["reverse"])
    B, T, D = f.shape
    # the states again, block by block from the kept ones
    blocks = states.shape[1]
    pad = blocks * BLOCK - T
    fb = torch.nn.functional.pad(f, (0, 0, 0, pad), value=1.0).view(B * blocks, BLOCK, D)
    bb = torch.nn.functional.pad(w * v, (0, 0, 0, pad)).view(B * blocks, BLOCK, D)
    a, b = _doubling(fb, bb)
    start = states.reshape(B * blocks, 1, D)
    before = torch.cat([start, (a * start + b)[:, :-1]], 1).view(B, blocks * BLOCK, D)[:, :T]
    dh = _in_order(state["dh"].float(), lengths, case["reverse"])
    if live is not None:
        dh = torch.where(live, dh, 0.0)
    # G_t = dh_t + f_{t+1} G_{t+1}, from the last step on; the gradient of the last state comes in behind it
    ones = torch.ones(B, 1, D, device=f.device)
    a, b = _doubling(torch.cat([ones, f[:, 1:].flip(1)], 1), dh.flip(1))
    G = (a * state["dh_last"][:, None] + b).flip(1)
    dx, dg = w * G, f * w * (before - v) * G
    dh0 = f[:, 0] * G[:, 0]
    dtype = state["x"].dtype
    return (_in_order(dx, lengths, case["reverse"]).to(dtype), _in_order(dg, lengths, case["reverse"]).to(dtype), dh0)


def _adapter_parts(state):
    """Adapters of every request in 32 bits, its scale (0 without a voice) and the rows that count."""
    voices = state["voices"].long()
    at = voices.clamp(min=0)
    scale = torch.where(voices >= 0, state["scale"][at], 0.0)[:, None, None]
    return state["down"].float()[at], state["up"].float()[at], scale, _alive(state["x"], state["lengths"])


def _plain_adapter(state):
    down, up, scale, live = _adapter_parts(state)
    y = state["y"].float()
    z = scale * torch.bmm(torch.bmm(state["x"].float(), down.transpose(1, 2).contiguous()), up)
    if live is not None:
        z = torch.where(live, z, 0.0)
    return (y + z).to(state["y"].dtype)


def _plain_adapter_backward(state):
    down, up, scale, live = _adapter_parts(state)
    x, dy = state["x"].float(), scale * state["dy"].float()
    if live is not None:
        x, dy = torch.where(live, x, 0.0), torch.where(live, dy, 0.0)
    u = torch.bmm(x, down.transpose(1, 2).contiguous())
    du = torch.bmm(dy, up.transpose(1, 2).contiguous())
    dx = torch.bmm(du, down)
    each_down = torch.bmm(du.transpose(1, 2).contiguous(), x)
    each_up = torch.bmm(u.transpose(1, 2).contiguous(), dy)
    at = state["voices"].long().clamp(min=0)   # a request without a voice has a scale of zero: it adds nothing
    V = state["down"].shape[0]
    member = (torch.arange(V, device=at.device)[:, None] == at[None, :]).float()
    ddown = torch.mm(member, each_down.flatten(1)).view(V, *each_down.shape[1:])
    dup = torch.mm(member, each_up.flatten(1)).view(V, *each_up.shape[1:])
    dtype = state["x"].dtype
    return dx.to(dtype), ddown.to(dtype), dup.to(dtype)


def _run_plain(state):
    op, case = state["op"], state["case"]
    if op == "scan":
        h, last, states = _plain_scan(state["x"], state["g"], state["h0"], state["lengths"], case["reverse"],
                                      case["keep"])
        return (h, last, states) if case["keep"] else (h, last)
    if op == "scan_backward":
        return _plain_scan_backward(state)
    if op == "step":
        g = state["g"].float()
        h = torch.sigmoid(g) * state["h"] + torch.sigmoid(-g) * state["x"].float()
        return h.to(state["x"].dtype), h
    if op == "adapter":
        return _plain_adapter(state)
    return _plain_adapter_backward(state)


def _run_own(state):
    from tts_amd import adapters, recurrence
    op, case = state["op"], state["case"]
    if op == "scan":
        return recurrence.gated_scan(state["x"], state["g"], h0=state["h0"], lengths=state["lengths"],
                                     reverse=case["reverse"], save_states=case["keep"])
    if op == "scan_backward":
        return recurrence.gated_scan_backward(state["dh"], state["x"], state["g"], state["states"],
                                              dh_last=state["dh_last"], lengths=state["lengths"],
                                              reverse=case["reverse"])
    if op == "step":
        return recurrence.gated_step(state["x"], state["g"], state["h"])
    if op == "adapter":
        return adapters.adapter_add(state["y"], state["x"], state["down"], state["up"], state["voices"],
                                    scale=state["scale"], lengths=state["lengths"])
    return adapters.adapter_backward(state["dy"], state["x"], state["down"], state["up"], state["voices"],
                                     scale=state["scale"], lengths=state["lengths"])


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ----------------------------------------------------------------------------------------------- 64-bit definition
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "step":
        f = 1.0 / (1.0 + torch.exp(-s["g"].double()))
        w = 1.0 / (1.0 + torch.exp(s["g"].double()))
        h = f * s["h"].double() + w * s["x"].double()
        return h, h.clone()
    B, T = case["B"], case["T"]
    lens = [T] * B if s["lengths"] is None else s["lengths"].tolist()
    if op in ("scan", "scan_backward"):
        return _exact_scan(s, case, lens)
    voices, scale = s["voices"].tolist(), s["scale"].double()
    x, down, up = s["x"].double(), s["down"].double(), s["up"].double()
    if op == "adapter":
        out = s["y"].double()
        for b, (n, v) in enumerate(zip(lens, voices)):
            if v >= 0 and n > 0:
                out[b, :n] += scale[v] * ((x[b, :n] @ down[v].t()) @ up[v])
        return out
    dx, ddown, dup = torch.zeros_like(x), torch.zeros_like(down), torch.zeros_like(up)
    for b, (n, v) in enumerate(zip(lens, voices)):
        if v >= 0 and n > 0:
            xb, dz = x[b, :n], scale[v] * s["dy"][b, :n].double()
            du = dz @ up[v].t()
            dx[b, :n] = du @ down[v]
            ddown[v] += du.t() @ xb
            dup[v] += (xb @ down[v].t()).t() @ dz
    return dx, ddown, dup


def _exact_scan(s, case, lens):
    """Step by step over the rows of every request, in 64 bits."""
    B, T, D = case["B"], case["T"], case["D"]
    back, order = case["op"] == "scan_backward", []
    g, x = s["g"].double(), s["x"].double()
    f, w = 1.0 / (1.0 + torch.exp(-g)), 1.0 / (1.0 + torch.exp(g))
    full = min(lens) == T
    ends = torch.tensor(lens, device="cuda")
    for p in range(T):   # row of every request at step p
        order.append((T - 1 - p if case["reverse"] else p) if full else
                     torch.where(ends > p, ends - 1 - p if case["reverse"] else torch.full_like(ends, p), 0))
    every = torch.arange(B, device="cuda")
    pick = (lambda t, r: t[:, r]) if full else (lambda t, r: t[every, r])
    h = s["h0"].double()
    before, states = [], []
    out = torch.zeros(B, T, D, dtype=torch.float64, device="cuda")
    for p, r in enumerate(order):
        if p % BLOCK == 0:
            states.append(h)
        if back:
            before.append(h)
        new = pick(f, r) * h + pick(w, r) * pick(x, r)
        if full:
            h = new
            out[:, r] = h
        else:
            live = ends > p
            h = torch.where(live[:, None], new, h)
            out[every[live], r[live]] = h[live]
    if not back:
        return (out, h, torch.stack(states, 1)) if case["keep"] else (out, h)
    G = s["dh_last"].double()
    dh = s["dh"].double()
    dx, dg = torch.zeros_like(out), torch.zeros_like(out)
    for p in range(T - 1, -1, -1):
        r = order[p]
        ft, wt = pick(f, r), pick(w, r)
        total = pick(dh, r) + G
        gx, gg = wt * total, ft * wt * (before[p] - pick(x, r)) * total
        if full:
            dx[:, r], dg[:, r], G = gx, gg, ft * total
        else:
            live = ends > p
            at = r[live]
            dx[every[live], at], dg[every[live], at] = gx[live], gg[live]
            G = torch.where(live[:, None], ft * total, G)
    return dx, dg, G
