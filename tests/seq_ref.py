"""The sequence operators in float64 on the CPU, written from their formulas (test infrastructure)."""
import torch

F32 = torch.finfo(torch.float32).eps / 2


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def scan(x, g, h0=None, lengths=None, reverse=False, block=64):
    """h, h_last, states of the gated recurrence, step by step."""
    x, g = x.double(), g.double()
    B, T, D = x.shape
    f, w = 1 / (1 + torch.exp(-g)), 1 / (1 + torch.exp(g))
    h = torch.zeros(B, T, D, dtype=torch.float64)
    last = torch.zeros(B, D, dtype=torch.float64)
    states = torch.zeros(B, -(-T // block), D, dtype=torch.float64)
    for b in range(B):
        n = T if lengths is None else int(lengths[b])
        s = torch.zeros(D, dtype=torch.float64) if h0 is None else h0[b].double()
        for p in range(n):
            if p % block == 0:
                states[b, p // block] = s
            t = n - 1 - p if reverse else p
            s = f[b, t] * s + w[b, t] * x[b, t]
            h[b, t] = s
        states[b, -(-n // block):] = s
        last[b] = s
    return h, last, states


def scan_backward(dh, x, g, h0=None, dh_last=None, lengths=None, reverse=False):
    """dx, dg, dh0 and, for error bounds, G and the state in front of every step."""
    dh, x, g = dh.double(), x.double(), g.double()
    B, T, D = x.shape
    f, w = 1 / (1 + torch.exp(-g)), 1 / (1 + torch.exp(g))
    h, _, _ = scan(x, g, h0, lengths, reverse)
    dx, dg, G_all, before = (torch.zeros(B, T, D, dtype=torch.float64) for _ in range(4))
    dh0 = torch.zeros(B, D, dtype=torch.float64)
    for b in range(B):
        n = T if lengths is None else int(lengths[b])
        r = torch.zeros(D, dtype=torch.float64) if dh_last is None else dh_last[b].double()
        for p in range(n - 1, -1, -1):
            t = n - 1 - p if reverse else p
            prev = t + 1 if reverse else t - 1
            if p == 0:
                hp = torch.zeros(D, dtype=torch.float64) if h0 is None else h0[b].double()
            else:
                hp = h[b, prev]
            G = dh[b, t] + r
            dx[b, t], dg[b, t] = w[b, t] * G, f[b, t] * w[b, t] * (hp - x[b, t]) * G
            r = f[b, t] * G
            G_all[b, t], before[b, t] = G, hp
        dh0[b] = r
    return dx, dg, dh0, G_all, before


def scan_error(x, g, h0, T, lengths=None):
    """Bound on the error of a state kept in fp32.  Per step w = 1 / (1 + e^g) carries at most (|g| + 6) F32 of itself
    (the exponent's argument, the exponential, the sum, the reciprocal's 2) and f = 1 - w that and half a unit, the update
    2 more; as w |g| <= 0.28 that is below 8 F32 of the largest magnitude m of x and h0, which bounds h too.  Composing pairs instead of steps
    rounds each factor at most twice: 16.  The errors of n steps add up while the memory 1 / w lasts."""
    x, g = x.double(), g.double()
    if lengths is not None:
        live = torch.arange(x.shape[1])[None, :] < torch.as_tensor(lengths)[:, None]
        x = torch.where(live[:, :, None], x, 0.0)
        g = torch.where(live[:, :, None], g, 0.0)
    m = max(float(x.abs().max()), 0.0 if h0 is None else float(h0.abs().max()))
    memory = 1.0 + float(torch.exp(g.max()))
    return 16 * F32 * m * min(T, memory)


# u handed from one product to the next as two 16-bit numbers: each leaves at most half a step of the type
SPLIT = {torch.float64: 0.0, torch.float32: 0.0, torch.bfloat16: 2.0 ** -16, torch.float16: 2.0 ** -22}


def _live(lengths, b, T):
    return T if lengths is None else max(0, min(T, int(lengths[b])))


def adapter(y, x, down, up, voices, scale=None, lengths=None):
    """out and a bound on its error before the one rounding to y's type.  Sums of n fp32 products are off by at most
    n F32 of the sum of their magnitudes; u carries that into the second product, and the split of its type."""
    dtype, T = y.dtype, y.shape[1]
    y, x, down, up = (t.double() for t in (y, x, down, up))
    out, tol = y.clone(), torch.zeros_like(y)
    K, R = x.shape[2], down.shape[1]
    for b in range(y.shape[0]):
        n, v = _live(lengths, b, T), int(voices[b])
        if not 0 <= v < down.shape[0] or n == 0:
            continue
        s = 1.0 if scale is None else float(scale[v])
        u = x[b, :n] @ down[v].t()
        size = x[b, :n].abs() @ down[v].abs().t()
        out[b, :n] += s * (u @ up[v])
        top = u.abs().amax(1, keepdim=True)
        eu = (K + 4) * F32 * size + SPLIT[dtype] * top
        tol[b, :n] = abs(s) * ((eu @ up[v].abs()) + (2 * R + 4) * F32 * ((u.abs() + eu) @ up[v].abs()))
        tol[b, :n] += 2 * F32 * (y[b, :n].abs() + out[b, :n].abs())
    return out, tol


def adapter_backward(dy, x, down, up, voices, scale=None, lengths=None):
    """(dx, bound), (ddown, bound), (dup, bound)."""
    dtype, T = dy.dtype, dy.shape[1]
    dy, x, down, up = (t.double() for t in (dy, x, down, up))
    dx, gd, gu = torch.zeros_like(x), torch.zeros_like(down), torch.zeros_like(up)
    tx, td, tu = torch.zeros_like(x), torch.zeros_like(down), torch.zeros_like(up)
    K, N, R = x.shape[2], dy.shape[2], down.shape[1]
    rows = torch.zeros(down.shape[0])
    for b in range(dy.shape[0]):
        n, v = _live(lengths, b, T), int(voices[b])
        if 0 <= v < down.shape[0]:
            rows[v] += n
    for b in range(dy.shape[0]):
        n, v = _live(lengths, b, T), int(voices[b])
        if not 0 <= v < down.shape[0] or n == 0:
            continue
        s = 1.0 if scale is None else float(scale[v])
        xb, d = x[b, :n], dy[b, :n]
        u, du = s * xb @ down[v].t(), s * d @ up[v].t()
        eu = abs(s) * (K + 4) * F32 * (xb.abs() @ down[v].abs().t()) + SPLIT[dtype] * u.abs().amax(1, keepdim=True)
        edu = abs(s) * (N + 4) * F32 * (d.abs() @ up[v].abs().t()) + SPLIT[dtype] * du.abs().amax(1, keepdim=True)
        dx[b, :n] = du @ down[v]
        tx[b, :n] = edu @ down[v].abs() + (2 * R + 4) * F32 * ((du.abs() + edu) @ down[v].abs())
        gd[v] += du.t() @ xb
        gu[v] += u.t() @ d
        many = (2 * float(rows[v]) + 4) * F32
        td[v] += edu.t() @ xb.abs() + many * ((du.abs() + edu).t() @ xb.abs())
        tu[v] += eu.t() @ d.abs() + many * ((u.abs() + eu).t() @ d.abs())
    return (dx, tx), (gd, td), (gu, tu)
