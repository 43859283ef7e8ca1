"""Gated linear recurrence over long sequences, running on libttsx (gfx950).

    f_t = sigmoid(g_t)        h_t = f_t h_{t-1} + (1 - f_t) x_t

A recurrent layer whose gates depend on the input alone: the time axis is a prefix scan instead of the chain of
dependent steps that the encoder's BiLSTM and the decoders' cells are (Tacotron2/TTS/models.py:419-427), so a text of
thousands of positions costs one pass over its activations.  The reference has no counterpart.

    h, h_last          = gated_scan(x, g)                       # whole sequences, carried state in and out
    h, h_last, states  = gated_scan(x, g, save_states=True)     # the same for training
    dx, dg, dh0        = gated_scan_backward(dh, x, g, states)
    y, h               = gated_step(x, g, h)                    # the next position of every stream

Values and gate logits are float32, bfloat16 or float16 tensors on the GPU, alike in type; states are float32 whatever
that type.  As elsewhere in this package there is no CPU path and no autograd graph: gradients are a call of their own,
so inputs that require them are refused outside `torch.no_grad()`, and inputs with a tangent anywhere.  Every call
works on the current stream of the tensors' device, allocates through torch and does not synchronise (a `lengths` on
the host is copied over first, which does), so it can be captured into a graph.
"""
import functools

import torch

from . import _lib
from ._seq import DTYPES, are_tensors, call, lengths_on, on_device, overlapping, pointer, rows, same_place, ways

STATE_BLOCK = 64             # steps between two kept states (TTSX_STATE_BLOCK)
MAX_CHANNELS = FURTHEST = 1 << 20   # channels, and elements between two rows, of a call
MAX_STEPS = 1 << 30          # steps, and requests


@functools.lru_cache(maxsize=512)
def _workspace_bytes(B, T, D, dtype, backward):
    n = _lib.load().ttsx_gated_scan_workspace(B, T, D, dtype, backward)
    if n < 0:
        _lib.check(int(n), "ttsx_gated_scan_workspace")
    return n


def _values_and_gates(what, x, g, axes):
    are_tensors(what, ("x", x), ("g", g))
    if x.dim() != len(axes) or g.shape != x.shape:
        raise ValueError("%s: x and g must both be [%s], got %s and %s"
                         % (what, ", ".join(axes), tuple(x.shape), tuple(g.shape)))
    if x.dtype not in DTYPES or g.dtype != x.dtype:
        raise ValueError("%s: x and g must both be float32, bfloat16 or float16, got %s and %s" % (what, x.dtype, g.dtype))
    if x.shape[-1] > MAX_CHANNELS:
        raise ValueError("%s: at most %d channels, got %d" % (what, MAX_CHANNELS, x.shape[-1]))
    if x.shape[0] > MAX_STEPS or x.shape[-2] > MAX_STEPS:
        raise ValueError("%s: at most %d requests and steps, got %s" % (what, MAX_STEPS, tuple(x.shape)))


def _state(what, name, t, B, D):
    if t is None:
        return None
    are_tensors(what, (name, t))
    if t.shape != (B, D) or t.dtype != torch.float32:
        raise ValueError("%s: %s must be float32 [%d, %d], got %s %s" % (what, name, B, D, t.dtype, tuple(t.shape)))
    return t


def _contiguous(t):
    return None if t is None else t.contiguous()


def gated_scan(x, g, h0=None, lengths=None, reverse=False, save_states=False):
    """Runs the recurrence over x, g [B,T,D] from the state h0 [B,D] (zero without it).

    `lengths` [B] makes the batch ragged: request b has the rows below lengths[b], and the rest of h is zero;
    a length of 0 leaves the state as it came.  `reverse` runs from the last of those rows to the first.  Returns h of
    x's type and the float32 state behind the last step; with `save_states` also the float32 states [B,ceil(T/64),D] in
    front of every 64th step, which `gated_scan_backward` starts from.

    x and g may be slices of one projection (any strides; the last axis is copied if it is not contiguous, and all of
    it if its rows lie more than 2^20 elements apart)."""
    done = ways.ordinary.scan(x, g, h0, lengths, reverse, save_states)
    if done is not None:
        return done
    what = "gated_scan"
    _values_and_gates(what, x, g, "BTD")
    B, T, D = x.shape
    h0 = _state(what, "h0", h0, B, D)
    dev = on_device(what, ("x", x), ("g", g), ("h0", h0))
    h0 = _contiguous(h0)
    lengths = lengths_on(what, lengths, B, T, x)
    x, g = rows(x, FURTHEST), rows(g, FURTHEST)
    h = x.new_empty((B, T, D))
    states = x.new_empty((B, -(-T // STATE_BLOCK), D), dtype=torch.float32) if save_states else None
    if B == 0 or T == 0 or D == 0:
        h_last = x.new_zeros((B, D), dtype=torch.float32) if h0 is None else h0.clone()
        return (h, h_last, states) if save_states else (h, h_last)
    h_last = x.new_empty((B, D), dtype=torch.float32) if h0 is None else torch.empty_like(h0)
    dtype = DTYPES[x.dtype]
    need = _workspace_bytes(B, T, D, dtype, 0)
    ws = x.new_empty((need,), dtype=torch.uint8) if need else None
    xs, gs = x.stride(), g.stride()
    call("ttsx_gated_scan", dev, x.data_ptr(), xs[0], xs[1], g.data_ptr(), gs[0], gs[1], pointer(h0), pointer(lengths),
         B, T, D, dtype, 1 if reverse else 0, h.data_ptr(), h_last.data_ptr(), pointer(states), pointer(ws), need)
    return (h, h_last, states) if save_states else (h, h_last)


def gated_scan_backward(dh, x, g, states, dh_last=None, lengths=None, reverse=False):
    """Gradients of `gated_scan` for x, g and h0, from the gradient dh [B,T,D] of h and (if given) dh_last [B,D] of the
    last state.  `states` is what the forward call with the same x, g, h0, lengths and reverse kept.  Returns dx and dg
    of x's type (zero behind a request's end; not summed over axes that x or g were broadcast along) and the float32
    dh0."""
    done = ways.ordinary.scan_backward(dh, x, g, states, dh_last, lengths, reverse)
    if done is not None:
        return done
    what = "gated_scan_backward"
    _values_and_gates(what, x, g, "BTD")
    are_tensors(what, ("dh", dh), ("states", states))
    B, T, D = x.shape
    if dh.shape != x.shape or dh.dtype != x.dtype:
        raise ValueError("%s: dh must be %s %s like x, got %s %s" % (what, x.dtype, tuple(x.shape), dh.dtype, tuple(dh.shape)))
    blocks = -(-T // STATE_BLOCK)
    if states.shape != (B, blocks, D) or states.dtype != torch.float32:
        raise ValueError("%s: states must be float32 [%d, %d, %d] as gated_scan(save_states=True) returns them, got %s %s"
                         % (what, B, blocks, D, states.dtype, tuple(states.shape)))
    dh_last = _state(what, "dh_last", dh_last, B, D)
    dev = on_device(what, ("x", x), ("g", g), ("dh", dh), ("states", states), ("dh_last", dh_last))
    dh_last = _contiguous(dh_last)
    lengths = lengths_on(what, lengths, B, T, x)
    dh, x, g, states = rows(dh, FURTHEST), rows(x, FURTHEST), rows(g, FURTHEST), states.contiguous()
    dx, dg = x.new_empty((B, T, D)), x.new_empty((B, T, D))
    if B == 0 or T == 0 or D == 0:
        return dx, dg, x.new_zeros((B, D), dtype=torch.float32) if dh_last is None else dh_last.clone()
    dh0 = x.new_empty((B, D), dtype=torch.float32)
    dtype = DTYPES[x.dtype]
    need = _workspace_bytes(B, T, D, dtype, 1)
    ws = x.new_empty((need,), dtype=torch.uint8) if need else None
    xs, gs, ds = x.stride(), g.stride(), dh.stride()
    call("ttsx_gated_scan_backward", dev, dh.data_ptr(), ds[0], ds[1], x.data_ptr(), xs[0], xs[1], g.data_ptr(), gs[0],
         gs[1], states.data_ptr(), pointer(dh_last), pointer(lengths), B, T, D, dtype, 1 if reverse else 0,
         dx.data_ptr(), dg.data_ptr(), dh0.data_ptr(), pointer(ws), need)
    return dx, dg, dh0


def gated_step(x, g, h, out=None):
    """The next step of B streams: x, g [B,D], float32 state h [B,D].  Returns (y, h'): the new state in x's type for
    the layer above, and in float32 for the next step.  `out` takes h' (a contiguous float32 [B,D]); out=h updates the
    state in place."""
    done = ways.ordinary.step(x, g, h, out)
    if done is not None:
        return done
    what = "gated_step"
    _values_and_gates(what, x, g, "BD")
    are_tensors(what, ("h", h))
    B, D = x.shape
    _state(what, "h", h, B, D)
    if out is not None:
        are_tensors(what, ("out", out))
    dev = on_device(what, ("x", x), ("g", g), ("h", h), ("out", out))
    state = h.contiguous()
    if out is None:
        out = torch.empty_like(state)
    else:
        if out.shape != (B, D) or out.dtype != torch.float32 or not out.is_contiguous():
            raise ValueError("%s: out must be contiguous float32 [%d, %d], got %s %s"
                             % (what, B, D, out.dtype, tuple(out.shape)))
        others = (x, g) if out is h or same_place(h, out) else (x, g, h)
        i = overlapping(out, others)
        if i is not None:
            raise ValueError("%s: out overlaps %s" % (what, "xgh"[i]))
    x, g = rows(x), rows(g)
    y = x.new_empty((B, D))
    if B and D:
        call("ttsx_gated_step", dev, x.data_ptr(), x.stride(0), g.data_ptr(), g.stride(0), state.data_ptr(), B, D,
             DTYPES[x.dtype], y.data_ptr(), out.data_ptr())
    return y, out
