"""Low-rank adapters of many voices beside a shared projection, running on libttsx (gfx950).

    out[b,t] = y[b,t] + scale[v] (x[b,t] down[v]^T) up[v],        v = voices[b],   y = x W^T

A voice of the reference is one embedding added to the encoder outputs (Tacotron2/TTS/models.py:838-849).  An adapter
lets it change a projection too, at R (K + N) numbers per voice, and a batch may hold as many voices as requests: the
shared product runs once for all of them, `adapter_add` adds each request's own part.

    out             = adapter_add(y, x, down, up, voices)        # whole sequences [B,T,.] or single positions [B,.]
    dx, ddown, dup  = adapter_backward(dy, x, down, up, voices)  # for fitting the adapters

Activations and adapters are float32, bfloat16 or float16 tensors on the GPU, alike in type; products are summed in
float32.  As elsewhere in this package there is no CPU path and no autograd graph: gradients are a call of their own,
so inputs that require them are refused outside `torch.no_grad()`, and inputs with a tangent anywhere.  Calls work on
the current stream of the tensors' device, allocate through torch and do not synchronise (`voices` or `lengths` on the
host are copied over first, which does), so they can be captured into a graph.
"""
import functools

import torch

from . import _lib
from ._seq import (DTYPES, are_tensors, call, columns_apart, lengths_on, on_device, overlapping, overlaps, pointer, rows, same_place,
                   voices_on, ways, writable_rows)

MAX_RANK = 64                     # TTSX_ADAPTER_MAX_RANK
MAX_WIDTH = FURTHEST = 1 << 20   # columns, and elements between two rows, of a call
MAX_ROWS = 1 << 30                # positions, and requests
MAX_VOICES = 1 << 24


@functools.lru_cache(maxsize=512)
def _workspace_bytes(B, T, K, N, R, dtype):
    n = _lib.load().ttsx_adapter_backward_workspace(B, T, K, N, R, dtype)
    if n < 0:
        _lib.check(int(n), "ttsx_adapter_backward_workspace")
    return n


def _check(what, name, wide, x, down, up, scale):
    """Shapes and types: `wide` is y or dy."""
    are_tensors(what, (name, wide), ("x", x), ("down", down), ("up", up))
    if scale is not None:
        are_tensors(what, ("scale", scale))
    shape, x_shape, d_shape, u_shape = wide.shape, x.shape, down.shape, up.shape
    if len(shape) not in (2, 3) or len(x_shape) != len(shape) or x_shape[0] != shape[0] or x_shape[-2] != shape[-2]:
        raise ValueError("%s: %s [B,T,N] and x [B,T,K] (or [B,N] and [B,K]) must agree, got %s and %s"
                         % (what, name, tuple(wide.shape), tuple(x.shape)))
    K, N = x_shape[-1], shape[-1]
    if (len(d_shape) != 3 or len(u_shape) != 3 or d_shape[0] != u_shape[0] or d_shape[1] != u_shape[1]
            or d_shape[2] != K or u_shape[2] != N):
        raise ValueError("%s: down and up must be [V,R,%d] and [V,R,%d], got %s and %s"
                         % (what, K, N, tuple(down.shape), tuple(up.shape)))
    if max(K, N) > MAX_WIDTH:
        raise ValueError("%s: at most %d columns, got %d and %d" % (what, MAX_WIDTH, K, N))
    if shape[0] > MAX_ROWS or shape[-2] > MAX_ROWS:
        raise ValueError("%s: at most %d requests and positions, got %s" % (what, MAX_ROWS, tuple(shape)))
    V, R, _ = d_shape
    if V > MAX_VOICES:
        raise ValueError("%s: at most %d voices, got %d" % (what, MAX_VOICES, V))
    if not 1 <= R <= MAX_RANK or V < 1:
        raise ValueError("%s: the rank must lie in 1..%d, with at least one voice, got down %s"
                         % (what, MAX_RANK, tuple(down.shape)))
    dtype = x.dtype
    if dtype not in DTYPES or not dtype == wide.dtype == down.dtype == up.dtype:
        raise ValueError("%s: %s, x, down and up must all be float32, bfloat16 or float16, got %s, %s, %s and %s"
                         % (what, name, wide.dtype, x.dtype, down.dtype, up.dtype))
    if not down.is_contiguous() or not up.is_contiguous():
        raise ValueError("%s: down and up must be contiguous" % what)
    if scale is not None and (scale.shape != (V,) or scale.dtype != torch.float32):
        raise ValueError("%s: scale must be float32 [%d], got %s %s" % (what, V, scale.dtype, tuple(scale.shape)))
    dev = on_device(what, (name, wide), ("x", x), ("down", down), ("up", up), ("scale", scale))
    return dev, shape[0], shape[1] if len(shape) == 3 else 1, K, N, R, V


def _placed(t, keep=False):
    """t as an entry point takes it, with its batch and row strides (a single position has one row); `keep`: where it is."""
    single = t.dim() == 2
    if not keep:
        t = rows(t, None if single else FURTHEST)
    strides = t.stride()
    return t, strides[0], 0 if single else strides[1]


def adapter_add(y, x, down, up, voices, scale=None, lengths=None, out=None):
    """y [B,T,N] plus each request's adapter applied to x [B,T,K]; y [B,N] and x [B,K] are one position per request.

    down [V,R,K], up [V,R,N]: the adapters (ranks 1 to 64); voices [B]: which one each request has, -1 for none (on the
    device any number outside 0..V-1 is none); scale [V] float32: a factor per voice; lengths [B]: rows at positions >=
    lengths[b] stay y's and x is not read there.  `out` takes the result; out=y works in place and leaves rows without
    an adapter untouched.  The result has y's type, rounded once."""
    done = ways.ordinary.adapter_add(y, x, down, up, voices, scale, lengths, out)
    if done is not None:
        return done
    what = "adapter_add"
    dev, B, T, K, N, R, V = _check(what, "y", y, x, down, up, scale)
    in_place = False
    if out is not None:
        are_tensors(what, ("out", out))
        on_device(what, ("y", y), ("out", out))
        if out.shape != y.shape or out.dtype != y.dtype:
            raise ValueError("%s: out must be %s %s like y, got %s %s"
                             % (what, y.dtype, tuple(y.shape), out.dtype, tuple(out.shape)))
        writable_rows(what, "out", out)
        in_place = same_place(out, y)
        if not in_place and overlaps(out, y) and not columns_apart(out, y):
            raise ValueError("%s: out overlaps y" % what)
        if overlaps(out, x) and not columns_apart(out, x):
            raise ValueError("%s: out overlaps x" % what)
        if overlapping(out, (down, up) if scale is None else (down, up, scale)) is not None:
            raise ValueError("%s: out overlaps an adapter" % what)
        for name, t in (("voices", voices), ("lengths", lengths)):
            if isinstance(t, torch.Tensor) and t.is_cuda and overlaps(out, t):
                raise ValueError("%s: out overlaps %s" % (what, name))
    voices = voices_on(what, voices, B, V, x)
    lengths = lengths_on(what, lengths, B, T, x)
    if out is None:
        out = y.new_empty(y.shape)
    if B and T and N:
        if K == 0:
            if not in_place:
                out.copy_(y)
        else:
            (y, yb, yt), (x, xb, xt), (_, ob, ot) = _placed(y, in_place), _placed(x), _placed(out, True)
            scale = None if scale is None else scale.contiguous()
            call("ttsx_adapter_add", dev, y.data_ptr(), yb, yt, x.data_ptr(), xb, xt, down.data_ptr(), up.data_ptr(),
                 voices.data_ptr(), pointer(scale), pointer(lengths), B, T, K, N, R, V, DTYPES[y.dtype], out.data_ptr(), ob,
                 ot)
    return out


def adapter_backward(dy, x, down, up, voices, scale=None, lengths=None):
    """Gradients of `adapter_add` for x, down and up from dy [B,T,N], the gradient of its result (y's own gradient is dy).
    Returns dx [B,T,K] (zero in rows without an adapter; not summed over axes that x was broadcast along), ddown
    [V,R,K] and dup [V,R,N] of their inputs' type: sums over all rows of a voice, kept in float32 and in a fixed order,
    so that two runs agree to the bit.  `scale` is a constant."""
    done = ways.ordinary.adapter_backward(dy, x, down, up, voices, scale, lengths)
    if done is not None:
        return done
    what = "adapter_backward"
    dev, B, T, K, N, R, V = _check(what, "dy", dy, x, down, up, scale)
    voices = voices_on(what, voices, B, V, x)
    lengths = lengths_on(what, lengths, B, T, x)
    dx = x.new_empty(x.shape)
    if not (B and T and K and N):
        return dx.zero_(), torch.zeros_like(down), torch.zeros_like(up)
    ddown, dup = torch.empty_like(down), torch.empty_like(up)
    dtype = DTYPES[x.dtype]
    need = _workspace_bytes(B, T, K, N, R, dtype)
    ws = x.new_empty((need,), dtype=torch.uint8)
    (dy, db, dt), (x, xb, xt) = _placed(dy), _placed(x)
    scale = None if scale is None else scale.contiguous()
    call("ttsx_adapter_backward", dev, dy.data_ptr(), db, dt, x.data_ptr(), xb, xt, down.data_ptr(),
         up.data_ptr(), voices.data_ptr(), pointer(scale), pointer(lengths), B, T, K, N, R, V, dtype, dx.data_ptr(),
         ddown.data_ptr(), dup.data_ptr(), ws.data_ptr(), need)
    return dx, ddown, dup
