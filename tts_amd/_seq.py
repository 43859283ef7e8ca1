"""Argument checks shared by the sequence operators (`recurrence`, `adapters`).

A call has two ways in.  `ordinary` (csrc/seq_calls.cpp) makes the whole call from native code where every argument is as
the entry point takes it, and returns None without doing anything where one is not; that call is checked, converted or
refused here in Python."""
import ctypes
import types

import torch
from torch.autograd import forward_ad

from . import _lib

DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


# What torch.cuda.current_stream() and torch.cuda.current_device() wrap: a call of the smallest size is bound by the host.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_functions = {}


class _Unbound:
    """Before the library is loaded, and in place of `ordinary` to have every call checked in Python."""
    step = scan = scan_backward = adapter_add = adapter_backward = staticmethod(lambda *args: None)


ways = types.SimpleNamespace(ordinary=_Unbound)


def _bind():
    """Loads both libraries; from here on ordinary calls are made natively."""
    lib = _lib.load()
    try:
        from . import _seqcalls
    except ImportError as e:
        raise _lib.TtsxError("tts_amd/_seqcalls.so cannot be loaded (%s): build it with `make -C tts_amd/csrc`" % e)
    _seqcalls.bind(*(ctypes.cast(getattr(lib, name), ctypes.c_void_p).value for name in (
        "ttsx_gated_step", "ttsx_gated_scan", "ttsx_gated_scan_backward", "ttsx_gated_scan_workspace", "ttsx_adapter_add",
        "ttsx_adapter_backward", "ttsx_adapter_backward_workspace")))
    ways.ordinary = _seqcalls


def call(name, index, *args):
    """The entry point `name` with `args` and the current stream of device `index`, run on that device."""
    fn = _functions.get(name)
    if fn is None:
        if not _functions:
            _bind()
        fn = _functions[name] = getattr(_lib.load(), name)
    if _current_device() == index:
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc != _lib.OK:
        _lib.check(rc, name)


def are_tensors(what, *named):
    for name, t in named:
        if type(t) is not torch.Tensor and not isinstance(t, torch.Tensor):
            raise ValueError("%s: %s must be a tensor, got %s" % (what, name, type(t).__name__))


def on_device(what, *named):
    """The index of the one GPU they are all on; none may be part of an autograd graph, carry a tangent or be a negated view (None
    stands for an argument left out)."""
    grad, index = torch.is_grad_enabled(), None
    tangents = forward_ad._current_level >= 0 and torch._C._is_fwd_grad_enabled()
    for name, t in named:
        if t is None:
            continue
        if grad and t.requires_grad:
            raise ValueError("%s records no autograd graph: call it under torch.no_grad(); gradients are a call of "
                             "their own" % what)
        if tangents and forward_ad.unpack_dual(t).tangent is not None:
            raise ValueError("%s has no forward-mode derivative: %s carries a tangent" % (what, name))
        if t.is_neg():
            raise ValueError("%s: %s is a view that negates what it shows: pass its resolve_neg()" % (what, name))
        i = t.get_device() if t.is_cuda else -1
        if index is None:
            index = i
        elif i != index:
            where = [str(t.device) for _, t in named if t is not None]
            if -1 in (i, index):
                raise _lib.TtsxError("%s runs on the GPU only: its tensors are on %s (there is no CPU path)"
                                     % (what, ", ".join(where)))
            raise ValueError("%s: its tensors are on %s" % (what, ", ".join(where)))
    if index < 0:
        raise _lib.TtsxError("%s runs on the GPU only: its tensors are on the CPU (there is no CPU path)" % what)
    return index


def pointer(t):
    return None if t is None else t.data_ptr()


def rows(t, furthest=None):
    """t with a contiguous last axis; other strides stay, up to `furthest` between rows (a single row lies anywhere)."""
    strides = t.stride()
    if (strides[-1] != 1 and t.shape[-1] > 1) or (furthest is not None and t.shape[-2] > 1 and strides[-2] > furthest):
        return t.contiguous()
    return t


def _index_tensor(what, name, t, B, like, lowest, highest, error):
    """[B] int32 on the device of `like`.  On the device already, any number is fine there; on the host they are checked."""
    if not isinstance(t, torch.Tensor):
        t = torch.as_tensor(t)
        t = t if t.numel() else t.int()         # an empty list has no type of its own
    if t.dim() != 1 or t.shape[0] != B or t.dtype not in (torch.int32, torch.int64):
        raise ValueError("%s: %s must be int32 or int64 [%d], got %s %s" % (what, name, B, t.dtype, tuple(t.shape)))
    if not t.is_cuda:
        if B and (int(t.min()) < lowest or int(t.max()) > highest):
            raise error("%s: %s must lie in %d..%d" % (what, name, lowest, highest))
    elif t.get_device() != like.get_device():
        raise ValueError("%s: %s is on %s, the others are on %s" % (what, name, t.device, like.device))
    elif t.dtype == torch.int32 and t.is_contiguous():
        return t
    # one beyond either end stands for all numbers there
    return t.clamp(lowest - 1, highest + 1).to(device=like.device, dtype=torch.int32).contiguous()


def lengths_on(what, lengths, B, T, like):
    """Lengths of a ragged batch: 0..T, clamped to that by the kernels."""
    return None if lengths is None else _index_tensor(what, "lengths", lengths, B, like, 0, T, ValueError)


def voices_on(what, voices, B, V, like):
    """Voices of a batch: 0..V-1, or -1 (any other number on the device) for none."""
    return _index_tensor(what, "voices", voices, B, like, -1, V - 1, IndexError)


def _span(t):
    if t.is_contiguous():
        n, first = t.numel(), t.data_ptr()
        return (first, first + n * t.element_size()) if n else None
    last = 1
    for n, stride in zip(t.shape, t.stride()):
        if n == 0:
            return None
        last += (n - 1) * stride
    first = t.data_ptr()
    return first, first + last * t.element_size()


def overlaps(a, b):
    """Whether the two tensors' memory ranges meet (strided tensors may interleave and still count)."""
    return overlapping(a, (b,)) is not None


def overlapping(a, others):
    """The index of the first of `others` whose memory range meets a's, or None."""
    span = _span(a)
    if span is not None:
        for i, t in enumerate(others):
            s = _span(t)
            if s is not None and span[0] < s[1] and s[0] < span[1]:
                return i
    return None


def same_place(a, b):
    return a is b or a.data_ptr() == b.data_ptr() and a.shape == b.shape and a.stride() == b.stride()


def columns_apart(a, b):
    """Whether two [...,n] tensors are different columns of the same rows (slices of one buffer)."""
    if a.stride()[:-1] != b.stride()[:-1] or a.shape[:-1] != b.shape[:-1] or a.element_size() != b.element_size():
        return False
    d = (b.data_ptr() - a.data_ptr()) // a.element_size()
    first, second = (a.shape[-1], b.shape[-1]) if d >= 0 else (b.shape[-1], a.shape[-1])
    pitch = min([s for s, n in zip(a.stride()[:-1], a.shape[:-1]) if n > 1] or [abs(d) + second])
    return first <= abs(d) and abs(d) + second <= pitch


def writable_rows(what, name, t):
    """Refuses an output [...,n] whose rows are not contiguous or share memory."""
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError("%s: the last axis of %s must be contiguous" % (what, name))
    if t.is_contiguous():
        return
    need = t.shape[-1]
    for stride, n in sorted((s, n) for s, n in zip(t.stride()[:-1], t.shape[:-1]) if n > 1):
        if stride < need:
            raise ValueError("%s: rows of %s share memory" % (what, name))
        need = stride * (n - 1) + need
